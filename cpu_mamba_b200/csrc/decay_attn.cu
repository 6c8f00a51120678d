// Decay attention: linear attention whose state decays by a scalar per head,
//   S_t = e^{g_t} S_{t-1} + k_t v_t^T          (S: Dk x Dv, fp32)
//   o_t = scale * S_t^T q_t
// for whole prompts (dense (B, T, ...) or packed sequences) and for one token
// with the state updated in place.  q, k and v may have fewer heads than the
// H decays; head h reads q head h / (H / Hq) and so on.
//
// This file: argument checks, the choice of kernel, the recurrent prompt
// kernel (any width up to 256, any stride, fp32 arithmetic) and the one-token
// kernel.
#include "decay.cuh"

#include <type_traits>

namespace mb2 {
namespace decay {

// ------------------------------------------------------- recurrent prompt
// One CTA walks one (sequence or segment, head, column tile) token by token, the
// state in registers: KG neighbouring lanes share C columns, each holding R rows
// of them (rows 4 KG i + 4 kg .. + 3, so a group's k and q loads are neighbours and
// all other lanes' are broadcasts).  With R <= 32 rows a lane, widths up to 32 need
// no sum over lanes at all.
//
// Deferred decay: the registers hold u_t = S_t / A_t, A_t the product of the
// decays since the last renormalisation.  Then u += k (v / A_t)^T and
// o = (scale A_t) u^T q: two FMAs per state element and token instead of three
// operations, done for two rows at a time (fma.rn.f32x2).  A run ends (u *= A,
// A = 1) when log A leaves [-5.5, 5.5], so v / A grows by 2^8 at most (|v| > 1e36
// would overflow) and every product has the relative precision it has without the
// factor.
//
// Bound: the FP32 pipe, 2 Dk Dv FMAs per token and head, and the shared-memory
// loads of k and q (two 16-byte loads per 4 C packed FMAs; a warp's 16-byte load
// takes four cycles of its SM's path to the registers even where all lanes read the
// same).  Above 32 rows, four columns of 16 rows a lane instead of two of 32 halve
// those loads for one more exchange between lanes: 1083 -> 890 us at 192 tokens, 2048
// heads of 128 x 128; 278 -> 246 with heads of 64 x 64.  Up to 32 rows they lose (24 x
// 64: 181 us two columns of all rows, 193 four of half).  One warp per head of 64
// columns instead of four with eight lanes a column: 425 -> 192 us at 151 sequences
// of 180 tokens, 24 heads of 24 x 64 (the FMAs alone take 54).
// tokens staged at a time: more where few walks wait for each step's latency
template <int R> __host__ __device__ constexpr int stage_tokens() { return R == 8 ? 32 : 16; }
constexpr float kRun = 5.5f;          // bound on |log A| within a run

// Copies rows [0, n) of a strided matrix into shared memory as fp32 (pitch
// `pitch`): asynchronous copies of fp32 rows, 16 bytes each where they allow it;
// bf16 rows through registers.  A thread's place in a row and its step are divided out once.
template <typename T> struct Stager {
    int per, r, c, dr, dc;                // pieces a row; first piece; step
    bool vec;
    __device__ __forceinline__ Stager(int cols, bool vec_, int tid, int threads) : vec(vec_) {
        per = vec ? cols / (16 / (int)sizeof(T)) : cols;
        r = tid / per;
        c = tid - r * per;
        dr = threads / per;
        dc = threads - dr * per;
    }
    __device__ __forceinline__ void operator()(float *dst, int pitch, const T *src, int64_t ld,
                                               int n) const {
        constexpr int E = 16 / (int)sizeof(T);
        int y = r, x = c;
        while (y < n) {
            if (vec) {
                float *to = dst + y * pitch + x * E;
                const T *from = src + y * ld + x * E;
                if constexpr (sizeof(T) == 4) {
                    cp_async16(to, from);
                } else {
                    const uint4 v = *reinterpret_cast<const uint4 *>(from);
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        *reinterpret_cast<float2 *>(to + 2 * e) = make_float2(
                            __uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u));
                }
            } else {
                if constexpr (sizeof(T) == 4) cp_async4(dst + y * pitch + x, src + y * ld + x);
                else dst[y * pitch + x] = io<T>::to_f(src[y * ld + x]);
            }
            y += dr;
            x += dc;
            if (x >= per) {
                x -= per;
                ++y;
            }
        }
    }
};

// R rows and C columns of the state a lane, KG lanes the same columns.  R 16 to 32 is for
// calls that fill the machine.  R 8 (two columns) is for few walks, where the step's latency is the
// call's time: eight tokens at once unless a run starts among them (one after the other
// 0.24 us a token, four 0.22), and other warps stage what comes next (beside the walk
// 0.20; with eight tokens 0.12; R 32 without any of it 0.36).
// STATE: the pass over segments that leaves their states; no q, no outputs
template <typename T, int KG, int R, int C, bool STATE>
__global__ void __launch_bounds__(KG == 1 ? 32 : R == 8 ? 256 : 128, KG == 1 ? 14 : R == 8 ? 2 : 3)
decay_recurrent_kernel(const Args a, int vtile, bool vec_q, bool vec_k, bool vec_v, bool pair_o) {
    constexpr int DK = KG * R, QUADS = R / 4;              // padded rows
    constexpr int L = stage_tokens<R>();
    extern __shared__ __align__(16) float smem_f[];
    float *const ks = smem_f;                              // [2][L][DK]
    float *const vs = ks + 2 * L * DK;                     // [2][L][vtile]
    float *const qs = vs + 2 * L * vtile;                  // [2][L][DK]
    // per token: the factor on u before it (1: none), 1 / A, scale * A
    __shared__ float4 s_f[2][L];
    __shared__ uint32_t s_again[2];   // the chunk's tokens that start a run

    const int tiles = (int)ceil_div(a.dv, vtile);
    int64_t id = blockIdx.x;
    const int tile = (int)(id % tiles);
    id /= tiles;
    const int h = (int)(id % a.heads);
    const Span sp = span_of<STATE>(a, id / a.heads);
    if (STATE && sp.out < 0) return;
    const int64_t row0 = sp.row0, len = sp.len;
    const int64_t bq = a.cu ? 0 : sp.seq;
    const float *const hin = !STATE && a.seg ? a.seg_state : a.h0;
    float *const hout = STATE ? a.seg_state : a.h_last;
    const T *q = static_cast<const T *>(a.q) + bq * a.qs[0] + row0 * a.qs[1] + (h / a.q_rep) * a.qs[2];
    const T *k = static_cast<const T *>(a.k) + bq * a.ks[0] + row0 * a.ks[1] + (h / a.k_rep) * a.ks[2];
    const int c0 = tile * vtile;
    const int cols = (int)(a.dv - c0 < vtile ? a.dv - c0 : vtile);
    const T *v = static_cast<const T *>(a.v) + bq * a.vs[0] + row0 * a.vs[1] +
                 (h / a.v_rep) * a.vs[2] + c0;
    const float *g = a.g + bq * a.gs[0] + row0 * a.gs[1] + h * a.gs[2];
    T *o = static_cast<T *>(a.o) + bq * a.os[0] + row0 * a.os[1] + h * a.os[2] + c0;

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // R 8: three warps stage the next chunk and a fourth takes its factors, beside the
    // warps that walk
    const int walkers = (int)blockDim.x - (R == 8 ? 128 : 0);
    const int loader = (int)threadIdx.x - (R == 8 ? walkers : 0);
    const int loaders = R == 8 ? 96 : (int)blockDim.x;
    const bool loads = loader >= 0 && loader < loaders;
    const bool first = R == 8 ? loader >= 96 : warp == 0;
    const int kg = lane & (KG - 1);
    const int col = C * ((int)threadIdx.x / KG);           // this lane's first column

    // columns past Dk and Dv are zero for the whole walk
    const int words = 2 * L * (vtile + (STATE ? 1 : 2) * DK);      // a multiple of 4
    for (int i = threadIdx.x; i < words / 4; i += blockDim.x)
        reinterpret_cast<float4 *>(smem_f)[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);

    uint64_t u[2 * QUADS][C];                              // row pairs x columns
    auto row_of = [&](int i) { return 4 * KG * (i >> 1) + 4 * kg + 2 * (i & 1); };
#pragma unroll
    for (int i = 0; i < 2 * QUADS; ++i)
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float e[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int dk = row_of(i) + j;
                e[j] = (sp.in >= 0 && dk < a.dk && col + c < cols)
                           ? hin[((sp.in * a.heads + h) * a.dk + dk) * a.dv + c0 + col + c]
                           : 0.0f;
            }
            u[i][c] = pair(__float_as_uint(e[0]), __float_as_uint(e[1]));
        }
    __syncthreads();

    const int nchunks = (int)ceil_div(len, (int64_t)L);
    const Stager<T> get_q((int)a.dk, vec_q, loader, loaders), get_k((int)a.dk, vec_k, loader, loaders),
        get_v(cols, vec_v, loader, loaders);
    auto load = [&](int n) {
        const int b = n & 1;
        const int64_t t0 = (int64_t)n * L;
        const int m = (int)(len - t0 < L ? len - t0 : L);
        if (!STATE) get_q(qs + b * L * DK, DK, q + t0 * a.qs[1], a.qs[1], m);
        get_k(ks + b * L * DK, DK, k + t0 * a.ks[1], a.ks[1], m);
        get_v(vs + b * L * vtile, vtile, v + t0 * a.vs[1], a.vs[1], m);
        cp_async_commit();
    };
    // log A is carried in 64 bits (the 16 or 32 decays of a chunk are added in 32): a head
    // that forgets over thousands of tokens adds as many equal decays, whose
    // roundings in 32 bits would all point one way.
    double run = 0.0;                 // log A after the chunk (the first warp)
    double span_g = 0.0;              // STATE: the sum of all log decays
    // the next chunk's decay of this lane's token, loaded a chunk ahead
    auto load_g = [&](int n) {
        const int64_t t = (int64_t)n * L + lane;
        return lane < L && t < len ? g[t * a.gs[1]] : 0.0f;
    };
    float gt_next = first ? load_g(0) : 0.0f;
    auto factors = [&](int n) {
        const int b = n & 1;
        const int64_t t0 = (int64_t)n * L;
        const int m = (int)(len - t0 < L ? len - t0 : L);
        const float gt = gt_next;
        gt_next = load_g(n + 1);
        float pre = gt, ren = 0.0f;
        bool r = false;
#pragma unroll
        for (int s = 1; s < L; s <<= 1) {
            const float below = __shfl_up_sync(0xffffffffu, pre, s);
            if (lane >= s) pre += below;
        }
        if (STATE) span_g += (double)__shfl_sync(0xffffffffu, pre, L - 1);
        double cum = run + (double)pre;
        // false for NaN and infinities too
        if (__all_sync(0xffffffffu, lane >= m || fabs(cum) <= kRun)) {
            run = __shfl_sync(0xffffffffu, cum, m - 1);
        } else {
            for (int t = 0; t < m; ++t) {
                const double next = run + (double)__shfl_sync(0xffffffffu, gt, t);
                const bool keep = fabs(next) <= kRun;
                run = keep ? next : 0.0;
                if (lane == t) { cum = run; ren = (float)next; r = !keep; }
            }
        }
        const uint32_t again_mask = __ballot_sync(0xffffffffu, r);
        if (lane == 0) s_again[b] = again_mask;
        if (lane < L) {
            const float hi = (float)cum, lo = (float)(cum - (double)hi);
            const float dn = expf(-hi), up = expf(hi);
            float again = 1.0f;
            if (r) again = expf(ren);
            s_f[b][lane] = make_float4(again, fmaf(dn, -lo, dn), fmaf(up, lo, up) * a.scale, 0.0f);
        }
    };

    if (nchunks > 0) {
        if (loads) load(0);
        if (first) factors(0);
    }
    for (int n = 0; n < nchunks; ++n) {
        const int b = n & 1;
        cp_async_wait<0>();
        __syncthreads();              // chunk n staged; chunk n - 1 read by every warp
        if (n + 1 < nchunks) {
            if (loads) load(n + 1);
            if (first) factors(n + 1);
        }
        if (R == 8 && loader >= 0) continue;
        const int64_t t0 = (int64_t)n * L;
        const int m = (int)(len - t0 < L ? len - t0 : L);
        const float *qb = qs + b * L * DK + 4 * kg;
        const float *kb = ks + b * L * DK + 4 * kg;
        const float *vb = vs + b * L * vtile + col;
        T *to = o + t0 * a.os[1] + col;
        // the start of a run
        auto again = [&](int t) {
            const float x = s_f[b][t].x;
            if (x == 1.0f) return;
            const uint64_t x2 = pair(x);
#pragma unroll
            for (int i = 0; i < 2 * QUADS; ++i)
#pragma unroll
                for (int c = 0; c < C; ++c) u[i][c] = mul2(u[i][c], x2);
        };
        // N tokens behind one another: their loads, sums over the lanes and stores overlap
        auto tokens = [&](auto count, int t) {
            constexpr int N = decltype(count)::value;
            float4 f[N];
            float vv[N][C], r[N][C];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                f[j] = s_f[b][t + j];
                const float *const from = vb + (t + j) * vtile;
                if constexpr (C == 4) {
                    const float4 x = *reinterpret_cast<const float4 *>(from);
                    vv[j][0] = x.x; vv[j][1] = x.y; vv[j][2] = x.z; vv[j][3] = x.w;
                } else {
                    const float2 x = *reinterpret_cast<const float2 *>(from);
                    vv[j][0] = x.x; vv[j][1] = x.y;
                }
            }
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (R != 8) again(t + j);
                uint64_t w[C], acc[C];
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    w[c] = pair(vv[j][c] * f[j].y);
                    acc[c] = 0;
                }
#pragma unroll
                for (int i = 0; i < QUADS; ++i) {
                    const ulonglong2 kk =
                        *reinterpret_cast<const ulonglong2 *>(kb + (t + j) * DK + 4 * KG * i);
#pragma unroll
                    for (int c = 0; c < C; ++c) {
                        u[2 * i][c] = fma2(kk.x, w[c], u[2 * i][c]);
                        u[2 * i + 1][c] = fma2(kk.y, w[c], u[2 * i + 1][c]);
                    }
                    if constexpr (!STATE) {
                        const ulonglong2 qq =
                            *reinterpret_cast<const ulonglong2 *>(qb + (t + j) * DK + 4 * KG * i);
#pragma unroll
                        for (int c = 0; c < C; ++c) acc[c] = fma2(qq.x, u[2 * i][c], acc[c]);
#pragma unroll
                        for (int c = 0; c < C; ++c) acc[c] = fma2(qq.y, u[2 * i + 1][c], acc[c]);
                    }
                }
#pragma unroll
                for (int c = 0; c < C; ++c)
                    r[j][c] = __uint_as_float(lo_of(acc[c])) + __uint_as_float(hi_of(acc[c]));
            }
            if constexpr (!STATE) {
                // the sum over the KG lanes; four columns are shared out between them
                int mine = col;                            // this lane's first sum
                if constexpr (C == 4) {
                    const bool odd = kg & 1, up = kg & 2;
                    mine += odd ? 2 : 0;
                    if (KG > 2) mine += up ? 1 : 0;
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const float g0 = odd ? r[j][0] : r[j][2], g1 = odd ? r[j][1] : r[j][3];
                        r[j][0] = (odd ? r[j][2] : r[j][0]) + __shfl_xor_sync(0xffffffffu, g0, 1);
                        r[j][1] = (odd ? r[j][3] : r[j][1]) + __shfl_xor_sync(0xffffffffu, g1, 1);
                        if constexpr (KG > 2) {
                            const float g2 = up ? r[j][0] : r[j][1];
                            r[j][0] = (up ? r[j][1] : r[j][0]) + __shfl_xor_sync(0xffffffffu, g2, 2);
#pragma unroll
                            for (int s = 4; s < KG; s <<= 1)
                                r[j][0] += __shfl_xor_sync(0xffffffffu, r[j][0], s);
                        }
                    }
                } else {
#pragma unroll
                    for (int s = 1; s < KG; s <<= 1)
#pragma unroll
                        for (int j = 0; j < N; ++j)
#pragma unroll
                            for (int c = 0; c < C; ++c)
                                r[j][c] += __shfl_xor_sync(0xffffffffu, r[j][c], s);
                }
                constexpr bool TWO = C == 2 || KG == 2;    // sums a lane stores
                if (kg < (C == 2 ? 1 : 4) && mine < cols) {
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        T *const at = to + j * a.os[1] + (mine - col);
                        const float x0 = r[j][0] * f[j].z, x1 = TWO ? r[j][1] * f[j].z : 0.0f;
                        if (TWO && pair_o) {
                            if constexpr (sizeof(T) == 4)
                                *reinterpret_cast<float2 *>(at) = make_float2(x0, x1);
                            else
                                *reinterpret_cast<__nv_bfloat162 *>(at) = __floats2bfloat162_rn(x0, x1);
                        } else {
                            at[0] = io<T>::from_f(x0);
                            if (TWO && mine + 1 < cols) at[1] = io<T>::from_f(x1);
                        }
                    }
                }
                to += N * a.os[1];
            }
        };
        if constexpr (R == 8) {
            const uint32_t starts = s_again[b];
#pragma unroll 1
            for (int t = 0; t < m;) {
                if (t + 8 <= m && !(starts >> t & 0xfeu)) {
                    again(t);
                    tokens(std::integral_constant<int, 8>{}, t);
                    t += 8;
                } else {
                    again(t);
                    tokens(std::integral_constant<int, 1>{}, t);
                    ++t;
                }
            }
        } else {
            constexpr int UNROLL = KG == 1 ? 2 : 1;        // more spills the wider states
#pragma unroll UNROLL
            for (int t = 0; t < m; ++t) tokens(std::integral_constant<int, 1>{}, t);
        }
    }
    if (STATE && first && lane == 0 && tile == 0) a.seg_g[sp.out * a.heads + h] = span_g;
    if (sp.out >= 0) {
        // the last run's decay: every thread needs log A of the last token
        __shared__ float s_last;
        if (first && lane == 0) s_last = (float)exp(run);
        __syncthreads();
        const float f = s_last;
#pragma unroll
        for (int i = 0; i < 2 * QUADS; ++i)
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int dk = row_of(i) + j;
                    const float x = __uint_as_float(j ? hi_of(u[i][c]) : lo_of(u[i][c]));
                    if (dk < a.dk && col + c < cols)
                        hout[((sp.out * a.heads + h) * a.dk + dk) * a.dv + c0 + col + c] = x * f;
                }
    }
}

template <typename T>
static bool vec16(const void *p, const int64_t (&s)[3], int64_t cols) {
    constexpr int64_t E = 16 / (int64_t)sizeof(T);
    return aligned(p, 16) && s[0] % E == 0 && s[1] % E == 0 && s[2] % E == 0 && cols % E == 0;
}

template <typename T, int KG, int R, int C, bool STATE>
static int launch_recurrent(const Args &a, cudaStream_t st) {
    constexpr int WV = 32 / KG * C;                        // columns of a warp
    const int most = KG == 1 ? 1 : 4;
    const int warps = (int)(ceil_div(a.dv, WV) < most ? ceil_div(a.dv, WV) : most);
    const int vtile = warps * WV;
    const int64_t grid = ceil_div(a.dv, vtile) * a.heads * spans(a);
    MB2_REQUIRE(grid <= 0x7fffffff, MB2_ERR_SHAPE, "decay_attention: too many sequences x heads");
    constexpr int L = stage_tokens<R>();
    const size_t smem = sizeof(float) * 2 * L * ((STATE ? 1 : 2) * KG * R + vtile);
    auto kern = decay_recurrent_kernel<T, KG, R, C, STATE>;
    const bool pairs = a.dv % 2 == 0 && aligned(a.o, 2 * sizeof(T)) && a.os[0] % 2 == 0 &&
                       a.os[1] % 2 == 0 && a.os[2] % 2 == 0;
    // all of the SM's shared memory: the walks resident at once are what hides latency
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
    if (e == cudaSuccess && smem > 48 * 1024)
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return fail(MB2_ERR_CUDA, "decay_attention: %s", cudaGetErrorString(e));
    kern<<<(unsigned)grid, warps * 32 + (R == 8 ? 128 : 0), smem, st>>>(
        a, vtile, vec16<T>(a.q, a.qs, a.dk), vec16<T>(a.k, a.ks, a.dk), vec16<T>(a.v, a.vs, a.dv),
        pairs);
    return check_launch("decay_recurrent_kernel");
}

template <typename T, bool STATE>
static int recurrent_of(const Args &a, cudaStream_t st) {
    if (a.narrow) {
        if (a.dk <= 16) return launch_recurrent<T, 2, 8, 2, STATE>(a, st);
        if (a.dk <= 32) return launch_recurrent<T, 4, 8, 2, STATE>(a, st);
        if (a.dk <= 64) return launch_recurrent<T, 8, 8, 2, STATE>(a, st);
        if (a.dk <= 128) return launch_recurrent<T, 16, 8, 2, STATE>(a, st);
        return launch_recurrent<T, 32, 8, 2, STATE>(a, st);
    }
    if (a.dk <= 16) return launch_recurrent<T, 1, 16, 2, STATE>(a, st);
    if (a.dk <= 24) return launch_recurrent<T, 1, 24, 2, STATE>(a, st);
    if (a.dk <= 32) return launch_recurrent<T, 1, 32, 2, STATE>(a, st);
    if (a.dk <= 64) return launch_recurrent<T, 4, 16, 4, STATE>(a, st);
    if (a.dk <= 128) return launch_recurrent<T, 8, 16, 4, STATE>(a, st);
    return launch_recurrent<T, 16, 16, 4, STATE>(a, st);
}
static int recurrent(const Args &a, bool state_only, cudaStream_t st) {
    if (a.dtype == MB2_F32)
        return state_only ? recurrent_of<float, true>(a, st) : recurrent_of<float, false>(a, st);
    return state_only ? recurrent_of<__nv_bfloat16, true>(a, st)
                      : recurrent_of<__nv_bfloat16, false>(a, st);
}

template <int VEC> struct vecf;
template <> struct vecf<4> { using t = float4; };
template <> struct vecf<1> { using t = float; };

// --------------------------------------------------------------- segments
// slot0[i]: the first slot of packed sequence i (one warp, a running sum)
__global__ void slots_kernel(const Args a, int32_t *slot0) {
    int64_t base = 0;
    for (int64_t i0 = 0; i0 < a.seqs; i0 += 32) {
        const int64_t i = i0 + threadIdx.x;
        int64_t row0 = 0, len = 0, n = 0;
        if (i < a.seqs) {
            bounds(a, i, row0, len);
            n = segments(len, a.seg);
        }
        int64_t sum = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, sum, d);
            if ((int)threadIdx.x >= d) sum += y;
        }
        // (overlapping sequences can ask for more slots than there are)
        const int64_t at = base + sum - n;
        if (i < a.seqs) slot0[i] = (int32_t)(at < a.slots ? at : a.slots);
        base += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (threadIdx.x == 0) slot0[a.seqs] = (int32_t)(base < a.slots ? base : a.slots);
}

// The segments' states, each from 0, become their initial states, element by
// element: S_{j+1} = e^{G_j} S_j + own_j, S_0 = h0.  A sequence's last slot takes
// its initial state without having held one.
template <int VEC>
__global__ void __launch_bounds__(128) seg_states_kernel(const Args a) {
    using V = typename vecf<VEC>::t;
    const int64_t per = a.dk * a.dv;
    const int64_t e = ((int64_t)blockIdx.x * 128 + threadIdx.x) * VEC;
    const int64_t seq = blockIdx.z, h = blockIdx.y;
    if (e >= per) return;
    const int64_t n = a.cu ? a.slot0[seq + 1] - a.slot0[seq] : segments(a.seqlen, a.seg);
    const int64_t first = a.cu ? a.slot0[seq] : seq * n;
    const int64_t step = a.heads * per;
    float *s = a.seg_state + (first * a.heads + h) * per + e;
    const double *g = a.seg_g + first * a.heads + h;
    V run = {};
    if (a.h0) run = *reinterpret_cast<const V *>(a.h0 + (seq * a.heads + h) * per + e);
    // the chain is short; the loads of eight segments run ahead of it
    for (int64_t j0 = 0; j0 < n; j0 += 8) {
        V own[8];
        float dec[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            own[i] = V{};
            dec[i] = 0.0f;
            if (j0 + i + 1 < n) {
                own[i] = *reinterpret_cast<const V *>(s + (j0 + i) * step);
                dec[i] = expf((float)g[(j0 + i) * a.heads]);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (j0 + i < n) {
                *reinterpret_cast<V *>(s + (j0 + i) * step) = run;
                float *r = reinterpret_cast<float *>(&run);
                const float *o = reinterpret_cast<const float *>(&own[i]);
#pragma unroll
                for (int v = 0; v < VEC; ++v) r[v] = fmaf(dec[i], r[v], o[v]);
            }
    }
}

// Tokens per segment, 0 for whole sequences.  A walk takes its steps of `unit`
// tokens one after the other, and `lanes` walks run at a time: with fewer sequences
// x heads x column tiles than that (or an uneven last round of them) segments
// shorten the longest chain, at the price of a first pass that costs `first` of the
// second's time a step, `fill` steps to start each walk, and the states' traffic
// (`join` steps and a tenth for each segment).
// Measured, one sequence of 8192 tokens, 24 heads of 128 x 64 in bf16: 186 us whole,
// 71 in segments (first pass 26, states 3, second pass 40).
static int64_t segment_tokens(const Args &a, int64_t walks, int64_t lanes, int64_t unit,
                              double first, double fill, double join, double &time) {
    time = 0.0;
    if (a.seqs == 0 || a.seqlen == 0) return 0;
    // packed: the lengths are not known here; the longest sequence is taken as one
    // and a half times the mean
    const int64_t units = ceil_div(a.cu ? ceil_div(a.seqlen, a.seqs) : a.seqlen, unit);
    const double even = (double)walks * (double)units / (double)lanes;
    const double whole = !a.cu ? (double)ceil_div(walks, lanes) * (double)units
                               : (even > 1.5 * units ? even : 1.5 * units);
    double best = whole * 0.9;            // segments have to save a tenth
    int64_t seg = 0;
    time = whole;
    for (int64_t n = 2; n <= 256 && n * 2 <= units; ++n) {
        const int64_t per = ceil_div(units, n);
        const double t = (double)ceil_div(walks * n, lanes) * (per + fill) +
                         (double)ceil_div(walks * (n - 1), lanes) * (first * per + fill) +
                         0.1 * n + join;
        if (t < best) {
            best = time = t;
            seg = per * unit;
        }
    }
    return seg;
}

// --------------------------------------------------------- relaid tensors
// The tensor-core kernel wants rows of 16-byte groups (TMA).  bf16 prompts whose
// widths or strides are others are laid out for it first, zeros behind Dk and Dv,
// and o and h_last copied back: two launches and their traffic, where the recurrent
// kernel took (us, both ways)
//   8 x 379 tokens, 12 heads of 87 x 64                   207 -> 18
//   15 x 2560, 6 heads of 64 x 14                         161 -> 67
//   51221 in 23 sequences, 1 head of 89 x 104             286 -> 57
//   40 x 568, 24 heads of 10 x 64                         295 -> 102
struct Relay {
    struct Item {
        const void *src;
        void *dst;
        int64_t s[3];                     // the caller's strides
        uint32_t n[3], rows;              // (batch, token, head); rows of n[2] that the caller has
        uint32_t width, padded;           // of a row: the caller's, ours
        int bytes;                        // an element's
    } item[4];
    int n;
    const int32_t *cu;                    // o: rows outside the sequences stay as they are
    int64_t seqs, seqlen;
};
constexpr int RELAY_THREADS = 256;

// a thread's 16 bytes of our rows: from the caller's (IN) or back (rows lo .. hi - 1, or
// those of any sequence of r where it is given)
template <typename E, bool IN>
__device__ __forceinline__ void relay_rows(const Relay::Item &it, int64_t lo, int64_t hi,
                                           const Relay *r = nullptr) {
    constexpr uint32_t V = 16 / sizeof(E);
    const uint32_t groups = it.padded / V;
    const uint64_t total = (uint64_t)it.n[0] * it.n[1] * it.n[2] * groups;
    for (uint64_t i = (uint64_t)blockIdx.x * RELAY_THREADS + threadIdx.x; i < total;
         i += (uint64_t)gridDim.x * RELAY_THREADS) {
        // 32-bit divisions where the numbers allow them
        const uint64_t row = i >> 32 ? i / groups : (uint32_t)i / groups;
        const uint32_t c = (uint32_t)(i - row * groups) * V;
        const uint64_t bt = row >> 32 ? row / it.n[2] : (uint32_t)row / it.n[2];
        const uint32_t h = (uint32_t)(row - bt * it.n[2]);
        const uint64_t b = bt >> 32 ? bt / it.n[1] : (uint32_t)bt / it.n[1];
        const int64_t t = (int64_t)(bt - b * it.n[1]);
        const int64_t at = (int64_t)b * it.s[0] + t * it.s[1] + (int64_t)h * it.s[2] + c;
        E x[V];
        if (IN) {
            const E *const src = static_cast<const E *>(it.src) + at;
#pragma unroll
            for (uint32_t e = 0; e < V; ++e) {
                x[e] = 0;
                if (h < it.rows && c + e < it.width) x[e] = src[e];
            }
            *reinterpret_cast<uint4 *>(static_cast<E *>(it.dst) + i * V) =
                *reinterpret_cast<const uint4 *>(x);
        } else {
            if (h >= it.rows || t < lo || t >= hi) continue;
            if (r) {
                bool any = false;
                for (int64_t i = 0; i < r->seqs && !any; ++i)
                    any = t >= clamp_row(r->cu[i], r->seqlen) && t < clamp_row(r->cu[i + 1], r->seqlen);
                if (!any) continue;
            }
            *reinterpret_cast<uint4 *>(x) =
                *reinterpret_cast<const uint4 *>(static_cast<const E *>(it.src) + i * V);
            E *const dst = static_cast<E *>(it.dst) + at;
#pragma unroll
            for (uint32_t e = 0; e < V; ++e)
                if (c + e < it.width) dst[e] = x[e];
        }
    }
}

template <bool IN>
__global__ void __launch_bounds__(RELAY_THREADS)
relay_kernel(const __grid_constant__ Relay r) {
    const Relay::Item &it = r.item[blockIdx.y];
    if (it.bytes == 4) {
        relay_rows<uint32_t, IN>(it, 0, INT64_MAX);
        return;
    }
    int64_t lo = 0, hi = INT64_MAX;
    if (!IN && r.cu) {
        // offsets that rise cover all rows between the first and the last; others do not
        bool falls = false;
        for (int64_t i = threadIdx.x; i < r.seqs; i += RELAY_THREADS)
            falls = falls || clamp_row(r.cu[i + 1], r.seqlen) < clamp_row(r.cu[i], r.seqlen);
        if (__syncthreads_or(falls)) {
            relay_rows<uint16_t, IN>(it, lo, hi, &r);
            return;
        }
        lo = clamp_row(r.cu[0], r.seqlen);
        hi = clamp_row(r.cu[r.seqs], r.seqlen);
    }
    relay_rows<uint16_t, IN>(it, lo, hi);
}

static int relay(const Relay &r, bool in, cudaStream_t st) {
    if (r.n == 0) return MB2_OK;
    uint64_t most = 1;
    for (int i = 0; i < r.n; ++i) {
        const Relay::Item &it = r.item[i];
        const uint64_t groups = (uint64_t)it.n[0] * it.n[1] * it.n[2] * (it.padded * it.bytes / 16);
        if (groups > most) most = groups;
    }
    const uint64_t blocks = (most + RELAY_THREADS - 1) / RELAY_THREADS;
    const dim3 grid((unsigned)(blocks < 8192 ? blocks : 8192), (unsigned)r.n);
    if (in) relay_kernel<true><<<grid, RELAY_THREADS, 0, st>>>(r);
    else relay_kernel<false><<<grid, RELAY_THREADS, 0, st>>>(r);
    return check_launch("relay_kernel");
}

static bool tma_rows(const void *p, const int64_t (&s)[3], int64_t batch, int64_t tokens,
                     int64_t heads) {
    const int64_t n[3] = {batch, tokens, heads};
    bool ok = aligned(p, 16);
    for (int i = 0; i < 3; ++i) ok = ok && s[i] % 8 == 0 && (s[i] > 0 || n[i] <= 1);
    return ok;
}

// Points `a` to rows in the workspace (from byte `at` on) where the caller's do not
// suit the tensor cores; what to copy before and after.  Returns the workspace's end.
static size_t relaid(Args &a, uint8_t *ws, size_t at, Relay &in, Relay &out) {
    in.n = out.n = 0;
    in.cu = out.cu = a.cu;
    in.seqs = out.seqs = a.seqs;
    in.seqlen = out.seqlen = a.seqlen;
    const int64_t batch = a.cu ? 1 : a.seqs;
    if (a.recurrent || batch >= (1ll << 31) || a.seqlen >= (1ll << 31)) return at;
    const int64_t dk = round_up(a.dk, 8), dv = round_up(a.dv, 8);
    const int64_t hq = a.heads / a.q_rep, hk = a.heads / a.k_rep, hv = a.heads / a.v_rep;
    auto take = [&](size_t bytes) {
        uint8_t *p = ws + at;
        at += (size_t)round_up((int64_t)bytes, 256);
        return p;
    };
    auto tokens = [&](Relay &r, const void *src, void *dst, int64_t (&s)[3], int64_t heads,
                      int64_t width, int64_t padded) {
        Relay::Item &it = r.item[r.n++];
        it = {src, dst, {s[0], s[1], s[2]}, {(uint32_t)batch, (uint32_t)a.seqlen, (uint32_t)heads},
              (uint32_t)heads, (uint32_t)width, (uint32_t)padded, 2};
        s[0] = a.seqlen * heads * padded;
        s[1] = heads * padded;
        s[2] = padded;
    };
    auto bytes = [&](int64_t heads, int64_t width) {
        return (size_t)(batch * a.seqlen * heads * width) * 2;
    };
    if (dk != a.dk || !tma_rows(a.q, a.qs, batch, a.seqlen, hq)) {
        void *p = take(bytes(hq, dk));
        tokens(in, a.q, p, a.qs, hq, a.dk, dk);
        a.q = p;
    }
    if (dk != a.dk || !tma_rows(a.k, a.ks, batch, a.seqlen, hk)) {
        void *p = take(bytes(hk, dk));
        tokens(in, a.k, p, a.ks, hk, a.dk, dk);
        a.k = p;
    }
    if (dv != a.dv || !tma_rows(a.v, a.vs, batch, a.seqlen, hv)) {
        void *p = take(bytes(hv, dv));
        tokens(in, a.v, p, a.vs, hv, a.dv, dv);
        a.v = p;
    }
    if (dv != a.dv || !tma_rows(a.o, a.os, batch, a.seqlen, a.heads)) {
        void *p = take(bytes(a.heads, dv));
        tokens(out, p, a.o, a.os, a.heads, a.dv, dv);
        a.o = p;
    }
    const bool pad = dk != a.dk || dv != a.dv;
    auto states = [&](Relay &r, const void *src, void *dst) {
        r.item[r.n++] = {src, dst, {a.heads * a.dk * a.dv, a.dk * a.dv, a.dv},
                         {(uint32_t)a.seqs, (uint32_t)a.heads, (uint32_t)dk},
                         (uint32_t)a.dk, (uint32_t)a.dv, (uint32_t)dv, 4};
    };
    const size_t state = (size_t)(a.seqs * a.heads * dk * dv) * 4;
    if (a.h0 && (pad || !aligned(a.h0, 16))) {
        float *p = reinterpret_cast<float *>(take(state));
        states(in, a.h0, p);
        a.h0 = p;
    }
    if (a.h_last && (pad || !aligned(a.h_last, 16))) {
        float *p = reinterpret_cast<float *>(take(state));
        states(out, p, a.h_last);
        a.h_last = p;
    }
    a.dk = dk;
    a.dv = dv;
    return at;
}

// The recurrent kernel's walks: 14 of one warp (up to 24 rows; 12 up to 32) or 12 warps'
// worth of them (up to four each) on an SM at a time; narrow ones 2 (1 above 128 rows):
// what registers and shared memory leave room for.
struct Walks { int64_t n, lanes; };
static Walks walks_of(const Args &a, bool narrow) {
    const int64_t sms = num_sms();
    int64_t cols = a.dk <= 32 ? 64 : a.dk <= 64 ? 128 : a.dk <= 128 ? 64 : 32;
    if (narrow) cols = a.dk <= 16 ? 128 : a.dk <= 32 ? 64 : a.dk <= 64 ? 32 : a.dk <= 128 ? 16 : 8;
    const int64_t warps = ceil_div(a.dv < cols ? a.dv : cols, cols / 4);
    return {a.seqs * a.heads * ceil_div(a.dv, cols),
            narrow         ? (a.dk <= 128 ? 2 : 1) * sms
            : a.dk <= 24   ? 14 * sms
            : a.dk <= 32   ? 12 * sms
                           : 12 / warps * sms};
}

// Short bf16 prompts the recurrent kernel does sooner: a walk of the tensor cores
// takes its 128 tokens whole.  In us, 64 heads of 64 x 64: 1 token 4.1 against 9.8, 16
// tokens 5.7 against 9.4, 32 tokens 7.8 against 9.2; 1024 heads of 16 x 120: 1 token 5.3
// against 71, 64 tokens 30 against 105.
static bool short_prompt(const Args &a) {
    if (a.seqs == 0) return true;
    const double tokens = (double)(a.cu ? ceil_div(a.seqlen, a.seqs) : a.seqlen);
    if (tokens > 128) return false;
    const Walks n = walks_of(a, true), w = walks_of(a, false);
    const double load = (double)w.n / (double)w.lanes, idle = a.dk <= 32 ? 0.27 : 0.36;
    const double recurrent = 3.5 + tokens * (n.n <= n.lanes ? 0.13
                                             : load <= 1.0 ? idle + (0.6 - idle) * load
                                                           : 0.6 * load);
    return recurrent < 4.5 + 4.0 * (double)ceil_div(a.seqs * a.heads * ceil_div(a.dv, 64), num_sms());
}

struct Plan { size_t slot0, g, state, bytes; };
// how a call runs, in a workspace at ws: sets a.seg and a.slots, and points a to the
// relaid tensors; the parts of the workspace
static Plan plan(Args &a, uint8_t *ws, Relay &in, Relay &out) {
    a.recurrent = a.dtype != MB2_BF16 || a.dk > 128 || short_prompt(a);
    // the workspace's first bytes stay empty: a tensor at a null workspace (only its
    // size is asked for) is none
    const size_t begin = relaid(a, ws, 256, in, out);
    // tensor cores: one walk of 64 columns an SM, 128 tokens a step; recurrent: compared
    // by 32 tokens, which a narrow walk takes in 4.2 us, others in 2.3 times that (above
    // 64 rows 1.6: in segments, 2048 tokens, 8 heads of 128 x 128, 136 us narrow, 103
    // else; above 128 rows 1.8, 3 up to 8 columns, whose wide walk is a single warp: 600
    // tokens, 296 heads of 200 x 8, 171 us narrow, 297 else; 500 tokens, 60 heads of 256 x
    // 32, 144 and 107).  Narrow ones lose once they share an SM by more than two (192 tokens of
    // fp32, heads of 64 x 64: 8 heads 25 us, others 66; 128 heads 35 and 67; 512 heads 126
    // and 87).
    double time, narrow_time;
    if (chunked_fits(a)) {
        a.seg = segment_tokens(a, a.seqs * a.heads * ceil_div(a.dv, 64), num_sms(), 128, 0.65, 2.2,
                               4.0, time);
    } else {
        const Walks w = walks_of(a, false), n = walks_of(a, true);
        const int64_t wide = segment_tokens(a, w.n, w.lanes, 32, 0.6, 2.2, 4.0, time);
        const int64_t narrow = segment_tokens(a, n.n, n.lanes, 32, 0.6, 0.9, 1.3, narrow_time);
        const double wider = a.dk <= 64 ? 2.3 : a.dk <= 128 ? 1.6 : a.dv <= 8 ? 3.0 : 1.8;
        a.narrow = n.n <= 2 * num_sms() && narrow_time <= wider * time;
        a.seg = a.narrow ? narrow : wide;
    }
    a.slots = 0;
    Plan p = {};
    p.bytes = in.n + out.n ? begin : 0;
    if (a.seg == 0) return p;
    a.slots = a.cu ? a.seqs + a.seqlen / a.seg : a.seqs * segments(a.seqlen, a.seg);
    p.slot0 = begin;
    p.g = begin + (size_t)round_up((a.seqs + 1) * 4, 256);
    p.state = p.g + (size_t)round_up(a.slots * a.heads * 8, 256);
    p.bytes = p.state + (size_t)(a.slots * a.heads * a.dk * a.dv) * 4;
    return p;
}

// rows of o before the first and behind the last packed sequence (a new o)
template <typename T>
__global__ void zero_tail_kernel(const Args a) {
    const int64_t end = clamp_row(a.cu[a.seqs], a.seqlen);
    int64_t begin = clamp_row(a.cu[0], a.seqlen);
    if (begin > end) begin = end;
    const int64_t per = a.heads * a.dv;
    T *o = static_cast<T *>(a.o);
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
         i < (begin + a.seqlen - end) * per; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t at = i / per, t = at < begin ? at : end - begin + at, r = i % per;
        o[t * a.os[1] + (r / a.dv) * a.os[2] + r % a.dv] = io<T>::from_f(0.0f);
    }
}

// -------------------------------------------------------------- one token
// HBM-bound: the state is read and written once (8 Dk Dv bytes per head), all
// else is small.  A CTA takes one (sequence, head, column tile): `lanes`
// threads per state row of VEC columns each, the CTA's row slots stepping
// through the Dk rows with ROWS rows' loads in flight per thread.  Partial
// sums of o over the row slots meet in shared memory, added in a fixed order.
template <typename T, int VEC, int STEP_THREADS>
__global__ void __launch_bounds__(STEP_THREADS)
decay_step_kernel(const Args a, float *__restrict__ state, int lanes) {
    constexpr int ROWS = 8;
    using V = typename vecf<VEC>::t;
    __shared__ float part[STEP_THREADS * VEC];
    __shared__ float sq[256], sk[256];
    const int ctile = lanes * VEC;
    const int tiles = (int)ceil_div(a.dv, ctile);
    int64_t id = blockIdx.x;
    const int tile = (int)(id % tiles);
    id /= tiles;
    const int h = (int)(id % a.heads);
    const int64_t b = id / a.heads;
    const int lane = threadIdx.x % lanes, slot = threadIdx.x / lanes;
    const int slots = STEP_THREADS / lanes;
    const int c = tile * ctile + lane * VEC;
    const bool live = slot < slots && c < a.dv;

    float *const s = state + ((b * a.heads + h) * a.dk) * a.dv + c;
    const T *q = static_cast<const T *>(a.q) + b * a.qs[0] + (h / a.q_rep) * a.qs[2];
    const T *k = static_cast<const T *>(a.k) + b * a.ks[0] + (h / a.k_rep) * a.ks[2];
    const T *v = static_cast<const T *>(a.v) + b * a.vs[0] + (h / a.v_rep) * a.vs[2];
    // the first rows' loads are issued before q and k are waited for
    V x[ROWS];
    const int dk = (int)a.dk;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = slot + i * slots;
        if (live && r < dk) x[i] = *reinterpret_cast<const V *>(s + (int64_t)r * a.dv);
    }
    for (int i = threadIdx.x; i < dk; i += STEP_THREADS) {
        sq[i] = io<T>::to_f(q[i]) * a.scale;
        sk[i] = io<T>::to_f(k[i]);
    }
    const float dec = expf(a.g[b * a.gs[0] + h * a.gs[2]]);
    float vv[VEC], acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        vv[j] = live ? io<T>::to_f(v[c + j]) : 0.0f;
        acc[j] = 0.0f;
    }
    __syncthreads();
    if (live) {
        for (int r0 = slot; r0 < dk; r0 += ROWS * slots) {
            if (r0 != slot) {
#pragma unroll
                for (int i = 0; i < ROWS; ++i) {
                    const int r = r0 + i * slots;
                    if (r < dk) x[i] = *reinterpret_cast<const V *>(s + (int64_t)r * a.dv);
                }
            }
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                const int r = r0 + i * slots;
                if (r < dk) {
                    float *e = reinterpret_cast<float *>(&x[i]);
                    const float kr = sk[r], qr = sq[r];
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        e[j] = fmaf(kr, vv[j], dec * e[j]);
                        acc[j] = fmaf(qr, e[j], acc[j]);
                    }
                    *reinterpret_cast<V *>(s + (int64_t)r * a.dv) = x[i];
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) part[threadIdx.x * VEC + j] = acc[j];
    __syncthreads();
    T *o = static_cast<T *>(a.o) + b * a.os[0] + h * a.os[2];
    for (int i = threadIdx.x; i < ctile; i += STEP_THREADS) {
        const int cc = tile * ctile + i;
        if (cc < a.dv) {
            float sum = 0.0f;
            for (int j = 0; j < slots; ++j) sum += part[j * ctile + i];
            o[cc] = io<T>::from_f(sum);
        }
    }
}

template <typename T>
static int step(const Args &a, float *state, cudaStream_t st) {
    const bool vec = a.dv % 4 == 0 && aligned(state, 16);
    const int per = vec ? 4 : 1;
    int lanes = (int)(ceil_div(a.dv, per) < 64 ? ceil_div(a.dv, per) : 64);
    const int64_t grid = ceil_div(a.dv, lanes * per) * a.heads * a.seqs;
    MB2_REQUIRE(grid <= 0x7fffffff, MB2_ERR_SHAPE, "decay_attention_step: batch x heads too large");
    // about 12 rows of 16 bytes a thread, or 64 of 4: small states want small CTAs, so that
    // more of them hide one another's start (us; 64, 128, 256 threads):
    //   334 x 12 heads of 24 x 64       8.7   13.2   22.4
    //   800 x 8 of 128 x 40            45.7   44.5   53.3
    //   512 x 24 of 128 x 64            127    122    121
    //   500 x 12 of 18 x 63            17.5   23.0   32.7
    //   561 x 24 of 115 x 46            138    134    145
    const int64_t need = a.dk * lanes / (vec ? 12 : 64);
    const int threads = need <= 64 ? 64 : need <= 128 ? 128 : 256;
    auto kern = vec ? threads == 64    ? decay_step_kernel<T, 4, 64>
                      : threads == 128 ? decay_step_kernel<T, 4, 128>
                                       : decay_step_kernel<T, 4, 256>
                    : threads == 64    ? decay_step_kernel<T, 1, 64>
                      : threads == 128 ? decay_step_kernel<T, 1, 128>
                                       : decay_step_kernel<T, 1, 256>;
    kern<<<(unsigned)grid, threads, 0, st>>>(a, state, lanes);
    return check_launch("decay_step_kernel");
}

int num_sms() {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
        cudaGetLastError();
        return 148;
    }
    return sms;
}

static int to_args(const mb2_decay_attn *d, bool one, Args &a) {
    const char *what = one ? "decay_attention_step" : "decay_attention";
    MB2_REQUIRE(d, MB2_ERR_ARG, "%s: null descriptor", what);
    MB2_REQUIRE(d->dtype == MB2_F32 || d->dtype == MB2_BF16, MB2_ERR_ARG, "%s: bad dtype", what);
    MB2_REQUIRE(d->batch >= 0 && d->seqlen >= 0 && d->n_seqs >= 0, MB2_ERR_SHAPE,
                "%s: negative size", what);
    MB2_REQUIRE(d->heads > 0 && d->dk > 0 && d->dv > 0, MB2_ERR_SHAPE,
                "%s: heads, dk and dv must be positive", what);
    MB2_REQUIRE(d->heads <= (1 << 20) && d->dv <= (1 << 20), MB2_ERR_SHAPE,
                "%s: heads or dv above 2^20", what);
    MB2_REQUIRE(d->dk <= 256, MB2_ERR_SHAPE, "%s: dk %lld > 256 not supported", what,
                (long long)d->dk);
    MB2_REQUIRE(d->q_heads > 0 && d->k_heads > 0 && d->v_heads > 0 &&
                    d->heads % d->q_heads == 0 && d->heads % d->k_heads == 0 &&
                    d->heads % d->v_heads == 0,
                MB2_ERR_SHAPE, "%s: the heads of q, k and v must divide the %lld decays", what,
                (long long)d->heads);
    MB2_REQUIRE(!d->cu_seqlens || (!one && d->batch == 1), MB2_ERR_SHAPE,
                "%s: packed sequences need batch 1", what);
    a.dtype = d->dtype;
    a.seqs = d->cu_seqlens ? d->n_seqs : d->batch;
    a.seqlen = d->seqlen;
    a.heads = d->heads;
    a.dk = d->dk;
    a.dv = d->dv;
    a.q_rep = (int)(d->heads / d->q_heads);
    a.k_rep = (int)(d->heads / d->k_heads);
    a.v_rep = (int)(d->heads / d->v_heads);
    a.q = d->q; a.k = d->k; a.v = d->v; a.g = d->g; a.o = d->o;
    for (int i = 0; i < 3; ++i) {
        a.qs[i] = d->q_stride[i];
        a.ks[i] = d->k_stride[i];
        a.vs[i] = d->v_stride[i];
        a.gs[i] = d->g_stride[i];
        a.os[i] = d->o_stride[i];
    }
    a.h0 = d->h0;
    a.h_last = d->h_last;
    a.cu = d->cu_seqlens;
    a.scale = d->scale;
    a.narrow = a.recurrent = 0;
    a.seg = a.slots = 0;
    a.slot0 = nullptr;
    a.seg_state = nullptr;
    a.seg_g = nullptr;
    return MB2_OK;
}

}  // namespace decay
}  // namespace mb2

using namespace mb2;

extern "C" size_t mb2_decay_attention_workspace_bytes(const mb2_decay_attn *d) {
    decay::Args a;
    decay::Relay in, out;
    return decay::to_args(d, false, a) == MB2_OK ? decay::plan(a, nullptr, in, out).bytes : 0;
}

extern "C" int mb2_decay_attention(const mb2_decay_attn *d, void *workspace, size_t workspace_bytes,
                                   mb2_stream_t stream) {
    decay::Args a;
    MB2_TRY(decay::to_args(d, false, a));
    if (a.seqs == 0 && !(a.cu && d->zero_tail)) return MB2_OK;
    MB2_REQUIRE((a.q && a.k && a.v && a.g && a.o) || a.seqlen == 0, MB2_ERR_ARG,
                "decay_attention: null pointer");
    const decay::Args given = a;
    decay::Relay in, out;
    const decay::Plan p = decay::plan(a, static_cast<uint8_t *>(workspace), in, out);
    MB2_REQUIRE(workspace_bytes >= p.bytes && (workspace || p.bytes == 0), MB2_ERR_WORKSPACE,
                "decay_attention: workspace of %llu bytes, %llu needed",
                (unsigned long long)workspace_bytes, (unsigned long long)p.bytes);
    MB2_REQUIRE(p.bytes == 0 || aligned(workspace, 256), MB2_ERR_ALIGN,
                "decay_attention: misaligned workspace");
    cudaStream_t st = (cudaStream_t)stream;
    if (a.cu && d->zero_tail && a.seqlen > 0) {
        if (a.dtype == MB2_F32)
            decay::zero_tail_kernel<float><<<64, 256, 0, st>>>(given);
        else
            decay::zero_tail_kernel<__nv_bfloat16><<<64, 256, 0, st>>>(given);
        MB2_TRY(check_launch("zero_tail_kernel"));
    }
    if (a.seqs == 0) return MB2_OK;
    MB2_TRY(decay::relay(in, true, st));
    bool used = false;
    if (a.seg) {
        uint8_t *ws = static_cast<uint8_t *>(workspace);
        int32_t *slot0 = reinterpret_cast<int32_t *>(ws + p.slot0);
        a.slot0 = slot0;
        a.seg_g = reinterpret_cast<double *>(ws + p.g);
        a.seg_state = reinterpret_cast<float *>(ws + p.state);
        MB2_REQUIRE(a.seqs < 65536 && a.heads < 65536, MB2_ERR_SHAPE,
                    "decay_attention: too many sequences or heads");
        if (a.cu) {
            decay::slots_kernel<<<1, 32, 0, st>>>(a, slot0);
            MB2_TRY(check_launch("slots_kernel"));
        }
        MB2_TRY(decay::chunked(a, true, st, &used));
        if (!used) MB2_TRY(decay::recurrent(a, true, st));
        const bool vec = a.dk * a.dv % 4 == 0 && (!a.h0 || aligned(a.h0, 16));
        const dim3 grid((unsigned)ceil_div(a.dk * a.dv, (int64_t)(vec ? 512 : 128)),
                        (unsigned)a.heads, (unsigned)a.seqs);
        if (vec) decay::seg_states_kernel<4><<<grid, 128, 0, st>>>(a);
        else decay::seg_states_kernel<1><<<grid, 128, 0, st>>>(a);
        MB2_TRY(check_launch("seg_states_kernel"));
    }
    MB2_TRY(decay::chunked(a, false, st, &used));
    if (!used) MB2_TRY(decay::recurrent(a, false, st));
    return decay::relay(out, false, st);
}

extern "C" int mb2_decay_attention_step(const mb2_decay_attn *d, float *state, mb2_stream_t stream) {
    decay::Args a;
    MB2_TRY(decay::to_args(d, true, a));
    if (a.seqs == 0) return MB2_OK;
    MB2_REQUIRE(a.q && a.k && a.v && a.g && a.o && state, MB2_ERR_ARG,
                "decay_attention_step: null pointer");
    return a.dtype == MB2_F32 ? decay::step<float>(a, state, (cudaStream_t)stream)
                              : decay::step<__nv_bfloat16>(a, state, (cudaStream_t)stream);
}
