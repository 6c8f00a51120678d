// Decay attention over prompts on the tensor cores (bf16): chunks of 128 tokens,
// one CTA walking the chunks of a (sequence, head, 64 columns of v) with the
// state S (Dk x 64) in fp32 registers.  Within a chunk, with G_i the sum of the
// log decays up to token i and S0 the state before it,
//   P_ij = e^{G_i - G_j} (q_i . k_j)  for j <= i, else 0
//   o_i  = scale (sum_j P_ij v_j + e^{G_i} q_i^T S0)
//   S    = e^{G_C} S0 + sum_j k_j (e^{G_C - G_j} v_j)^T
// so four products: Q K^T (128 x 128 x Dk), P V (128 x 64 x 128), Q S0
// (128 x 64 x Dk) and K^T V~ (Dk x 64 x 128), V~ the decayed rows of V.
//
// Decays.  All exponents are sums of g over tokens between j and i: per 32-token
// block b, colf_j = e^{(block's total) - (sum up to j)}, so off-diagonal blocks
// of P take a row and a column factor (both <= 1 for g <= 0) and only the
// diagonal 32 x 32 blocks an exponential per element.  Sums are 64-bit prefix
// scans, so strong decays earlier in a chunk cost later differences nothing; g
// below -256 counts as -256, whose e^g is below every fp32 product's reach.
//
// Roundings to bf16: P and S0 as MMA operands (the products of a flash-attention
// style kernel; outputs are bf16 anyway).  V~ is held as three bf16 parts
// (24 bits), multiplied side by side as one N = 192 MMA, because the state is an
// fp32 output and lives for many chunks.
//
// Causality with infinities and NaN: a masked P_ij is 0, but 0 * inf = NaN, so a
// row whose P V comes out non-finite is computed again from its own tokens alone.
//
// Roles (16 warps): 0 TMA loads, 1 MMA issue, 4-7 decays, V~ and the state,
// 8-15 P and the output rows.  Every mbarrier completes once per chunk (twice
// staged ones once per two), so its phase follows from the chunk count.  All
// waits are bounded; a wait that expires sets the device status.
#include <cuda.h>
#include <cudaTypedefs.h>

#include "decay.cuh"
#include "tc_prims.cuh"

namespace mb2 {
namespace decay {

using namespace tc;

constexpr int C = 128;                       // tokens per chunk
constexpr int DV = 64;                       // columns of v per CTA
constexpr int THREADS = 512;
constexpr uint32_t SUB = 128 * 128;          // one 128-row x 128-byte operand tile
// shared memory (bytes from a 1024-aligned base)
constexpr uint32_t OFF_Q = 0;                            // [2][2 SUB]
constexpr uint32_t OFF_K = OFF_Q + 4 * SUB;              // [2][2 SUB]
constexpr uint32_t OFF_V = OFF_K + 4 * SUB;              // [2][SUB]
constexpr uint32_t OFF_VT = OFF_V + 2 * SUB;             // [3][SUB]
constexpr uint32_t OFF_H = OFF_VT + 3 * SUB;             // [SUB]
constexpr uint32_t OFF_COLF = OFF_H + SUB;               // float [2][128]
constexpr uint32_t OFF_TOT = OFF_COLF + 2 * C * 4;       // double [2][4]
constexpr uint32_t OFF_BARS = OFF_TOT + 2 * 4 * 8;
constexpr int NBARS = 6 + 6 + 11;
constexpr uint32_t OFF_TMEM = OFF_BARS + NBARS * 8;
constexpr uint32_t SMEM_BYTES = OFF_TMEM + 16;
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory");
// TMEM columns
constexpr uint32_t T_S = 0, T_P = 128, T_PV = 192, T_QH = 256, T_D = 320;

// UMMA descriptor of an MN-major operand, 128-byte swizzle: rows are the
// contraction index (128 bytes of 64 MN elements each), 8-row groups 1024 B
// apart, further 64-element MN atoms SUB apart.
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(SUB >> 4) << 16) |
           ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// D fp32, A and B bf16, M = 128
constexpr uint32_t idesc(uint32_t n, bool a_mn, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) |
           ((n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id,
                                       uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(accum));
}
__device__ __forceinline__ void mma_ts_bf16(uint32_t d, uint32_t a, uint64_t b, uint32_t id,
                                            uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(id), "r"(accum));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]),
          "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
          "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// generic-proxy writes to shared memory become visible to MMA and TMA
__device__ __forceinline__ void fence_async_smem() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, uint32_t bar,
                                            int32_t x, int32_t head, int32_t tok, int32_t b) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(head), "r"(tok),
          "r"(b)
        : "memory");
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float bf_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// e^x of a 64-bit sum, to fp32 precision
__device__ __forceinline__ float exp_of(double x) {
    const float hi = (float)x;
    const float e = expf(hi);
    const float lo = (float)(x - (double)hi);
    return e == 0.0f || hi != hi ? e : fmaf(e, lo, e);
}

struct Item {
    int tile, h;
    int64_t seq, row0, len;
};
__device__ __forceinline__ Item item_of(const Args &a, int tiles, int64_t id) {
    Item it;
    it.tile = (int)(id % tiles);
    id /= tiles;
    it.h = (int)(id % a.heads);
    it.seq = id / a.heads;
    bounds(a, it.seq, it.row0, it.len);
    return it;
}
// g of token t of an item's chunk (0 behind its end); below -256 e^g is 0 for
// every fp32 product, and a finite sum keeps later differences
__device__ __forceinline__ float load_g(const Args &a, const Item &it, int64_t t) {
    if (t >= it.len) return 0.0f;
    const int64_t bq = a.cu ? 0 : it.seq;
    const float g = a.g[bq * a.gs[0] + (it.row0 + t) * a.gs[1] + it.h * a.gs[2]];
    return g < -256.0f ? -256.0f : g;
}
__device__ __forceinline__ double scan32(float g) {
    double x = g;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, x, s);
        if ((int)(threadIdx.x & 31) >= s) x += y;
    }
    return x;
}

// a bounded wait of a whole warp; every lane gets the same answer
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, int where) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, where));
}

// sum_j P_ij v_j of row t over its own tokens j <= t of the chunk, from global
// memory: for rows that met an infinity or a NaN, perhaps in a masked token
__device__ __forceinline__ void masked_row(const Args &a, const Item &it, int64_t t0, int64_t t,
                                           int col, float (&y)[32]) {
    const int64_t bq = a.cu ? 0 : it.seq;
    const __nv_bfloat16 *q = static_cast<const __nv_bfloat16 *>(a.q) + bq * a.qs[0] +
                             (it.row0 + t) * a.qs[1] + (it.h / a.q_rep) * a.qs[2];
#pragma unroll
    for (int i = 0; i < 32; ++i) y[i] = 0.0f;
    double sum = 0.0;
    for (int64_t j = t; j >= t0; --j) {
        const __nv_bfloat16 *k = static_cast<const __nv_bfloat16 *>(a.k) + bq * a.ks[0] +
                                 (it.row0 + j) * a.ks[1] + (it.h / a.k_rep) * a.ks[2];
        const __nv_bfloat16 *v = static_cast<const __nv_bfloat16 *>(a.v) + bq * a.vs[0] +
                                 (it.row0 + j) * a.vs[1] + (it.h / a.v_rep) * a.vs[2] + col;
        float d = 0.0f;
        for (int e = 0; e < (int)a.dk; ++e)
            d = fmaf(__bfloat162float(q[e]), __bfloat162float(k[e]), d);
        const float p = io<__nv_bfloat16>::round(d * __expf((float)sum));
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (col + i < a.dv) y[i] = fmaf(p, __bfloat162float(v[i]), y[i]);
        sum += load_g(a, it, j);
    }
}

__global__ void __launch_bounds__(THREADS, 1)
decay_chunk_kernel(const __grid_constant__ CUtensorMap map_q,
                   const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, const __grid_constant__ Args a,
                   int tiles, int64_t items) {
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t base = smem_u32(smem);
    float *const colf = reinterpret_cast<float *>(smem + OFF_COLF);
    double *const tot = reinterpret_cast<double *>(smem + OFF_TOT);
    uint32_t *const tmem_slot = reinterpret_cast<uint32_t *>(smem + OFF_TMEM);
    auto bar = [&](int i) { return base + OFF_BARS + 8u * i; };
    auto full_q = [&](int s) { return bar(s); };
    auto full_k = [&](int s) { return bar(2 + s); };
    auto full_v = [&](int s) { return bar(4 + s); };
    auto empty_q = [&](int s) { return bar(6 + s); };
    auto empty_k = [&](int s) { return bar(8 + s); };
    auto empty_v = [&](int s) { return bar(10 + s); };
    const uint32_t s_full = bar(12);    // Q K^T in TMEM
    const uint32_t vt_full = bar(13);   // V~ and the decays of a chunk in shared memory
    const uint32_t d_full = bar(14);    // K^T V~ in TMEM
    const uint32_t d_free = bar(15);    // ... read
    const uint32_t h_full = bar(16);    // S0 (bf16) in shared memory
    const uint32_t h_free = bar(17);    // ... read
    const uint32_t p_full = bar(18);    // P in TMEM, S read
    const uint32_t o_full = bar(19);    // P V and Q S0 in TMEM
    const uint32_t o_free = bar(20);    // ... read
    const uint32_t t_full = bar(21);    // the four blocks' decay totals in shared memory
    const uint32_t drain = bar(22);     // every MMA complete (once, at the end)

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool wide = a.dk > 64;                         // two 64-column operand tiles
    const int ks = (int)ceil_div(a.dk, 16);              // MMA steps over Dk
    if (threadIdx.x == 0) {
        for (int i = 0; i < 12; ++i) mbar_init(bar(i), 1);
        mbar_init(s_full, 1);
        mbar_init(vt_full, 128);
        mbar_init(d_full, 1);
        mbar_init(d_free, 128);
        mbar_init(h_full, 128);
        mbar_init(h_free, 1);
        mbar_init(p_full, 256);
        mbar_init(o_full, 1);
        mbar_init(o_free, 256);
        mbar_init(t_full, 128);
        mbar_init(drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(base + OFF_TMEM), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        // -------------------------------------------------------- TMA loads
        if (lane == 0) {
            uint32_t c = 0;
            bool ok = true;
            for (int64_t id = blockIdx.x; id < items && ok; id += gridDim.x) {
                const Item it = item_of(a, tiles, id);
                const int bq = a.cu ? 0 : (int)it.seq;
                for (int64_t t0 = 0; t0 < it.len; t0 += C, ++c) {
                    const int s = c & 1;
                    const uint32_t ph = ((c >> 1) & 1) ^ 1;
                    const int tok = (int)(it.row0 + t0);
                    const uint32_t qk = wide ? 2 * SUB : SUB;
                    const uint32_t dk_ = base + OFF_K + s * 2 * SUB, dq = base + OFF_Q + s * 2 * SUB;
                    if (!(ok = mbar_wait(empty_k(s), ph, 0x401))) break;
                    mbar_expect_tx(full_k(s), qk);
                    tma_load_4d(dk_, &map_k, full_k(s), 0, it.h / a.k_rep, tok, bq);
                    if (wide) tma_load_4d(dk_ + SUB, &map_k, full_k(s), 64, it.h / a.k_rep, tok, bq);
                    if (!(ok = mbar_wait(empty_q(s), ph, 0x402))) break;
                    mbar_expect_tx(full_q(s), qk);
                    tma_load_4d(dq, &map_q, full_q(s), 0, it.h / a.q_rep, tok, bq);
                    if (wide) tma_load_4d(dq + SUB, &map_q, full_q(s), 64, it.h / a.q_rep, tok, bq);
                    if (!(ok = mbar_wait(empty_v(s), ph, 0x403))) break;
                    mbar_expect_tx(full_v(s), SUB);
                    tma_load_4d(base + OFF_V + s * SUB, &map_v, full_v(s), it.tile * DV,
                                it.h / a.v_rep, tok, bq);
                }
            }
            // no load is in flight when the CTA ends (its consumers may have given up)
            for (uint32_t n = c > 2 ? c - 2 : 0; n < c; ++n) {
                mbar_wait(full_k(n & 1), (n >> 1) & 1, 0x404);
                mbar_wait(full_q(n & 1), (n >> 1) & 1, 0x404);
                mbar_wait(full_v(n & 1), (n >> 1) & 1, 0x404);
            }
        }
    } else if (warp == 1) {
        // -------------------------------------------------------- MMA issue
        if (lane == 0) {
            uint32_t c = 0;
            bool ok = true;
            for (int64_t id = blockIdx.x; id < items && ok; id += gridDim.x) {
                const Item it = item_of(a, tiles, id);
                for (int64_t t0 = 0; t0 < it.len && ok; t0 += C, ++c) {
                    const int s = c & 1;
                    const uint32_t ph2 = (c >> 1) & 1, ph = c & 1, prev = ph ^ 1;
                    const uint32_t q = base + OFF_Q + s * 2 * SUB, k = base + OFF_K + s * 2 * SUB;
                    const uint32_t v = base + OFF_V + s * SUB;
                    // S = Q K^T (P of the chunk before read the last S before p_full)
                    if (!(ok = mbar_wait(full_k(s), ph2, 0x411) && mbar_wait(full_q(s), ph2, 0x412)))
                        break;
                    fence_after();
                    for (int i = 0; i < ks; ++i) {
                        const uint32_t off = (i >> 2) * SUB + (i & 3) * 32;
                        mma_ss(tmem + T_S, smem_desc(q + off), smem_desc(k + off),
                               idesc(128, false, false), i > 0);
                    }
                    mma_commit(s_full);
                    // K^T V~, three parts side by side
                    if (!(ok = mbar_wait(vt_full, ph, 0x413) && mbar_wait(d_free, prev, 0x414))) break;
                    fence_after();
#pragma unroll
                    for (int i = 0; i < C / 16; ++i)
                        mma_ss(tmem + T_D, smem_desc_mn(k + i * 2048),
                               smem_desc_mn(base + OFF_VT + i * 2048), idesc(192, true, true), i > 0);
                    mma_commit(d_full);
                    mma_commit(empty_k(s));
                    // Q S0
                    if (!(ok = mbar_wait(h_full, ph, 0x415) && mbar_wait(o_free, prev, 0x416))) break;
                    fence_after();
                    for (int i = 0; i < ks; ++i)
                        mma_ss(tmem + T_QH, smem_desc(q + (i >> 2) * SUB + (i & 3) * 32),
                               smem_desc_mn(base + OFF_H + i * 2048), idesc(64, false, true), i > 0);
                    mma_commit(h_free);
                    mma_commit(empty_q(s));
                    // P V
                    if (!(ok = mbar_wait(p_full, ph, 0x417))) break;
                    fence_after();
#pragma unroll
                    for (int i = 0; i < C / 16; ++i)
                        mma_ts_bf16(tmem + T_PV, tmem + T_P + i * 8, smem_desc_mn(v + i * 2048),
                                    idesc(64, false, true), i > 0);
                    mma_commit(o_full);
                    mma_commit(empty_v(s));
                }
            }
            mma_commit(drain);                           // before TMEM is given back
            mbar_wait(drain, 0, 0x418);
        }
        __syncwarp();
    } else if (warp >= 4 && warp < 8) {
        // ------------------------------------------- decays, V~ and the state
        const int w = warp & 3, r = 32 * w + lane;        // token of a chunk, row of the state
        const uint32_t quarter = tmem + ((uint32_t)(32 * w) << 16);
        uint32_t c = 0;
        bool ok = true;
        for (int64_t id = blockIdx.x; id < items && ok; id += gridDim.x) {
            const Item it = item_of(a, tiles, id);
            const int c0 = it.tile * DV;
            const int64_t at = ((it.seq * a.heads + it.h) * a.dk + r) * a.dv + c0;
            float h[DV];
            if (a.h0 && r < a.dk) {
#pragma unroll
                for (int i = 0; i < DV; i += 4) {
                    float4 x = make_float4(0, 0, 0, 0);
                    if (c0 + i < a.dv) x = *reinterpret_cast<const float4 *>(a.h0 + at + i);
                    h[i] = x.x; h[i + 1] = x.y; h[i + 2] = x.z; h[i + 3] = x.w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < DV; ++i) h[i] = 0.0f;
            }
            float gn = load_g(a, it, r);
            for (int64_t t0 = 0; t0 < it.len; t0 += C, ++c) {
                const int s = c & 1;
                const uint32_t ph = c & 1, prev = ph ^ 1;
                const int m = (int)(it.len - t0 < C ? it.len - t0 : C);
                const double gl = scan32(gn);
                gn = load_g(a, it, t0 + C + r);
                const double bt = __shfl_sync(0xffffffffu, gl, 31);
                const float cf = exp_of(bt - gl);
                colf[s * C + r] = cf;
                if (lane == 0) tot[s * 4 + w] = bt;
                mbar_arrive(t_full);
                if (!(ok = wait_warp(t_full, ph, 0x420))) break;
                double later = 0.0, all = 0.0;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const double x = tot[s * 4 + b];
                    all += x;
                    if (b > w) later += x;
                }
                const float dec = exp_of(all);            // e^{G_C}
                const float wj = cf * exp_of(later);      // e^{G_C - G_j}
                if (!(ok = wait_warp(full_v(s), (c >> 1) & 1, 0x421))) break;
                uint8_t *const vrow = smem + OFF_V + s * SUB + r * 128;
                uint8_t *const trow = smem + OFF_VT + r * 128;
                if (m < C && !(ok = wait_warp(full_k(s), (c >> 1) & 1, 0x422))) break;
                if (r < m) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t off = (uint32_t)((i ^ (r & 7)) << 4);
                        const uint4 x4 = *reinterpret_cast<const uint4 *>(vrow + off);
                        const uint32_t *x = reinterpret_cast<const uint32_t *>(&x4);
                        uint32_t p0[4], p1[4], p2[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float lo = bf_lo(x[e]) * wj, hi = bf_hi(x[e]) * wj;
                            p0[e] = pack_bf16(lo, hi);
                            lo -= bf_lo(p0[e]);
                            hi -= bf_hi(p0[e]);
                            p1[e] = pack_bf16(lo, hi);
                            p2[e] = pack_bf16(lo - bf_lo(p1[e]), hi - bf_hi(p1[e]));
                        }
                        *reinterpret_cast<uint4 *>(trow + off) = make_uint4(p0[0], p0[1], p0[2], p0[3]);
                        *reinterpret_cast<uint4 *>(trow + SUB + off) = make_uint4(p1[0], p1[1], p1[2], p1[3]);
                        *reinterpret_cast<uint4 *>(trow + 2 * SUB + off) = make_uint4(p2[0], p2[1], p2[2], p2[3]);
                    }
                } else {
                    // rows behind the sequence (another one's, or nothing): zero in
                    // V, V~ and K, whose values a product would otherwise meet
                    const uint4 z = make_uint4(0, 0, 0, 0);
                    uint8_t *const krow = smem + OFF_K + s * 2 * SUB + r * 128;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        *reinterpret_cast<uint4 *>(vrow + i * 16) = z;
                        *reinterpret_cast<uint4 *>(trow + i * 16) = z;
                        *reinterpret_cast<uint4 *>(trow + SUB + i * 16) = z;
                        *reinterpret_cast<uint4 *>(trow + 2 * SUB + i * 16) = z;
                        *reinterpret_cast<uint4 *>(krow + i * 16) = z;
                        *reinterpret_cast<uint4 *>(krow + SUB + i * 16) = z;
                    }
                }
                fence_async_smem();
                mbar_arrive(vt_full);
                // S0 of this chunk for Q S0
                if (!(ok = wait_warp(h_free, prev, 0x423))) break;
                uint8_t *const hrow = smem + OFF_H + r * 128;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    uint4 x;
                    x.x = pack_bf16(h[8 * i], h[8 * i + 1]);
                    x.y = pack_bf16(h[8 * i + 2], h[8 * i + 3]);
                    x.z = pack_bf16(h[8 * i + 4], h[8 * i + 5]);
                    x.w = pack_bf16(h[8 * i + 6], h[8 * i + 7]);
                    *reinterpret_cast<uint4 *>(hrow + ((i ^ (r & 7)) << 4)) = x;
                }
                fence_async_smem();
                mbar_arrive(h_full);
                // S = e^{G_C} S0 + K^T V~
                if (!(ok = wait_warp(d_full, ph, 0x424))) break;
                fence_after();
#pragma unroll
                for (int half = 0; half < 4; ++half) {
                    uint32_t d0[16], d1[16], d2[16];
                    tmem_ld16_async(quarter + T_D + half * 16, d0);
                    tmem_ld16_async(quarter + T_D + 64 + half * 16, d1);
                    tmem_ld16_async(quarter + T_D + 128 + half * 16, d2);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        h[half * 16 + i] =
                            fmaf(dec, h[half * 16 + i],
                                 __uint_as_float(d0[i]) +
                                     (__uint_as_float(d1[i]) + __uint_as_float(d2[i])));
                }
                fence_before();
                mbar_arrive(d_free);
            }
            if (ok && a.h_last && r < a.dk) {
#pragma unroll
                for (int i = 0; i < DV; i += 4)
                    if (c0 + i < a.dv)
                        *reinterpret_cast<float4 *>(a.h_last + at + i) =
                            make_float4(h[i], h[i + 1], h[i + 2], h[i + 3]);
            }
        }
    } else if (warp >= 8) {
        // --------------------------------------------------- P and the outputs
        const int w = warp & 3, half = (warp - 8) >> 2, r = 32 * w + lane;
        const uint32_t quarter = tmem + ((uint32_t)(32 * w) << 16);
        uint32_t c = 0;
        bool ok = true;
        for (int64_t id = blockIdx.x; id < items && ok; id += gridDim.x) {
            const Item it = item_of(a, tiles, id);
            const int64_t bq = a.cu ? 0 : it.seq;
            const int col = it.tile * DV + 32 * half;
            __nv_bfloat16 *const o = static_cast<__nv_bfloat16 *>(a.o) + bq * a.os[0] +
                                     it.row0 * a.os[1] + it.h * a.os[2] + col;
            float gn = load_g(a, it, r);
            for (int64_t t0 = 0; t0 < it.len; t0 += C, ++c) {
                const int s = c & 1;
                const uint32_t ph = c & 1;
                const double gl = scan32(gn);
                gn = load_g(a, it, t0 + C + r);
                const float ghi = (float)gl, glo = (float)(gl - (double)ghi);
                if (!(ok = wait_warp(vt_full, ph, 0x431))) break;
                // e^{G_i - (G at the end of block b)} for the blocks before this
                // one, and e^{G_i}
                double sum = gl;
                float f[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int b = 2; b >= 0; --b)
                    if (b < w) {
                        f[b] = __expf((float)sum);
                        sum += tot[s * 4 + b];
                    }
                const float ei = __expf((float)sum) * a.scale;
                if (!(ok = wait_warp(s_full, ph, 0x432))) break;
                fence_after();
#pragma unroll
                for (int bb = 0; bb < 2; ++bb) {
                    const int b = 2 * half + bb;
                    uint32_t p[16];
                    if (b > w) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) p[i] = 0u;
                    } else {
                        uint32_t x[32];
                        tmem_ld32_async(quarter + T_S + 32 * b, x);
                        tmem_wait_ld();
                        if (b < w) {
                            const float fb = b == 0 ? f[0] : b == 1 ? f[1] : f[2];
                            const float4 *cf = reinterpret_cast<const float4 *>(colf + s * C + 32 * b);
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float4 y = cf[i];
                                p[2 * i] = pack_bf16(__uint_as_float(x[4 * i]) * (y.x * fb),
                                                     __uint_as_float(x[4 * i + 1]) * (y.y * fb));
                                p[2 * i + 1] = pack_bf16(__uint_as_float(x[4 * i + 2]) * (y.z * fb),
                                                         __uint_as_float(x[4 * i + 3]) * (y.w * fb));
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                float e[2];
#pragma unroll
                                for (int z = 0; z < 2; ++z) {
                                    const int j = 2 * i + z;
                                    const float d = (ghi - __shfl_sync(0xffffffffu, ghi, j)) +
                                                    (glo - __shfl_sync(0xffffffffu, glo, j));
                                    e[z] = j <= lane ? __uint_as_float(x[j]) * __expf(d) : 0.0f;
                                }
                                p[i] = pack_bf16(e[0], e[1]);
                            }
                        }
                    }
                    tmem_st16(quarter + T_P + 16 * b, p);
                }
                tmem_wait_st();
                fence_before();
                mbar_arrive(p_full);

                if (!(ok = wait_warp(o_full, ph, 0x433))) break;
                fence_after();
                uint32_t pv[32], qh[32];
                tmem_ld32_async(quarter + T_PV + 32 * half, pv);
                tmem_ld32_async(quarter + T_QH + 32 * half, qh);
                tmem_wait_ld();
                fence_before();
                mbar_arrive(o_free);
                const int64_t t = t0 + r;
                if (t < it.len) {
                    float y[32];
                    float bad = 0.0f;                     // 0, or NaN
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        y[i] = __uint_as_float(pv[i]);
                        bad = fmaf(0.0f, y[i], bad);
                    }
                    if (bad != 0.0f) masked_row(a, it, t0, t, col, y);
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        y[i] = fmaf(y[i], a.scale, __uint_as_float(qh[i]) * ei);
                    __nv_bfloat16 *const row = o + t * a.os[1];
#pragma unroll
                    for (int i = 0; i < 32; i += 8)
                        if (col + i < a.dv) {
                            uint4 x;
                            x.x = pack_bf16(y[i], y[i + 1]);
                            x.y = pack_bf16(y[i + 2], y[i + 3]);
                            x.z = pack_bf16(y[i + 4], y[i + 5]);
                            x.w = pack_bf16(y[i + 6], y[i + 7]);
                            *reinterpret_cast<uint4 *>(row + i) = x;
                        }
                }
            }
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// ----------------------------------------------------------------- host
static PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;

static int get_encode() {
    if (g_encode) return MB2_OK;
    cudaDriverEntryPointQueryResult q;
    void *fn = nullptr;
    cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
    if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || !fn)
        return fail(MB2_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
    g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    return MB2_OK;
}

// (batch, tokens, heads, width) bf16 as a 4D map of 128-token x 64-column boxes;
// *ok = false when TMA cannot address it
static int token_map(CUtensorMap *map, const void *p, const int64_t (&s)[3], int64_t batch,
                     int64_t tokens, int64_t heads, int64_t width, bool *ok) {
    const int64_t n[3] = {batch, tokens, heads};
    int64_t st[3];
    *ok = aligned(p, 16) && tokens < 0x7fffff00 && batch < 0x7fffffff;
    for (int i = 0; i < 3; ++i) {
        st[i] = n[i] > 1 ? s[i] : 8;
        if (st[i] <= 0 || st[i] % 8 || st[i] >= (1ll << 38)) *ok = false;
    }
    if (!*ok) return MB2_OK;
    cuuint64_t dims[4] = {(cuuint64_t)width, (cuuint64_t)heads, (cuuint64_t)tokens, (cuuint64_t)batch};
    cuuint64_t strides[3] = {(cuuint64_t)st[2] * 2, (cuuint64_t)st[1] * 2, (cuuint64_t)st[0] * 2};
    cuuint32_t box[4] = {64, 1, (cuuint32_t)C, 1};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(p), dims,
                          strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(MB2_ERR_CUDA, "decay_attention: cuTensorMapEncodeTiled failed (%d)", (int)r);
    return MB2_OK;
}

// bf16 prompts with widths in whole 16-byte groups, at rows TMA can address
static bool fits(const Args &a) {
    return a.dtype == MB2_BF16 && a.dk <= 128 && a.dk % 8 == 0 && a.dv % 8 == 0 && a.seqlen > 0 &&
           aligned(a.o, 16) && a.os[0] % 8 == 0 && a.os[1] % 8 == 0 && a.os[2] % 8 == 0 &&
           (!a.h0 || aligned(a.h0, 16)) && (!a.h_last || aligned(a.h_last, 16));
}

int chunked(const Args &a, cudaStream_t st, bool *used) {
    *used = false;
    if (!fits(a)) return MB2_OK;
    MB2_TRY(get_encode());
    CUtensorMap mq, mk, mv;
    const int64_t batch = a.cu ? 1 : a.seqs;
    bool ok[3];
    MB2_TRY(token_map(&mq, a.q, a.qs, batch, a.seqlen, a.heads / a.q_rep, a.dk, &ok[0]));
    MB2_TRY(token_map(&mk, a.k, a.ks, batch, a.seqlen, a.heads / a.k_rep, a.dk, &ok[1]));
    MB2_TRY(token_map(&mv, a.v, a.vs, batch, a.seqlen, a.heads / a.v_rep, a.dv, &ok[2]));
    if (!ok[0] || !ok[1] || !ok[2]) return MB2_OK;
    *used = true;
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(decay_chunk_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)SMEM_BYTES);
    if (e != cudaSuccess) return fail(MB2_ERR_CUDA, "decay_attention: %s", cudaGetErrorString(e));
    const int tiles = (int)ceil_div(a.dv, DV);
    const int64_t items = (int64_t)tiles * a.heads * a.seqs;
    const unsigned grid = (unsigned)(items < sms ? items : sms);
    decay_chunk_kernel<<<grid, THREADS, SMEM_BYTES, st>>>(mq, mk, mv, a, tiles, items);
    return check_launch("decay_chunk_kernel");
}

int tc_status(int *code, int clear) {
    cudaError_t e = cudaMemcpyFromSymbol(code, g_mb2_device_error, sizeof(int));
    if (e == cudaSuccess && clear) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_mb2_device_error, &zero, sizeof(int));
    }
    if (e != cudaSuccess) return fail(MB2_ERR_CUDA, "device_status: %s", cudaGetErrorString(e));
    return MB2_OK;
}

}  // namespace decay
}  // namespace mb2
