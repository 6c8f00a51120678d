// The norms around a block, fused with its gate and the residual add:
//   u = RMSNorm(x) w silu(z)   or   RMSNorm(x silu(z)) w     (norm and gate optional,
//                                                             the norm by groups of columns)
//   r = residual + s u          (s a number or a vector)
//   n = RMSNorm(r) w'           (the next block's norm)
// HBM-bound: a row's operands are read once, all loads issued before the first
// reduction, and the row stays in registers through both norms.  Sums and all
// arithmetic in fp32; r and n are each rounded once (n from the unrounded r).
#include "common.cuh"

namespace mb2 {
namespace {

struct NormArgs {
    int64_t rows;
    int width, group;                    // group: columns per first norm
    const void *x, *gate, *weight, *resid, *rscale, *next_w;
    void *out, *next_out;
    int64_t ld_x, ld_gate, ld_resid, ld_out, ld_next;
    float scale, eps;
    int before;                          // norm, then gate
    int wf32, sf32, nf32;                // vector operands held in fp32
};

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Pack { T e[VEC]; };

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const void *p, int64_t i, float (&r)[VEC]) {
    if constexpr (sizeof(T) * VEC > 16) {
        constexpr int H = 16 / (int)sizeof(T);
#pragma unroll
        for (int h = 0; h < VEC / H; ++h) {
            const Pack<T, H> v = *reinterpret_cast<const Pack<T, H> *>(static_cast<const T *>(p) + i + h * H);
#pragma unroll
            for (int e = 0; e < H; ++e) r[h * H + e] = io<T>::to_f(v.e[e]);
        }
    } else {
        const Pack<T, VEC> v = *reinterpret_cast<const Pack<T, VEC> *>(static_cast<const T *>(p) + i);
#pragma unroll
        for (int e = 0; e < VEC; ++e) r[e] = io<T>::to_f(v.e[e]);
    }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(void *p, int64_t i, const float (&r)[VEC]) {
    constexpr int H = sizeof(T) * VEC > 16 ? 16 / (int)sizeof(T) : VEC;
#pragma unroll
    for (int h = 0; h < VEC / H; ++h) {
        Pack<T, H> v;
#pragma unroll
        for (int e = 0; e < H; ++e) v.e[e] = io<T>::from_f(r[h * H + e]);
        *reinterpret_cast<Pack<T, H> *>(static_cast<T *>(p) + i + h * H) = v;
    }
}
// a vector operand (weights): T or fp32
template <typename T, int VEC>
__device__ __forceinline__ void load_w(const void *p, int f32, int64_t i, float (&r)[VEC]) {
    if (f32) load_vec<float, VEC>(p, i, r);
    else load_vec<T, VEC>(p, i, r);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// A row per warp (WARP) or per CTA; thread i of the row's TPR threads holds the
// VEC-wide vectors i + j TPR, j < VPT.
template <typename T, typename RT, int VEC, int VPT, bool WARP, int MAXT>
__global__ void __launch_bounds__(MAXT)
gated_norm_kernel(const NormArgs a) {
    extern __shared__ float dyn[];       // grouped norms that a shuffle cannot reduce
    __shared__ float red[2][32];
    const int tpr = WARP ? 32 : (int)blockDim.x;
    const int tid = WARP ? (int)(threadIdx.x & 31) : (int)threadIdx.x;
    const int rpc = WARP ? (int)(blockDim.x >> 5) : 1;
    const int64_t row = (int64_t)blockIdx.x * rpc + (WARP ? (threadIdx.x >> 5) : 0);
    if (row >= a.rows) return;           // whole warps (WARP); never else
    const int nv = a.width / VEC;
    const float inv_w = 1.0f / (float)a.width;

    float u[VPT][VEC], z[VPT][VEC], rs[VPT][VEC];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int i = tid + j * tpr;
        if (i < nv) load_vec<T, VEC>(a.x, row * a.ld_x + (int64_t)i * VEC, u[j]);
    }
    if (a.gate) {
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int i = tid + j * tpr;
            if (i < nv) load_vec<T, VEC>(a.gate, row * a.ld_gate + (int64_t)i * VEC, z[j]);
        }
    }
    if (a.resid) {
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int i = tid + j * tpr;
            if (i < nv) load_vec<RT, VEC>(a.resid, row * a.ld_resid + (int64_t)i * VEC, rs[j]);
        }
    }
    // a sum over the row's threads (every thread of the row calls it)
    auto row_sum = [&](float v, int slot) {
        v = warp_sum(v);
        if (WARP) return v;
        const int wid = threadIdx.x >> 5, nw = (int)(blockDim.x >> 5);
        if ((threadIdx.x & 31) == 0) red[slot][wid] = v;
        __syncthreads();
        v = (int)(threadIdx.x & 31) < nw ? red[slot][threadIdx.x & 31] : 0.0f;
        return warp_sum(v);
    };

    if (a.gate) {
#pragma unroll
        for (int j = 0; j < VPT; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                z[j][e] = silu_f(z[j][e]);
                if (!a.before) u[j][e] *= z[j][e];
            }
    }
    if (a.weight) {
        float ss[VPT];
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            ss[j] = 0.0f;
            if (tid + j * tpr < nv) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) ss[j] = fmaf(u[j][e], u[j][e], ss[j]);
            }
        }
        const int gv = a.group / VEC;    // vectors per group
        if (gv == nv) {
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < VPT; ++j) s += ss[j];
            s = rsqrtf(row_sum(s, 0) * inv_w + a.eps);
#pragma unroll
            for (int j = 0; j < VPT; ++j) ss[j] = s;
        } else if (gv <= 32 && (gv & (gv - 1)) == 0) {
            // a group is gv neighbouring lanes (tpr is a multiple of 32)
            const float inv_g = 1.0f / (float)a.group;
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                float s = ss[j];
                for (int o = gv >> 1; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
                ss[j] = rsqrtf(s * inv_g + a.eps);
            }
        } else {
            // partial sums through shared memory, one warp per group
            const float inv_g = 1.0f / (float)a.group;
            const int ng = nv / gv;
            float *part = dyn + (WARP ? (threadIdx.x >> 5) * (nv + ng) : 0);
            float *grp = part + nv;
#pragma unroll
            for (int j = 0; j < VPT; ++j)
                if (tid + j * tpr < nv) part[tid + j * tpr] = ss[j];
            if (WARP) __syncwarp(); else __syncthreads();
            const int lane = threadIdx.x & 31;
            for (int gi = WARP ? 0 : (int)(threadIdx.x >> 5); gi < ng; gi += WARP ? 1 : tpr >> 5) {
                float s = 0.0f;
                for (int i = lane; i < gv; i += 32) s += part[gi * gv + i];
                s = warp_sum(s);
                if (lane == 0) grp[gi] = rsqrtf(s * inv_g + a.eps);
            }
            if (WARP) __syncwarp(); else __syncthreads();
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                const int i = tid + j * tpr;
                if (i < nv) ss[j] = grp[i / gv];
            }
        }
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int i = tid + j * tpr;
            if (i < nv) {
                float w[VEC];
                load_w<T, VEC>(a.weight, a.wf32, (int64_t)i * VEC, w);
#pragma unroll
                for (int e = 0; e < VEC; ++e) u[j][e] = u[j][e] * ss[j] * w[e];
            }
        }
    }
    if (a.gate && a.before) {
#pragma unroll
        for (int j = 0; j < VPT; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e) u[j][e] *= z[j][e];
    }
    if (!a.resid) {
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int i = tid + j * tpr;
            if (i < nv) store_vec<T, VEC>(a.out, row * a.ld_out + (int64_t)i * VEC, u[j]);
        }
        return;
    }
    float s2 = 0.0f;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int i = tid + j * tpr;
        if (i < nv) {
            float sc[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) sc[e] = a.scale;
            if (a.rscale) load_w<T, VEC>(a.rscale, a.sf32, (int64_t)i * VEC, sc);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                u[j][e] = fmaf(sc[e], u[j][e], rs[j][e]);
                s2 = fmaf(u[j][e], u[j][e], s2);
            }
            store_vec<RT, VEC>(a.out, row * a.ld_out + (int64_t)i * VEC, u[j]);
        }
    }
    if (a.next_w) {
        const float rstd = rsqrtf(row_sum(s2, 1) * inv_w + a.eps);
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int i = tid + j * tpr;
            if (i < nv) {
                float w[VEC];
                load_w<T, VEC>(a.next_w, a.nf32, (int64_t)i * VEC, w);
#pragma unroll
                for (int e = 0; e < VEC; ++e) u[j][e] = u[j][e] * rstd * w[e];
                store_vec<T, VEC>(a.next_out, row * a.ld_next + (int64_t)i * VEC, u[j]);
            }
        }
    }
}

template <typename T, typename RT, int VEC, int VPT, bool WARP, int MAXT>
static int launch(const NormArgs &a, cudaStream_t st) {
    const int nv = a.width / VEC;
    const int threads = WARP ? 128 : (int)round_up(ceil_div(nv, VPT), 32);
    const int rpc = WARP ? 4 : 1;
    const int64_t grid = ceil_div(a.rows, rpc);
    MB2_REQUIRE(grid <= 0x7fffffff, MB2_ERR_SHAPE, "gated_norm: too many rows");
    const int gv = a.group / VEC;
    const bool shfl = gv == nv || (gv <= 32 && (gv & (gv - 1)) == 0);
    const size_t smem = shfl || !a.weight ? 0 : sizeof(float) * (size_t)rpc * (nv + nv / gv);
    auto kern = gated_norm_kernel<T, RT, VEC, VPT, WARP, MAXT>;
    if (smem > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)smem);
        if (e != cudaSuccess) return fail(MB2_ERR_CUDA, "gated_norm: %s", cudaGetErrorString(e));
    }
    kern<<<(unsigned)grid, threads, smem, st>>>(a);
    return check_launch("gated_norm_kernel");
}

// A warp per row where the row fits its registers and there are rows to fill
// the GPU with; a CTA per row otherwise.
template <typename T, typename RT>
static int dispatch(const NormArgs &a, bool vec, cudaStream_t st) {
    constexpr int V = 16 / (int)sizeof(T);
    const bool many = a.rows >= 148 * 16;
    if (vec) {
        const int nv = a.width / V;
        if (many && nv <= 32) return launch<T, RT, V, 1, true, 128>(a, st);
        if (many && nv <= 64) return launch<T, RT, V, 2, true, 128>(a, st);
        if (many && nv <= 96) return launch<T, RT, V, 3, true, 128>(a, st);
        if (many && nv <= 128) return launch<T, RT, V, 4, true, 128>(a, st);
        if (nv <= 256) return launch<T, RT, V, 1, false, 256>(a, st);
        if (nv <= 512) return launch<T, RT, V, 2, false, 256>(a, st);
        if (nv <= 1024) return launch<T, RT, V, 4, false, 256>(a, st);
        return launch<T, RT, V, 16 / V, false, 1024>(a, st);   // width <= 16384
    }
    if (many && a.width <= 128) return launch<T, RT, 1, 4, true, 128>(a, st);
    // odd rows, an element at a time; few elements a thread, since 16 of three operands
    // spill (8000 rows of 3501 in fp32, all parts: 230 us with 16, 167 with 4; 4000 of
    // 7001: 241 and 200 with 8; 21 rows of 3501 in bf16: 11.3 and 5.4)
    if (many && a.width <= 256) return launch<T, RT, 1, 8, true, 128>(a, st);
    if (a.width <= 1024) return launch<T, RT, 1, 4, false, 256>(a, st);
    if (a.width <= 2048) return launch<T, RT, 1, 8, false, 256>(a, st);
    if (a.width <= 4096) return launch<T, RT, 1, 4, false, 1024>(a, st);
    if (a.width <= 8192) return launch<T, RT, 1, 8, false, 1024>(a, st);
    return launch<T, RT, 1, 16, false, 1024>(a, st);
}

}  // namespace
}  // namespace mb2

using namespace mb2;

extern "C" int mb2_gated_norm(const mb2_gated_norm_desc *d, mb2_stream_t stream) {
    MB2_REQUIRE(d, MB2_ERR_ARG, "gated_norm: null descriptor");
    MB2_REQUIRE((d->dtype == MB2_F32 || d->dtype == MB2_BF16) &&
                    (d->residual_dtype == d->dtype || d->residual_dtype == MB2_F32),
                MB2_ERR_ARG, "gated_norm: bad dtype");
    MB2_REQUIRE(d->rows >= 0 && d->width > 0, MB2_ERR_SHAPE, "gated_norm: bad size");
    MB2_REQUIRE(d->width <= 16384, MB2_ERR_SHAPE, "gated_norm: width %lld > 16384 not supported",
                (long long)d->width);
    const int64_t group = d->group > 0 ? d->group : d->width;
    MB2_REQUIRE(d->width % group == 0, MB2_ERR_SHAPE,
                "gated_norm: group %lld does not divide width %lld", (long long)group,
                (long long)d->width);
    if (d->rows == 0) return MB2_OK;
    MB2_REQUIRE(d->x && d->out, MB2_ERR_ARG, "gated_norm: null pointer");
    MB2_REQUIRE(d->residual || (!d->residual_scale && !d->next_weight), MB2_ERR_ARG,
                "gated_norm: residual_scale and next_weight need a residual");
    MB2_REQUIRE(!d->next_weight || d->next_out, MB2_ERR_ARG, "gated_norm: null next_out");
    NormArgs a;
    a.rows = d->rows;
    a.width = (int)d->width;
    a.group = (int)group;
    a.x = d->x; a.gate = d->gate; a.weight = d->weight; a.resid = d->residual;
    a.rscale = d->residual_scale; a.next_w = d->next_weight;
    a.out = d->out; a.next_out = d->next_out;
    a.ld_x = d->ld_x; a.ld_gate = d->ld_gate; a.ld_resid = d->ld_residual;
    a.ld_out = d->ld_out; a.ld_next = d->ld_next;
    a.scale = d->scale; a.eps = d->eps; a.before = d->norm_before_gate;
    a.wf32 = d->weight_f32; a.sf32 = d->scale_f32; a.nf32 = d->next_f32;
    const size_t e = dtype_size(d->dtype), re = dtype_size(d->residual ? d->residual_dtype : d->dtype);
    const int64_t V = 16 / (int64_t)e;
    auto ok = [&](const void *p, int64_t ld, size_t sz) {
        return !p || (aligned(p, 16) && (ld * (int64_t)sz) % 16 == 0);
    };
    const bool vec = a.width % V == 0 && group % V == 0 && ok(a.x, a.ld_x, e) &&
                     ok(a.gate, a.ld_gate, e) && ok(a.resid, a.ld_resid, re) &&
                     ok(a.out, a.ld_out, re) && ok(a.next_out, a.ld_next, e) &&
                     ok(a.weight, 0, 4) && ok(a.rscale, 0, 4) && ok(a.next_w, 0, 4);
    cudaStream_t st = (cudaStream_t)stream;
    if (d->dtype == MB2_F32) return dispatch<float, float>(a, vec, st);
    if (d->residual && d->residual_dtype == MB2_F32)
        return dispatch<__nv_bfloat16, float>(a, vec, st);
    return dispatch<__nv_bfloat16, __nv_bfloat16>(a, vec, st);
}
