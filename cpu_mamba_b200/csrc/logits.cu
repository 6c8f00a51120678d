// Adjustment of logits before a token is chosen: penalties for tokens that were seen,
// biases, temperature, a grammar's bit mask, in one pass over each row.
//
// A CTA has a slice of a row, kept in registers as it was loaded.  While the loads are on
// their way it goes through the row's history: tokens that fall in the slice are counted
// in a table in shared memory, one word a token (the number of times generated; the top
// bit for a token of the prompt), so that a token's place in the history does not matter
// and the sums are integers; biases are found by their last entry's index.  Then each
// thread takes the tokens of its own vectors that were met, one after the other (its
// lane's n-th beside the other lanes' n-th), puts their values in the table, and the pass
// over the slice picks them up.  Each logit is read and written once, the history is read
// once a slice, from L2.
#include "common.cuh"

#include <algorithm>

namespace mb2 {
namespace {

constexpr int THREADS = 256;
constexpr int SLICE = 4096;                     // tokens of a CTA

struct LogitArgs {
    const void *logits;
    void *out;
    int64_t ld, ld_out, vocab;
    int splits;
    const void *tokens, *lengths, *prompts;
    int64_t ld_tokens, capacity;
    int tokens64, lengths64, prompts64;
    const float *rep, *freq, *pres, *temp;
    float rep1, freq1, pres1, temp1;
    const void *bias_tokens;
    int64_t ld_bias_tokens, ld_bias, n_bias;
    int bias64;
    const float *bias;
    const uint32_t *mask;
    int64_t ld_mask;
};

__device__ __forceinline__ int64_t int_at(const void *p, int wide, int64_t i) {
    return wide ? static_cast<const int64_t *>(p)[i] : static_cast<const int32_t *>(p)[i];
}

// tokens j, j + THREADS, ... of a list of n, all loads on their way at once; -1 for what
// does not fit 31 bits or is behind the list
template <int MANY> struct Some {
    int t[MANY];
    __device__ __forceinline__ void load(const void *tokens, int wide, int j, int n) {
        if (wide) {
            const int2 *p = static_cast<const int2 *>(tokens) + j;
            int2 v[MANY];
#pragma unroll
            for (int k = 0; k < MANY; ++k)
                v[k] = j + k * THREADS < n ? p[k * THREADS] : make_int2(-1, -1);
#pragma unroll
            for (int k = 0; k < MANY; ++k) t[k] = v[k].y == 0 ? v[k].x : -1;
        } else {
            const int *p = static_cast<const int *>(tokens) + j;
#pragma unroll
            for (int k = 0; k < MANY; ++k) t[k] = j + k * THREADS < n ? p[k * THREADS] : -1;
        }
    }
    template <typename F> __device__ __forceinline__ void each(int j, int n, F f) const {
#pragma unroll
        for (int k = 0; k < MANY; ++k) {
            if ((j & ~31) + k * THREADS >= n) break;          // the whole warp's
            if (j + k * THREADS < n) f(j + k * THREADS, t[k]);
        }
    }
};
// a row of a list of tokens
__device__ __forceinline__ const void *list_row(const void *p, int wide, int64_t at) {
    return static_cast<const char *>(p) + at * (wide ? 8 : 4);
}

// 16 bytes of logits as values and back
template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void get(const uint4 &v, float *z) {
        z[0] = __uint_as_float(v.x), z[1] = __uint_as_float(v.y);
        z[2] = __uint_as_float(v.z), z[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ uint4 put(const float *z) {
        return make_uint4(__float_as_uint(z[0]), __float_as_uint(z[1]), __float_as_uint(z[2]),
                          __float_as_uint(z[3]));
    }
};
template <> struct Vec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void get(const uint4 &v, float *z) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            z[2 * i] = __uint_as_float(w[i] << 16);
            z[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ uint4 put(const float *z) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(z[2 * i], z[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// z / rep for z > 0 (a product by the reciprocal and its correction: the quotient to
// within half a unit and a little; what is not finite stays as the product has it),
// z rep otherwise
__device__ __forceinline__ float penalised(float z, float rep, float inverse) {
    float q = z * (z > 0.0f ? inverse : rep);
    const float c = fmaf(fmaf(-q, rep, z), inverse, q);
    if (z > 0.0f && fabsf(c) < INFINITY) q = c;
    return q;
}

template <typename T>
__global__ void __launch_bounds__(THREADS) adjust_kernel(const LogitArgs a) {
    constexpr int N = Vec<T>::N, NV = SLICE / N / THREADS;
    extern __shared__ __align__(16) unsigned table[];
    const int row = blockIdx.x / a.splits;
    const int tid = threadIdx.x, vocab = (int)a.vocab;
    const bool history = a.tokens != nullptr, biases = a.n_bias > 0, any = history || biases;
    // a bit for each token that was met; its words; later its value in the first of them
    unsigned *met = table, *seen = table + SLICE / 32, *last = seen + (history ? SLICE : 0);
    float *value = reinterpret_cast<float *>(seen);
    // vectors from the aligned address at or below the row's start: the slice's first token
    // may lie before it (a vector at the row's ends holds one of its tokens, so that its 16
    // bytes are inside the allocation)
    const T *src = static_cast<const T *>(a.logits) + row * a.ld;
    const int lead = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
    const int slice0 = (int)(blockIdx.x % a.splits) * SLICE - lead;
    if (slice0 >= vocab) return;                // a row that starts aligned may need one less
    src += slice0;
    uint4 raw[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int i = tid + k * THREADS, t = slice0 + i * N;
        if (t < vocab && t + N > 0) raw[k] = __ldcs(reinterpret_cast<const uint4 *>(src) + i);
    }
    unsigned mine[NV] = {};                     // bit e: token e of the vector was met
    if (any) {
        // the first tokens are asked for before the row's length is known
        constexpr int MANY = 4, MANY_BIAS = 2;
        Some<MANY> tokens;
        Some<MANY_BIAS> marks;
        const void *list = list_row(a.tokens, a.tokens64, row * a.ld_tokens);
        const void *bias_list = list_row(a.bias_tokens, a.bias64, row * a.ld_bias_tokens);
        if (history) tokens.load(list, a.tokens64, tid, (int)a.capacity);
        if (biases) marks.load(bias_list, a.bias64, tid, (int)a.n_bias);
        int len = (int)a.capacity, prompt = 0;
        if (history && a.lengths)
            len = (int)min(max(int_at(a.lengths, a.lengths64, row), (int64_t)0), a.capacity);
        if (history && a.prompts)
            prompt = (int)min(max(int_at(a.prompts, a.prompts64, row), (int64_t)0), a.capacity);
        const float rep = a.rep ? a.rep[row] : a.rep1, freq = a.freq ? a.freq[row] : a.freq1;
        const float pres = a.pres ? a.pres[row] : a.pres1;
        const float inverse_rep = 1.0f / rep;
        const int words = SLICE / 32 + (history ? SLICE : 0) + (biases ? SLICE : 0);
        for (int i = tid * 4; i < words; i += THREADS * 4)
            *reinterpret_cast<uint4 *>(table + i) = make_uint4(0, 0, 0, 0);
        __syncthreads();
        // the row's tokens in the slice: lowest .. lowest + span
        const int lowest = max(slice0, 0), below = lowest - slice0;
        const unsigned span = min(slice0 + SLICE, vocab) - lowest;
        if (history) {
            auto one = [&](int j, int t) {
                const unsigned u = (unsigned)(t - lowest);
                if (u >= span) return;
                const unsigned i = u + below;
                if (j < prompt) atomicOr(&seen[i], 0x80000000u);
                else atomicAdd(&seen[i], 1u);
                atomicOr(&met[i >> 5], 1u << (i & 31));
            };
            tokens.each(tid, len, one);
            for (int j = tid + MANY * THREADS; j < len; j += MANY * THREADS) {
                tokens.load(list, a.tokens64, j, len);
                tokens.each(j, len, one);
            }
        }
        if (biases) {
            const int n = (int)a.n_bias;
            auto one = [&](int j, int t) {
                const unsigned u = (unsigned)(t - lowest);
                if (u >= span) return;
                const unsigned i = u + below;
                atomicMax(&last[i], (unsigned)j + 1);
                atomicOr(&met[i >> 5], 1u << (i & 31));
            };
            marks.each(tid, n, one);
            for (int j = tid + MANY_BIAS * THREADS; j < n; j += MANY_BIAS * THREADS) {
                marks.load(bias_list, a.bias64, j, n);
                marks.each(j, n, one);
            }
        }
        __syncthreads();
        unsigned left = 0;                      // all of the thread's tokens that were met
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int i = (tid + k * THREADS) * N;
            mine[k] = met[i >> 5] >> (i & 31) & ((1u << N) - 1u);
            left |= mine[k] << k * N;
        }
        while (left) {
            const int e = __ffs(left) - 1, i = (tid + e / N * THREADS) * N + e % N;
            left &= left - 1;
            float z = io<T>::to_f(src[i]);
            if (history) {
                const unsigned s = seen[i], times = s & 0x7fffffffu;
                if (s) z = penalised(z, rep, inverse_rep);
                if (times) z = z - freq * (float)times - pres;
            }
            if (biases) {
                const unsigned b = last[i];
                if (b) z += a.bias[row * a.ld_bias + b - 1];
            }
            value[i] = z;
        }
    }
    float temp = a.temp ? a.temp[row] : a.temp1;
    if (temp == 0.0f) temp = 1.0f;
    // a product by the reciprocal, off by up to one unit and as torch divides by a number (so
    // that a sampler has the same bits with rules and without); a corrected quotient, half a
    // unit, took 66 instead of 61 us at 512 x 50257.  Divided where the reciprocal may not be
    // normal
    const bool divide = !(fabsf(temp) > 1e-30f && fabsf(temp) < 1e30f);
    const float inverse = 1.0f / temp;
    T *dst = static_cast<T *>(a.out) + row * a.ld_out + slice0;
    const bool together = (reinterpret_cast<uintptr_t>(dst) & 15) == 0;       // as the source
    const uint32_t *mask = a.mask ? a.mask + row * a.ld_mask : nullptr;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int i = (tid + k * THREADS) * N, t = slice0 + i;
        if (t >= vocab || t + N <= 0) continue;
        float z[N];
        Vec<T>::get(raw[k], z);
#pragma unroll
        for (int q = 0; q < N; q += 4) {
            if (!(mine[k] >> q & 15u)) continue;
            const float4 v = *reinterpret_cast<const float4 *>(value + i + q);
            z[q] = mine[k] >> q & 1u ? v.x : z[q];
            z[q + 1] = mine[k] >> q & 2u ? v.y : z[q + 1];
            z[q + 2] = mine[k] >> q & 4u ? v.z : z[q + 2];
            z[q + 3] = mine[k] >> q & 8u ? v.w : z[q + 3];
        }
        if (temp != 1.0f) {
            if (divide) {
#pragma unroll
                for (int e = 0; e < N; ++e) z[e] = z[e] / temp;
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) z[e] = z[e] * inverse;
            }
        }
        if (mask) {
            // bit e: token t + e, from two words at most
            uint32_t bits = mask[max(t, 0) >> 5];
            if (t < 0) bits <<= -t;
            else bits = __funnelshift_r(bits, mask[min(t + N, vocab) - 1 >> 5], t & 31);
#pragma unroll
            for (int e = 0; e < N; ++e) z[e] = bits >> e & 1u ? z[e] : -INFINITY;
        }
        const uint4 out = Vec<T>::put(z);
        if (together && t >= 0 && t + N <= vocab) {
            *reinterpret_cast<uint4 *>(dst + i) = out;
        } else {
            T v[N];
            *reinterpret_cast<uint4 *>(v) = out;
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (t + e >= 0 && t + e < vocab) dst[i + e] = v[e];
        }
    }
}

}  // namespace
}  // namespace mb2

using namespace mb2;

extern "C" int mb2_adjust_logits(const mb2_adjust_logits_desc *d, mb2_stream_t stream) {
    const char *what = "adjust_logits";
    MB2_REQUIRE(d, MB2_ERR_ARG, "%s: null descriptor", what);
    MB2_REQUIRE(d->dtype == MB2_F32 || d->dtype == MB2_BF16, MB2_ERR_ARG, "%s: bad dtype", what);
    MB2_REQUIRE(d->rows >= 0 && d->vocab > 0 && d->capacity >= 0 && d->n_bias >= 0, MB2_ERR_SHAPE,
                "%s: bad size", what);
    MB2_REQUIRE(d->vocab <= 1 << 30 && d->capacity <= 1 << 30 && d->n_bias <= 1 << 30,
                MB2_ERR_SHAPE, "%s: more than 2^30: vocabulary %lld, %lld tokens, %lld biases", what,
                (long long)d->vocab, (long long)d->capacity, (long long)d->n_bias);
    if (d->rows == 0) return MB2_OK;
    MB2_REQUIRE(d->logits && d->out && (d->n_bias == 0 || (d->bias && d->bias_tokens)), MB2_ERR_ARG,
                "%s: null pointer", what);
    MB2_REQUIRE(d->repetition_penalty || d->repetition > 0.0f, MB2_ERR_ARG,
                "%s: repetition penalty must be positive", what);
    MB2_REQUIRE(d->temperatures || d->temperature >= 0.0f, MB2_ERR_ARG,
                "%s: temperature must not be negative", what);
    LogitArgs a{};
    a.logits = d->logits, a.out = d->out, a.ld = d->ld, a.ld_out = d->ld_out, a.vocab = d->vocab;
    a.splits = (int)ceil_div(d->vocab + 16 / (int64_t)dtype_size(d->dtype) - 1, SLICE);
    a.tokens = d->capacity ? d->tokens : nullptr;
    a.lengths = d->lengths, a.prompts = d->prompt_lengths;
    a.ld_tokens = d->ld_tokens, a.capacity = d->capacity;
    a.tokens64 = d->tokens_i64, a.lengths64 = d->lengths_i64, a.prompts64 = d->prompt_lengths_i64;
    a.rep = d->repetition_penalty, a.freq = d->frequency_penalty, a.pres = d->presence_penalty;
    a.temp = d->temperatures, a.rep1 = d->repetition, a.freq1 = d->frequency;
    a.pres1 = d->presence, a.temp1 = d->temperature;
    a.bias_tokens = d->bias_tokens, a.ld_bias_tokens = d->ld_bias_tokens, a.ld_bias = d->ld_bias;
    a.n_bias = d->n_bias, a.bias64 = d->bias_tokens_i64, a.bias = d->bias;
    a.mask = d->mask, a.ld_mask = d->ld_mask;
    const int64_t blocks = d->rows * a.splits;
    MB2_REQUIRE(blocks < (1ll << 31), MB2_ERR_SHAPE, "%s: too many rows", what);
    cudaStream_t st = (cudaStream_t)stream;
    const int tables = (a.tokens ? 1 : 0) + (a.n_bias ? 1 : 0);
    const size_t smem = tables ? (SLICE / 32 + tables * SLICE) * sizeof(unsigned) : 0;
    if (d->dtype == MB2_F32) adjust_kernel<float><<<(unsigned)blocks, THREADS, smem, st>>>(a);
    else adjust_kernel<__nv_bfloat16><<<(unsigned)blocks, THREADS, smem, st>>>(a);
    return check_launch(what);
}
