// Beam search on the GPU: the selection over beams and vocabulary, and the
// reordering of the beams' recurrent states.
//
// beam_select: candidate (k, v) of a batch has the value
//   scores[k] + logits[k, v] - log sum_v' exp(logits[k, v'])
// and the best `num` of all K V candidates come out in order, ties to the
// lowest beam, then the lowest token.  Two kernels:
//   beam_rows   one CTA per (row, slice of up to 32 KB): the slice stays in
//               registers, so the logits are read once; its maximum, its sum
//               of exponentials and its best `num` (value, token) pairs
//   beam_merge  one CTA per batch: the rows' normalisers (64-bit sums of the
//               slices') and a merge of the slices' sorted lists, comparing the
//               candidates' 64-bit values
// The logits have to be read once; what bounds each kernel instead stands there.
#include "common.cuh"
#include "pair.cuh"

#include <algorithm>
#include <exception>
#include <utility>
#include <vector>

namespace mb2 {
namespace {

constexpr int ROW_THREADS = 256;
constexpr int NV = 8;                         // 16-byte vectors of logits per thread, at most
constexpr int SLICE = ROW_THREADS * NV;       // vectors of a slice, at most
constexpr int LIST = 1024;                    // candidates above a slice's threshold
constexpr int HELD = 256;                     // vectors with a value at the threshold
constexpr int MAX_NUM = 64;
constexpr int MAX_BEAMS = 32;
constexpr int MAX_VOCAB = 1 << 20;

// fp32 ordered as unsigned, 0 below every value; NaN orders as -inf
__device__ __forceinline__ uint32_t order_key(float v) {
    if (v != v) v = -INFINITY;
    const uint32_t b = __float_as_uint(v + 0.0f);           // -0 -> +0
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

struct RowArgs {
    const void *logits;
    int64_t s_batch, s_beam;                  // strides
    int beams, vocab, num, splits;
    int per;                                  // 16-byte vectors of a slice
    const uint8_t *finished;
    float *part_max, *part_sum;               // (rows, splits)
    uint64_t *part_list;                      // (rows, splits, num): key << 32 | ~token, 0: none
};

// a vector of logits: the values of its 32-bit words
template <typename T> struct Word;
template <> struct Word<float> {
    static constexpr int N = 1;
    static __device__ __forceinline__ float at(uint32_t w, int) { return __uint_as_float(w); }
    static __device__ __forceinline__ uint32_t masked(uint32_t w, int, bool in) {
        return in ? w : 0xff800000u;
    }
    // the larger values (a NaN loses), the largest, and whether one is >= t
    static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }
    static __device__ __forceinline__ float top(uint32_t w) { return __uint_as_float(w); }
    static __device__ __forceinline__ bool reaches(uint32_t w, uint32_t t) {
        return __uint_as_float(w) >= __uint_as_float(t);
    }
    static __device__ __forceinline__ uint32_t splat(float v) { return __float_as_uint(v); }
};
template <> struct Word<__nv_bfloat16> {
    static constexpr int N = 2;
    static __device__ __forceinline__ float at(uint32_t w, int i) {
        return __uint_as_float(i ? w & 0xffff0000u : w << 16);
    }
    static __device__ __forceinline__ uint32_t masked(uint32_t w, int i, bool in) {
        return in ? w : i ? (w & 0xffffu) | 0xff800000u : (w & 0xffff0000u) | 0xff80u;
    }
    static __device__ __forceinline__ __nv_bfloat162 two(uint32_t w) {
        return *reinterpret_cast<const __nv_bfloat162 *>(&w);
    }
    static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) {
        const __nv_bfloat162 m = __hmax2(two(a), two(b));
        return *reinterpret_cast<const uint32_t *>(&m);
    }
    static __device__ __forceinline__ float top(uint32_t w) { return fmaxf(at(w, 0), at(w, 1)); }
    static __device__ __forceinline__ bool reaches(uint32_t w, uint32_t t) {
        return __hge2_mask(two(w), two(t)) != 0;
    }
    static __device__ __forceinline__ uint32_t splat(float v) {
        return (__float_as_uint(v) >> 16) * 0x10001u;        // v is a bf16 value
    }
};

// The slice is kept as it was loaded (32 registers a thread), four CTAs to an SM.
// 512 rows of 50257 bf16 logits, 25 us = 2.1 TB/s: issue slots bound it, half of
// them the search for the best, whose cost per slice does not shrink with it.
//   as fp32 keys                                     60 us
//   as loaded, slices of 16 KB                       33
//   slices of 32 KB, three CTAs to an SM             28
//   four                                             25   (64 KB, two: 27)
// Loads and maxima alone take 7 us, the exponentials 4 more.
template <typename T>
__global__ void __launch_bounds__(ROW_THREADS, 4)
beam_rows_kernel(const RowArgs a) {
    constexpr int VEC = 16 / (int)sizeof(T), WARPS = ROW_THREADS / 32;
    constexpr int WN = Word<T>::N;                // values per 32-bit word
    __shared__ uint64_t list[LIST];
    __shared__ uint64_t best[WARPS];
    __shared__ float redf[2][WARPS];
    __shared__ uint32_t reach_key[WARPS];
    __shared__ uint4 held_vec[HELD];
    __shared__ int held_at[HELD];
    __shared__ int count, held;
    const int split = blockIdx.x, row = blockIdx.y;
    if (a.finished && a.finished[row]) return;              // beam_merge writes its candidates
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const T *p = static_cast<const T *>(a.logits) + (int64_t)(row / a.beams) * a.s_batch +
                 (int64_t)(row % a.beams) * a.s_beam;
    // 16-byte loads from the aligned address at or below the row's start; the
    // elements outside the row are dropped (their 16 bytes hold one inside it)
    const int lead = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
    const T *base = p - lead;
    const int nvec = (a.vocab + lead + VEC - 1) / VEC;
    const int v0 = split * a.per + tid, end = min(nvec, (split + 1) * a.per);
    if (tid == 0) count = held = 0;

    constexpr uint32_t kNone = Word<T>::N == 2 ? 0xff80ff80u : 0xff800000u;   // -inf
    uint32_t raw[NV][4];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int v = v0 + j * ROW_THREADS;
        uint4 x = make_uint4(kNone, kNone, kNone, kNone);
        if (v < end) x = __ldcs(reinterpret_cast<const uint4 *>(base) + v);
        raw[j][0] = x.x; raw[j][1] = x.y; raw[j][2] = x.z; raw[j][3] = x.w;
    }
    // token of value (j, w, i)
    auto token = [&](int j, int w, int i) {
        return (v0 + j * ROW_THREADS) * VEC + w * WN + i - lead;
    };
    uint32_t vmax[NV], wmax = kNone;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int v = v0 + j * ROW_THREADS;
        if (v == 0 || v == nvec - 1) {                       // the row's first and last 16 bytes
#pragma unroll
            for (int w = 0; w < 4; ++w)
#pragma unroll
                for (int i = 0; i < WN; ++i) {
                    const int t = token(j, w, i);
                    raw[j][w] = Word<T>::masked(raw[j][w], i, t >= 0 && t < a.vocab);
                }
        }
        vmax[j] = Word<T>::max(Word<T>::max(raw[j][0], raw[j][1]),
                               Word<T>::max(raw[j][2], raw[j][3]));
        wmax = Word<T>::max(wmax, vmax[j]);
    }
    const float tmax = fmaxf(Word<T>::top(wmax), -INFINITY);

    // A threshold that at least `num` threads reach by their largest value, so that
    // the slice's best `num` are among the values at or above it: the least of the
    // warps' ceil(num / 8)-th largest thread maxima.
    const int quota = (a.num + WARPS - 1) / WARPS;
    const uint32_t kmax = v0 < end ? order_key(tmax) : 0u;
    {
        uint32_t left = kmax, got = 0;
        for (int r = 0; r < quota; ++r) {
            got = __reduce_max_sync(0xffffffffu, left);
            if (r == 0 && lane == 0) redf[0][wid] = got ? key_value(got) : -INFINITY;
            const uint32_t who = __ballot_sync(0xffffffffu, left == got);
            if (lane == __ffs(who) - 1) left = 0;
        }
        if (lane == 0) reach_key[wid] = got;                 // 0: fewer threads than that
    }
    __syncthreads();
    float m = -INFINITY;
    uint32_t thr = 0xffffffffu;
    int full = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        m = fmaxf(m, redf[0][w]);
        const uint32_t k = reach_key[w];
        if (k) {
            ++full;
            thr = k < thr ? k : thr;
        }
    }
    // x - m first: a large common offset has to cancel.  All masked: every term is
    // e^-inf; a NaN or +inf makes the sum NaN
    const float off = m == -INFINITY ? 0.0f : m;
    const uint64_t noff = pair(-off), log2e = pair(kLog2e);
    uint64_t sums[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        if (v0 - lane + j * ROW_THREADS >= end) break;       // behind the slice, for the whole warp
#pragma unroll
        for (int n = 0; n < VEC; n += 2) {
            const uint64_t y = mul2(add2(pair(__float_as_uint(Word<T>::at(raw[j][n / WN], n % WN)),
                                              __float_as_uint(Word<T>::at(raw[j][(n + 1) / WN],
                                                                          (n + 1) % WN))),
                                         noff), log2e);
            sums[n / 2 % 2] = add2(sums[n / 2 % 2],
                                   pair(__float_as_uint(ex2(__uint_as_float(lo_of(y)))),
                                        __float_as_uint(ex2(__uint_as_float(hi_of(y))))));
        }
    }
    sums[0] = add2(sums[0], sums[1]);
    float sum = __uint_as_float(lo_of(sums[0])) + __uint_as_float(hi_of(sums[0]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) redf[1][wid] = sum;

    if (full * quota < a.num) {
        // a short slice or a large `num`: bisection of the key's bits, stopped once few
        // more threads than needed reach it
        thr = 1;
        const int reach = __syncthreads_count(kmax > 0);
        if (reach > a.num) {
            thr = 0;
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t t = thr | (1u << bit);
                const int c = __syncthreads_count(kmax >= t);
                if (c >= a.num) thr = t;
                if (c >= a.num && c <= a.num + 8) break;
            }
            // the bits need not be a value of T: the least thread maximum that
            // reaches them is, and the same threads reach it
            __shared__ uint32_t least;
            if (tid == 0) least = 0xffffffffu;
            __syncthreads();
            if (kmax >= thr) atomicMin(&least, kmax);
            __syncthreads();
            thr = least;
        }
    }
    // The vectors with a value at the threshold (NaN, worth -inf, only counts where
    // the threshold is that low) go through shared memory, so that their values are
    // looked at by as many threads: taken from the registers, that is 1000 instructions
    // of which a few are used.
    {
        const uint32_t tw = Word<T>::splat(key_value(thr));
        const bool all = thr <= order_key(-INFINITY);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (v0 + j * ROW_THREADS < end && (all || Word<T>::reaches(vmax[j], tw))) {
                const int at = atomicAdd(&held, 1);
                if (at < HELD) {
                    held_vec[at] = make_uint4(raw[j][0], raw[j][1], raw[j][2], raw[j][3]);
                    held_at[at] = v0 + j * ROW_THREADS;
                }
            }
        }
    }
    __syncthreads();
    for (int i = tid; i < min(held, HELD) * VEC; i += ROW_THREADS) {
        const uint32_t *words = reinterpret_cast<const uint32_t *>(held_vec);
        const uint32_t k = order_key(Word<T>::at(words[i / WN], i % WN));
        const int t = held_at[i / VEC] * VEC + i % VEC - lead;
        if (k >= thr && t >= 0 && t < a.vocab) {
            const int at = atomicAdd(&count, 1);
            if (at < LIST) list[at] = (uint64_t)k << 32 | (uint32_t)~(uint32_t)t;
        }
    }
    __syncthreads();
    const int64_t part = (int64_t)row * a.splits + split;
    uint64_t *out = a.part_list + part * a.num;
    if (tid == 0) {
        float s = redf[1][0];
        for (int w = 1; w < ROW_THREADS / 32; ++w) s += redf[1][w];
        a.part_max[part] = m;
        a.part_sum[part] = s;
    }
    const int c = count;
    if (held <= HELD && c <= LIST) {
        // distinct entries: each one's rank is the number of larger ones
        for (int i = wid; i < c; i += WARPS) {
            const uint64_t mine = list[i];
            int rank = 0;
            for (int j = 0; j < c; j += 32)
                rank += __popc(__ballot_sync(0xffffffffu, j + lane < c && list[j + lane] > mine));
            if (lane == 0 && rank < a.num) out[rank] = mine;
        }
        for (int i = c + tid; i < a.num; i += ROW_THREADS) out[i] = 0;
        return;
    }
    // many equal logits at the threshold: pick one after the other, from memory again
    // (the values kept in registers for this would cost every call its occupancy)
    uint64_t last = ~0ull;
    for (int n = 0; n < a.num; ++n) {
        uint64_t b = 0;
#pragma unroll 1
        for (int v = v0; v < end; v += ROW_THREADS) {
            const uint4 x = reinterpret_cast<const uint4 *>(base)[v];
            const uint32_t words[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int w = 0; w < 4; ++w)
#pragma unroll
                for (int i = 0; i < WN; ++i) {
                    const int t = v * VEC + w * WN + i - lead;
                    const uint64_t e = (uint64_t)order_key(Word<T>::at(words[w], i)) << 32 |
                                       (uint32_t)~(uint32_t)t;
                    if (t >= 0 && t < a.vocab && e < last && e > b) b = e;
                }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const uint64_t x = __shfl_xor_sync(0xffffffffu, b, o);
            b = x > b ? x : b;
        }
        if (lane == 0) best[wid] = b;
        __syncthreads();
        last = best[0];
        for (int w = 1; w < ROW_THREADS / 32; ++w) last = best[w] > last ? best[w] : last;
        if (tid == 0) out[n] = last;
        __syncthreads();
    }
}

struct MergeArgs {
    int beams, vocab, num, splits;
    int pad;
    const float *scores;
    const uint8_t *finished;
    const float *part_max, *part_sum;
    const uint64_t *part_list;
    float *out_scores;
    int64_t *out_parents, *out_tokens;
    int staged;                               // the lists' entries fit shared memory
};

// a 64-bit value (never NaN) ordered as unsigned, 0 below all; compares as integers,
// and a warp's largest takes three reductions
__device__ __forceinline__ uint64_t order_key64(double v) {
    const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
    return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ double key_value64(uint64_t k) {
    return __longlong_as_double((long long)((k >> 63) ? k & 0x7fffffffffffffffull : ~k));
}
// the larger value, then the lower flat index
__device__ __forceinline__ bool better(uint64_t v, int at, uint64_t v2, int at2) {
    return v > v2 || (v == v2 && at < at2);
}
// a warp's best (value, flat index)
__device__ __forceinline__ void warp_best(uint64_t &v, int &at) {
    const uint32_t hi = (uint32_t)(v >> 32), lo = (uint32_t)v;
    const uint32_t top = __reduce_max_sync(0xffffffffu, hi);
    const uint32_t low = __reduce_max_sync(0xffffffffu, hi == top ? lo : 0u);
    at = __reduce_min_sync(0xffffffffu, hi == top && lo == low ? at : INT32_MAX);
    v = (uint64_t)top << 32 | low;
}

// a launch has 48 KB of shared memory, the kernel's own arrays (1.6 KB) among them
constexpr size_t MERGE_STAGE = 46 * 1024;

// Bound: latency, a chain of `num` warp reductions behind three dependent reads (64
// batches of 32 lists of 16: 9.1 us, of which 16 rounds 4; with the outputs written
// inside the rounds 10.2; lists of 16 KB slices, 56 of them, 13).
__global__ void __launch_bounds__(1024)
beam_merge_kernel(const MergeArgs a) {
    extern __shared__ __align__(16) uint8_t dyn[];
    const int lists = a.beams * a.splits;
    // [lists][num] when staged: values and flat indices (-1: none); entries taken
    const int stage = a.staged ? lists * a.num : 0;
    uint64_t *const s_val = reinterpret_cast<uint64_t *>(dyn);
    int *const s_at = reinterpret_cast<int *>(s_val + stage);
    int *const heads = s_at + stage;
    // a beam's score, largest logit and log sum of exp(logit - largest): a large
    // common offset of the logits must cancel before the other terms join
    __shared__ double s_score[MAX_BEAMS], s_max[MAX_BEAMS], s_logsum[MAX_BEAMS];
    __shared__ int s_kind[MAX_BEAMS];         // 0 live, 1 finished, 2 no continuation
    __shared__ uint64_t w_val[2][32];
    __shared__ int w_at[2][32];
    const int batch = blockIdx.x, tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const int warps = blockDim.x >> 5;

    for (int l = tid; l < lists; l += blockDim.x) heads[l] = 0;
    for (int k = wid; k < a.beams; k += warps) {
        const int row = batch * a.beams + k;
        const double sc = (double)a.scores[row];
        int kind = a.finished && a.finished[row] ? 1 : 0;
        double top = 0.0, logsum = 0.0;
        if (kind == 0) {
            const float *pm = a.part_max + (int64_t)row * a.splits;
            const float *ps = a.part_sum + (int64_t)row * a.splits;
            float m = -INFINITY;
            for (int i = lane; i < a.splits; i += 32) m = fmaxf(m, pm[i]);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            double s = 0.0;
            for (int i = lane; i < a.splits; i += 32)
                if (ps[i] != 0.0f) s += (double)ps[i] * exp((double)pm[i] - (double)m);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            top = (double)m;
            logsum = log(s);
        }
        if (!isfinite(top) || !isfinite(logsum) || !isfinite(sc)) kind = 2;
        if (lane == 0) {
            s_kind[k] = kind;
            s_score[k] = sc;
            s_max[k] = top;
            s_logsum[k] = logsum;
        }
    }
    __syncthreads();

    // entry `h` of a list: false when it has none
    auto entry = [&](int l, int h, uint64_t &val, int &at) {
        const int k = l / a.splits, sp = l - k * a.splits;
        const int kind = s_kind[k];
        const int flat = k * a.vocab;
        if (kind != 0) {
            // a finished beam continues with the pad token alone; every other
            // token, and all of a beam without continuation, are worth -inf
            if (sp != 0 || h >= a.vocab) return false;
            const int tok = kind == 2 ? h : (h == 0 ? a.pad : h - 1 + (h - 1 >= a.pad));
            val = order_key64(kind == 1 && h == 0 ? s_score[k] : -INFINITY);
            at = flat + tok;
            return true;
        }
        if (h >= a.num) return false;
        const uint64_t e = a.part_list[((int64_t)(batch * a.beams + k) * a.splits + sp) * a.num + h];
        if (e == 0) return false;
        val = order_key64(s_score[k] +
                          (((double)key_value((uint32_t)(e >> 32)) - s_max[k]) - s_logsum[k]));
        at = flat + (int)~(uint32_t)e;
        return true;
    };
    // all entries at once, so that the rounds below wait for no global load
    if (a.staged) {
        for (int i = tid; i < lists * a.num; i += blockDim.x) {
            uint64_t v = 0;
            int at = -1;
            if (!entry(i / a.num, i % a.num, v, at)) at = -1;
            s_val[i] = v;
            s_at[i] = at;
        }
        __syncthreads();
    }
    // few lists: one warp merges, without barriers
    const int active = lists <= 128 ? 1 : warps;
    if (wid >= active) return;
    // this thread's best head over its lists
    uint64_t val;
    int at, which;
    auto refresh = [&]() {
        which = -1;
        val = 0;
        at = INT32_MAX;
        for (int l = tid; l < lists; l += active * 32) {
            uint64_t v = 0;
            int p = -1;
            const int h = heads[l];
            bool has;
            if (a.staged) {
                has = h < a.num;
                if (has) {
                    v = s_val[l * a.num + h];
                    p = s_at[l * a.num + h];
                    has = p >= 0;
                }
            } else {
                has = entry(l, h, v, p);
            }
            if (has && (which < 0 || better(v, p, val, at))) {
                val = v;
                at = p;
                which = l;
            }
        }
    };
    refresh();
    // the n-th best stays with lane n % 32 of the first warp, written when all are known
    uint64_t kept[2] = {0, 0};
    int kept_at[2] = {INT32_MAX, INT32_MAX};
#pragma unroll 1
    for (int n = 0; n < a.num; ++n) {
        uint64_t bv = val;
        int ba = at;
        warp_best(bv, ba);
        if (active > 1) {
            if (lane == 0) { w_val[n & 1][wid] = bv; w_at[n & 1][wid] = ba; }
            __syncthreads();
            bv = lane < active ? w_val[n & 1][lane] : 0;
            ba = lane < active ? w_at[n & 1][lane] : INT32_MAX;
            warp_best(bv, ba);
        }
        if (ba == INT32_MAX) break;           // num <= beams x vocab: not reached
        if (lane == (n & 31)) {
            if (n < 32) { kept[0] = bv; kept_at[0] = ba; }
            else { kept[1] = bv; kept_at[1] = ba; }
        }
        if (at == ba) {                       // the thread that offered it
            ++heads[which];
            refresh();
        }
        __syncwarp();
    }
    if (wid != 0) return;
#pragma unroll
    for (int r = 0; r < MAX_NUM / 32; ++r) {
        const int n = r * 32 + lane;
        if (n >= a.num || kept_at[r] == INT32_MAX) continue;
        const int64_t i = (int64_t)batch * a.num + n;
        a.out_scores[i] = (float)key_value64(kept[r]);
        a.out_parents[i] = kept_at[r] / a.vocab;
        a.out_tokens[i] = kept_at[r] % a.vocab;
    }
}

// ------------------------------------------------------------ state reorder
// Row b K + j of every tensor becomes row b K + parents[b, j], in place: one
// thread holds the same bytes of all K rows of a batch, so it has read every
// source before it writes.  Rows that stay are neither read nor written.  All
// tensors of a call share one launch.  Bound: HBM, the moved rows once each way.
constexpr int MAX_TENSORS = 64;
struct Reorder {
    struct Item { uint8_t *p; int64_t row_bytes; int vec; int block0; } item[MAX_TENSORS];
    int n, beams;
    const int64_t *parents;
};
constexpr int MOVE_THREADS = 128;

template <typename V, int KMAX>
__device__ __forceinline__ void move_rows(uint8_t *p, int64_t row_bytes, int64_t i, int K,
                                          const int *src) {
    const int64_t n = row_bytes / (int64_t)sizeof(V);
    if (i >= n) return;
    V x[KMAX];
#pragma unroll
    for (int j = 0; j < KMAX; ++j)
        if (j < K && src[j] != j) x[j] = reinterpret_cast<const V *>(p + src[j] * row_bytes)[i];
#pragma unroll
    for (int j = 0; j < KMAX; ++j)
        if (j < K && src[j] != j) reinterpret_cast<V *>(p + j * row_bytes)[i] = x[j];
}

template <int KMAX>
__global__ void __launch_bounds__(MOVE_THREADS)
reorder_kernel(const __grid_constant__ Reorder r) {
    __shared__ int src[MAX_BEAMS];
    int t = 0;
    while (t + 1 < r.n && (int)blockIdx.x >= r.item[t + 1].block0) ++t;
    const int64_t row_bytes = r.item[t].row_bytes;
    const int vec = r.item[t].vec, K = r.beams, batch = blockIdx.y;
    if ((int)threadIdx.x < K) {
        // a parent outside the beams leaves its row as it is
        const int64_t s = r.parents[(int64_t)batch * K + threadIdx.x];
        src[threadIdx.x] = s >= 0 && s < K ? (int)s : (int)threadIdx.x;
    }
    __syncthreads();
    uint8_t *p = r.item[t].p + (int64_t)batch * K * row_bytes;
    const int64_t i = (int64_t)((int)blockIdx.x - r.item[t].block0) * MOVE_THREADS + threadIdx.x;
    if (vec == 16) move_rows<uint4, KMAX>(p, row_bytes, i, K, src);
    else if (vec == 4) move_rows<uint32_t, KMAX>(p, row_bytes, i, K, src);
    else if (vec == 2) move_rows<uint16_t, KMAX>(p, row_bytes, i, K, src);
    else move_rows<uint8_t, KMAX>(p, row_bytes, i, K, src);
}

// a row's 16-byte vectors (one more where it may start off a 16-byte boundary) and
// its slices, which share them evenly: a short last slice has no `num` threads of
// its own at a threshold and would have to search for one.  Few rows are cut in
// slices of 16 KB, for more of the SMs (16 rows of 32000 fp32 logits: 4.7 us, in
// slices of up to 64 KB 5.5).
int64_t beam_vecs(int64_t vocab, size_t e) {
    const int64_t vec = 16 / (int64_t)e;
    return ceil_div(vocab + vec - 1, vec);
}
int beam_splits(int64_t rows, int64_t vocab, size_t e) {
    const int64_t n = beam_vecs(vocab, e), fill = 4 * 148;
    const int64_t most = ceil_div(n, SLICE / 2), least = ceil_div(n, SLICE);
    return (int)std::max(least, std::min(most, ceil_div(fill, rows)));
}

}  // namespace
}  // namespace mb2

using namespace mb2;

extern "C" size_t mb2_beam_select_workspace_bytes(int dtype, int64_t batch, int64_t beams,
                                                  int64_t vocab, int64_t num) {
    if (batch <= 0 || beams <= 0 || vocab <= 0 || num <= 0 || vocab > MAX_VOCAB) return 0;
    const size_t lists = (size_t)(batch * beams) * beam_splits(batch * beams, vocab, dtype_size(dtype));
    return lists * ((size_t)num * 8 + 8);
}

extern "C" int mb2_beam_select(int dtype, const void *logits, int64_t batch_stride,
                               int64_t beam_stride, const float *scores, const uint8_t *finished,
                               int64_t pad_token, int64_t batch, int64_t beams, int64_t vocab,
                               int64_t num, float *out_scores, int64_t *out_parents,
                               int64_t *out_tokens, void *workspace, size_t workspace_bytes,
                               mb2_stream_t stream) {
    MB2_REQUIRE(dtype == MB2_F32 || dtype == MB2_BF16, MB2_ERR_ARG, "beam_select: bad dtype");
    MB2_REQUIRE(batch >= 0 && beams > 0 && vocab > 0 && num > 0, MB2_ERR_SHAPE,
                "beam_select: bad size");
    MB2_REQUIRE(beams <= MAX_BEAMS && num <= MAX_NUM && vocab <= MAX_VOCAB, MB2_ERR_SHAPE,
                "beam_select: at most %d beams, %d continuations and a vocabulary of %d",
                MAX_BEAMS, MAX_NUM, MAX_VOCAB);
    MB2_REQUIRE(num <= beams * vocab, MB2_ERR_SHAPE, "beam_select: more continuations than tokens");
    MB2_REQUIRE(pad_token >= 0 && pad_token < vocab, MB2_ERR_SHAPE,
                "beam_select: pad token outside the vocabulary");
    MB2_REQUIRE(batch * beams < 65536, MB2_ERR_SHAPE, "beam_select: batch x beams %lld >= 65536",
                (long long)(batch * beams));
    if (batch == 0) return MB2_OK;
    MB2_REQUIRE(logits && scores && out_scores && out_parents && out_tokens, MB2_ERR_ARG,
                "beam_select: null pointer");
    MB2_REQUIRE(workspace_bytes >= mb2_beam_select_workspace_bytes(dtype, batch, beams, vocab, num) &&
                    workspace,
                MB2_ERR_WORKSPACE, "beam_select: workspace too small");
    MB2_REQUIRE(aligned(workspace, 8), MB2_ERR_ALIGN, "beam_select: misaligned workspace");
    const int splits = beam_splits(batch * beams, vocab, dtype_size(dtype));
    const int64_t rows = batch * beams;
    RowArgs r;
    r.logits = logits;
    r.s_batch = batch_stride;
    r.s_beam = beam_stride;
    r.beams = (int)beams; r.vocab = (int)vocab; r.num = (int)num; r.splits = splits;
    r.per = (int)ceil_div(beam_vecs(vocab, dtype_size(dtype)), splits);
    r.finished = finished;
    r.part_list = static_cast<uint64_t *>(workspace);
    r.part_max = reinterpret_cast<float *>(r.part_list + rows * splits * num);
    r.part_sum = r.part_max + rows * splits;
    cudaStream_t st = (cudaStream_t)stream;
    const dim3 grid((unsigned)splits, (unsigned)rows);
    if (dtype == MB2_F32) beam_rows_kernel<float><<<grid, ROW_THREADS, 0, st>>>(r);
    else beam_rows_kernel<__nv_bfloat16><<<grid, ROW_THREADS, 0, st>>>(r);
    MB2_TRY(check_launch("beam_rows_kernel"));
    MergeArgs g;
    g.beams = r.beams; g.vocab = r.vocab; g.num = r.num; g.splits = splits;
    g.pad = (int)pad_token;
    g.scores = scores;
    g.finished = finished;
    g.part_max = r.part_max; g.part_sum = r.part_sum; g.part_list = r.part_list;
    g.out_scores = out_scores; g.out_parents = out_parents; g.out_tokens = out_tokens;
    const int lists = (int)beams * splits;
    // at most 32 x 2^20 candidates a batch: flat indices are 32-bit
    const int threads = lists <= 256 ? 256 : lists <= 512 ? 512 : 1024;
    const size_t staged = (size_t)lists * num * 12 + sizeof(int) * (size_t)lists;
    g.staged = staged <= MERGE_STAGE;
    beam_merge_kernel<<<(unsigned)batch, threads, g.staged ? staged : sizeof(int) * lists, st>>>(g);
    return check_launch("beam_merge_kernel");
}

extern "C" int mb2_reorder_rows(void *const *tensors, const int64_t *row_bytes, int64_t n_tensors,
                                const int64_t *parents, int64_t batch, int64_t beams,
                                mb2_stream_t stream) {
    MB2_REQUIRE(n_tensors >= 0 && batch >= 0 && beams > 0, MB2_ERR_SHAPE, "reorder_rows: bad size");
    MB2_REQUIRE(beams <= MAX_BEAMS, MB2_ERR_SHAPE, "reorder_rows: at most %d beams", MAX_BEAMS);
    MB2_REQUIRE(batch < 65536, MB2_ERR_SHAPE, "reorder_rows: batch %lld >= 65536", (long long)batch);
    if (n_tensors == 0 || batch == 0) return MB2_OK;
    MB2_REQUIRE(tensors && row_bytes && parents, MB2_ERR_ARG, "reorder_rows: null pointer");
    for (int64_t i = 0; i < n_tensors; ++i)
        MB2_REQUIRE(row_bytes[i] >= 0 && (tensors[i] || row_bytes[i] == 0), MB2_ERR_ARG,
                    "reorder_rows: bad tensor %lld", (long long)i);
    try {
        // moved in place side by side: no byte may belong to two tensors
        std::vector<std::pair<const uint8_t *, int64_t>> spans;
        spans.reserve((size_t)n_tensors);
        for (int64_t i = 0; i < n_tensors; ++i)
            if (row_bytes[i])
                spans.emplace_back(static_cast<const uint8_t *>(tensors[i]),
                                   row_bytes[i] * batch * beams);
        std::sort(spans.begin(), spans.end());
        for (size_t i = 1; i < spans.size(); ++i)
            MB2_REQUIRE(spans[i].first - spans[i - 1].first >= spans[i - 1].second, MB2_ERR_ARG,
                        "reorder_rows: tensors overlap");
    } catch (const std::exception &e) {           // no exception leaves a C entry
        return fail(MB2_ERR_UNSUPPORTED, "reorder_rows: %lld tensors: %s", (long long)n_tensors,
                    e.what());
    }
    for (int64_t t0 = 0; t0 < n_tensors; t0 += MAX_TENSORS) {
        Reorder r;
        r.n = 0;
        r.beams = (int)beams;
        r.parents = parents;
        int64_t blocks = 0;
        for (int64_t i = t0; i < n_tensors && i < t0 + MAX_TENSORS; ++i) {
            const int64_t rb = row_bytes[i];
            if (rb == 0) continue;
            int vec = 16;
            while (vec > 1 && (rb % vec || !aligned(tensors[i], vec))) vec = vec == 16 ? 4 : vec / 2;
            r.item[r.n].p = static_cast<uint8_t *>(tensors[i]);
            r.item[r.n].row_bytes = rb;
            r.item[r.n].vec = vec;
            r.item[r.n].block0 = (int)blocks;
            ++r.n;
            blocks += ceil_div(rb / vec, MOVE_THREADS);
            MB2_REQUIRE(blocks <= 0x7fffffff, MB2_ERR_SHAPE, "reorder_rows: rows too long");
        }
        if (blocks == 0) continue;
        const dim3 grid((unsigned)blocks, (unsigned)batch);
        cudaStream_t st = (cudaStream_t)stream;
        if (beams <= 4) reorder_kernel<4><<<grid, MOVE_THREADS, 0, st>>>(r);
        else if (beams <= 8) reorder_kernel<8><<<grid, MOVE_THREADS, 0, st>>>(r);
        else if (beams <= 16) reorder_kernel<16><<<grid, MOVE_THREADS, 0, st>>>(r);
        else reorder_kernel<32><<<grid, MOVE_THREADS, 0, st>>>(r);
        MB2_TRY(check_launch("reorder_kernel"));
    }
    return MB2_OK;
}
