// Decay attention over prompts on the tensor cores (bf16): chunks of 128 tokens,
// one CTA walking the chunks of a (sequence, head, 64 columns of v) with the
// state S (Dk x 64) in fp32 in TMEM.  Within a chunk, with G_i the sum of the
// log decays up to token i and S0 the state before it,
//   P_ij = e^{G_i - G_j} (q_i . k_j)  for j <= i, else 0
//   o_i  = scale (sum_j P_ij v_j + e^{G_i} q_i^T S0)      (scale joins P's factors)
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
// Operands: P and S0 are two bf16 parts each (16 bits: 2^-16 of a term, so an output's
// error is that of its own rounding, 1.66e-3 rms of 1.66e-3; with one part each it was
// 2.3e-3, and 8 sequences of 8192 tokens took 306 us instead of 357).  V~ is three
// (24 bits), because the state is an fp32 output and lives for many chunks.  An
// infinity stands in the first part alone.
//
// Room: S0's second part lies in the second half of the q stage of the chunk before,
// which Q K^T and Q S0 have read and the output rows leave free; the next q waits for
// the Q S0 that reads it.  (In the k stage or the v stage the next chunk's K^T V~ waits
// for it too: 412 and 478 us.)  P replaces its scores in TMEM.
//
// Causality with infinities and NaN: a masked P_ij is 0, but 0 * inf = NaN, so a
// row whose P V comes out non-finite is computed again from its own tokens alone (in
// the chunk that holds them; a state that is not finite costs later chunks nothing).
// K^T V~ splits an infinity into an infinity and NaN: such a chunk's state is taken
// token by token.  So states are those of the recurrence, infinities with their signs
// (until decays that sum below -104 in a chunk: 0 * inf), and so are the outputs that
// meet them, but for a q or a v that is infinite itself (its terms have both signs, or
// a padded row's 0: infinite or NaN).
//
// Roles (28 warps): 0-7 the state, 8-15 P, 16-19 the output rows, 20-23 V~, 24
// decays (its scheduler has the least of P's triangle), 25 TMA loads, 26 and 27 MMA
// issue.  One MMA warp issues P V (n), Q K^T (n + 1), the other K^T V~ (n), Q S0 (n),
// each as soon as its operands are there.  Every
// mbarrier completes once per chunk (staged ones once per two), so its phase
// follows from the chunk count.  All waits are bounded; a wait that expires sets
// the device status.
//
// Bound: neither bytes nor MMAs (2700 cycles a chunk) but the chain of hand-overs
// between the roles, about 5200 cycles = 2.7 us a chunk with 128-wide q and k, one
// CTA an SM (shared memory and TMEM are full): Q K^T 1400 with the wait for q, P 2500
// (its scheduler's FMA and ALU pipes, shared with V~ and the state), P V 900, the rest
// from one to the next.  What brought it there, at 8
// sequences of 8192 tokens, 24 heads of 128 x 64 (1.5 us of HBM time a chunk), with
// P and S0 in one part:
//   733 us  one role after the other, the state in registers
//   411     a short loop over 16-column pieces per role instead of straight-line
//           code, the state in TMEM: five roles share each scheduler's instruction
//           cache, and half of all issue slots waited for instructions
//   336     output rows through shared memory and TMA: 32 rows a store instruction
//           blocked the load/store unit for everyone
//   327     MMA descriptors provably uniform (else every MMA moves six operands
//           into uniform registers first)
//   303     two MMA warps, eight warps for the state, P's factors before its scores,
//           tiles fetched into L2 a chunk ahead
#include <cuda.h>
#include <cudaTypedefs.h>

#include "decay.cuh"
#include "tc_prims.cuh"

namespace mb2 {
namespace decay {

using namespace tc;

constexpr int C = 128;                       // tokens per chunk
constexpr int DV = 64;                       // columns of v per CTA
// first warp of each role: the state (8 warps), P (8), output rows, V~, MMA (2), TMA,
// decays
constexpr int W_P = 8, W_O = 16, W_V = 20, W_MMA = 26, W_TMA = 25, W_G = 24;
constexpr int THREADS = 28 * 32;
constexpr uint32_t SUB = 128 * 128;          // one 128-row x 128-byte operand tile
// shared memory (bytes from a 1024-aligned base)
constexpr uint32_t OFF_Q = 0;                            // [2][2 SUB]
constexpr uint32_t OFF_K = OFF_Q + 4 * SUB;              // [2][2 SUB]
constexpr uint32_t OFF_V = OFF_K + 4 * SUB;              // [2][SUB]
constexpr uint32_t OFF_VT = OFF_V + 2 * SUB;             // [3][SUB]
constexpr uint32_t OFF_H = OFF_VT + 3 * SUB;             // [SUB]: S0's first part
// S0's second part, of chunk c: where the second half of q of chunk c - 1 was
__device__ __forceinline__ uint32_t off_h2(uint32_t c) { return OFF_Q + ((c & 1) ^ 1) * 2 * SUB + SUB; }
constexpr uint32_t OFF_COLF = OFF_H + SUB;               // float [2][128]
constexpr uint32_t OFF_G2 = OFF_COLF + 2 * C * 4;        // float [2][128]
constexpr uint32_t OFF_SC = OFF_G2 + 2 * C * 4;          // float [2][16]
constexpr uint32_t OFF_DEC = OFF_SC + 2 * 16 * 4;        // float [4]
constexpr uint32_t OFF_CHUNK = OFF_DEC + 4 * 4;          // Chunk [4]
constexpr uint32_t OFF_BARS = OFF_CHUNK + 4 * 3 * 16;
constexpr int NBARS = 6 + 6 + 4 + 9 + 2 + 6;
constexpr uint32_t OFF_TMEM = OFF_BARS + NBARS * 8;
constexpr uint32_t SMEM_BYTES = OFF_TMEM + 16;
// scalars of a chunk (OFF_SC), all e^sums of whole blocks' decays
constexpr int SC_BEFORE = 0;     // [4] blocks before block w
constexpr int SC_AFTER = 4;      // [4] blocks after it
constexpr int SC_ALL = 8;        // the chunk
constexpr int SC_1 = 9, SC_12 = 10, SC_2 = 11;   // block 1; blocks 1 and 2; block 2
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory");
// TMEM columns
// (P takes the place of the scores: of every 16 tokens 8 columns of its first part, 8
// of its second.  T_QH: Q times S0's second part, then its first; T_D: K^T V~ of V~'s
// first part, then of the other two)
constexpr uint32_t T_S = 0, T_PV = 128, T_QH = 192, T_D = 320, T_H = 448;

// UMMA descriptor of an MN-major operand, 128-byte swizzle: rows are the
// contraction index (128 bytes of 64 MN elements each), 8-row groups 1024 B
// apart, further 64-element MN atoms `next` bytes apart.
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t addr, uint32_t next = SUB) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(next >> 4) << 16) |
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
__device__ __forceinline__ void tmem_ld8_async(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                   "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}
// waits for the loads into r: the registers pass through, so that no use of
// them can be scheduled before the wait
template <int N>
__device__ __forceinline__ void tmem_loaded(uint32_t (&r)[N]) {
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
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
__device__ __forceinline__ void tma_prefetch_4d(const CUtensorMap *map, int32_t x, int32_t head,
                                                int32_t tok, int32_t b) {
    asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global [%0, {%1, %2, %3, %4}];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(head), "r"(tok), "r"(b)
                 : "memory");
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap *map, uint32_t src, int32_t x,
                                             int32_t head, int32_t tok, int32_t b) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(src), "r"(x), "r"(head), "r"(tok), "r"(b)
                 : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;"); }
__device__ __forceinline__ void bulk_wait_read0() {
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}
__device__ __forceinline__ void bulk_wait0() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t pack_bf16(uint64_t v) {
    return pack_bf16(__uint_as_float(lo_of(v)), __uint_as_float(hi_of(v)));
}
// a bf16 pair as two fp32 values
__device__ __forceinline__ uint64_t unpack_bf16(uint32_t v) { return pair(v << 16, v & 0xffff0000u); }
// what a rounding to bf16 left behind (exact)
__device__ __forceinline__ uint64_t rest(uint64_t x, uint32_t rounded) {
    return fma2(unpack_bf16(rounded), pair(-1.0f), x);
}
// bad becomes NaN where v holds an infinity or NaN, else stays 0
__device__ __forceinline__ void poison(uint32_t &bad, uint32_t v) {
    asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(bad) : "r"(v), "r"(0));
}
// 0 for infinities and NaN
__device__ __forceinline__ uint32_t finite(uint32_t v) {
    if ((v & 0x7f80u) == 0x7f80u) v &= 0xffff0000u;
    if ((v & 0x7f800000u) == 0x7f800000u) v &= 0xffffu;
    return v;
}

// e^x of a 64-bit sum, to fp32 precision
__device__ __forceinline__ float exp_of(double x) {
    const float hi = (float)x;
    const float e = expf(hi);
    const float lo = (float)(x - (double)hi);
    return e == 0.0f || hi != hi ? e : fmaf(e, lo, e);
}

// An item of work: a span (32-bit: tokens and spans are below 2^31) x head x tile.
struct Item {
    int tile, h, seq, row0, len, in, out;
};
template <bool STATE>
__device__ __forceinline__ Item item_of(const Args &a, uint32_t tiles, uint32_t id) {
    Item it;
    const uint32_t n = id / tiles, heads = (uint32_t)a.heads, span = n / heads;
    it.tile = (int)(id - n * tiles);
    it.h = (int)(n - span * heads);
    const int len = (int)a.seqlen, seg = (int)a.seg;
    int seq = (int)span, j = 0, segs = 1;
    if (seg > 0) {
        if (a.cu) {
            int hi = (int)a.seqs;         // the last sequence whose first slot is <= span
            seq = 0;
            while (hi - seq > 1) {
                const int mid = (seq + hi) >> 1;
                if (a.slot0[mid] <= (int)span) seq = mid;
                else hi = mid;
            }
            j = (int)span - a.slot0[seq];
            segs = a.slot0[seq + 1] - a.slot0[seq];
        } else {
            segs = len > seg ? (int)((uint32_t)(len + seg - 1) / (uint32_t)seg) : 1;
            seq = (int)(span / (uint32_t)segs);
            j = (int)span - seq * segs;
        }
    }
    it.seq = seq;
    it.row0 = 0;
    it.len = len;
    if (a.cu) {
        const int b = a.cu[seq], e = a.cu[seq + 1];
        it.row0 = b < 0 ? 0 : b > len ? len : b;
        it.len = (e > len ? len : e) - it.row0;
        if (it.len < 0) it.len = 0;
    }
    it.in = a.h0 ? seq : -1;
    it.out = a.h_last ? seq : -1;
    if (seg > 0) {
        const bool last = j == segs - 1, valid = j < segs && (!STATE || !last);
        it.row0 += j * seg;
        it.len = it.len - j * seg < seg ? it.len - j * seg : seg;
        if (!valid || it.len < 0) it.len = 0;
        it.in = STATE ? -1 : (int)span;
        it.out = !valid ? -1 : STATE ? (int)span : last ? it.out : -1;
    }
    return it;
}
// A chunk as the roles see it, in shared memory beside its decays: one warp walks
// the items, the others read.
struct alignas(16) Chunk {
    int row, m;                          // first token (of the batch row), tokens; m 0: the end
    int first, last;                     // of its span
    int h, batch, tile;
    int in, out;                         // Span's
};
// the chunks of a CTA's items, in order; items without tokens go to `empty`
template <bool STATE> struct Walk {
    Item it;
    int t0 = 0;
    uint32_t id = blockIdx.x - gridDim.x;
    __device__ __forceinline__ Walk() { it.len = 0; }
    template <typename F>
    __device__ __forceinline__ bool next(const Args &a, uint32_t tiles, uint32_t items, F empty) {
        t0 += C;
        if (t0 < it.len) return true;
        t0 = 0;
        for (;;) {
            id += gridDim.x;
            if (id >= items) return false;
            it = item_of<STATE>(a, tiles, id);
            if (it.len > 0) return true;
            empty();
        }
    }
};
// g of token t of an item (0 behind its end)
__device__ __forceinline__ float load_g(const Args &a, const Item &it, int t) {
    if (t >= it.len) return 0.0f;
    return a.g[(a.cu ? 0 : it.seq) * a.gs[0] + (int64_t)(it.row0 + t) * a.gs[1] + it.h * a.gs[2]];
}
// below -256, e^g is 0 for every fp32 product, and a finite sum keeps later
// differences; NaN stays
__device__ __forceinline__ float clamp_g(float g) { return g < -256.0f ? -256.0f : g; }

// Bounded waits: about 20 cycles a try, 2^27 tries.  (A try_wait with a time hint
// sleeps instead of polling, but wakes later; polling by one lane takes 400 cycles a
// hand-over instead of 170.)
__device__ __forceinline__ bool wait_one(uint32_t bar, uint32_t parity, int where) {
    uint32_t ok, tries = 0;
    do {
        ok = mbar_try(bar, parity);
    } while (!ok && ++tries < (1u << 27));
    if (!ok) atomicCAS(&g_mb2_device_error, 0, where);
    return ok != 0;
}
// of a whole warp; every lane gets the same answer
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, int where) {
    return __all_sync(0xffffffffu, wait_one(bar, parity, where));
}

// a row of `tiles` operand tiles
__device__ __forceinline__ void zero_row(uint8_t *row, int tiles) {
#pragma unroll 1
    for (int i = 0; i < 8 * tiles; ++i)
        *reinterpret_cast<uint4 *>(row + (i >> 3) * SUB + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
}

// The output rows of a warp (`row0` .. row0 + 31 of the chunk) whose P V met an infinity
// or a NaN, perhaps in a later token's v: their own tokens' share again, from global
// memory.  The whole warp takes one row after the other: a lane the scores of four
// tokens, then two columns of v.  `base`: 16 rows of 64 fp32, what P V is added to; redo:
// the rows (a bit each) that get it.
__device__ __forceinline__ double prefix_sum(double x, int lane) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
    }
    return x;
}
__device__ __noinline__ void masked_rows(const Args &a, const Chunk &k, int row0, uint32_t redo,
                                         const float *base) {
    const int lane = threadIdx.x & 31;
    const int64_t bq = k.batch;
    const __nv_bfloat16 *const q = static_cast<const __nv_bfloat16 *>(a.q) + bq * a.qs[0] +
                                   (k.h / a.q_rep) * a.qs[2];
    const __nv_bfloat16 *const kk = static_cast<const __nv_bfloat16 *>(a.k) + bq * a.ks[0] +
                                    (int64_t)k.row * a.ks[1] + (k.h / a.k_rep) * a.ks[2];
    const __nv_bfloat16 *const v = static_cast<const __nv_bfloat16 *>(a.v) + bq * a.vs[0] +
                                   (int64_t)k.row * a.vs[1] + (k.h / a.v_rep) * a.vs[2] + k.tile * DV;
    const float *const g = a.g + bq * a.gs[0] + (int64_t)k.row * a.gs[1] + k.h * a.gs[2];
    __nv_bfloat16 *const o = static_cast<__nv_bfloat16 *>(a.o) + bq * a.os[0] + k.h * a.os[2] + k.tile * DV;
    const int cols = (int)(a.dv - k.tile * DV < DV ? a.dv - k.tile * DV : DV);
    double sum[4];                       // of g up to token 32 t + lane
    double before = 0.0;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int j = 32 * t + lane;
        sum[t] = before + prefix_sum(j < k.m ? (double)clamp_g(g[j * a.gs[1]]) : 0.0, lane);
        before = __shfl_sync(0xffffffffu, sum[t], 31);
    }
#pragma unroll 1
    for (int n = 0; n < 16 && row0 + n < k.m; ++n) {
        const int r = row0 + n;
        float y0 = base[64 * n + lane], y1 = base[64 * n + 32 + lane];
        if (redo >> n & 1) {
            double at = 0.0;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const double x = __shfl_sync(0xffffffffu, sum[t], r & 31);
                if (t == r >> 5) at = x;
            }
            const uint4 *const qr = reinterpret_cast<const uint4 *>(q + (int64_t)(k.row + r) * a.qs[1]);
            float add0 = 0.0f, add1 = 0.0f;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int j = 32 * t + lane;
                float p = 0.0f;
                if (j <= r) {
                    const uint4 *const kr = reinterpret_cast<const uint4 *>(kk + j * a.ks[1]);
#pragma unroll 1
                    for (int e = 0; e < (int)a.dk / 8; ++e) {
                        const uint4 x = qr[e], y = kr[e];
                        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            p = fmaf(__uint_as_float(xs[i] << 16), __uint_as_float(ys[i] << 16), p);
                            p = fmaf(__uint_as_float(xs[i] & 0xffff0000u),
                                     __uint_as_float(ys[i] & 0xffff0000u), p);
                        }
                    }
                    p *= expf((float)(at - sum[t])) * a.scale;
                }
#pragma unroll 1
                for (int i = 0; i < 32 && 32 * t + i <= r; ++i) {
                    const float pj = __shfl_sync(0xffffffffu, p, i);
                    const __nv_bfloat16 *const vj = v + (32 * t + i) * a.vs[1];
                    if (lane < cols) add0 = fmaf(pj, __bfloat162float(vj[lane]), add0);
                    if (32 + lane < cols) add1 = fmaf(pj, __bfloat162float(vj[32 + lane]), add1);
                }
            }
            y0 += add0;
            y1 += add1;
        }
        __nv_bfloat16 *const to = o + (int64_t)(k.row + r) * a.os[1];
        if (lane < cols) to[lane] = __float2bfloat16_rn(y0);
        if (32 + lane < cols) to[32 + lane] = __float2bfloat16_rn(y1);
    }
}

// 16 columns from `col` of row r of the state (at `taddr`) over a chunk's tokens, by the
// recurrence
__device__ __forceinline__ void walk_state(const Args &a, const Chunk &k, int r, int col, uint32_t taddr) {
    uint32_t h[16];
    tmem_ld16_async(taddr, h);
    tmem_loaded(h);
    const int64_t bq = k.batch;
    const __nv_bfloat16 *kk = static_cast<const __nv_bfloat16 *>(a.k) + bq * a.ks[0] +
                              (int64_t)k.row * a.ks[1] + (k.h / a.k_rep) * a.ks[2] + r;
    const __nv_bfloat16 *v = static_cast<const __nv_bfloat16 *>(a.v) + bq * a.vs[0] +
                             (int64_t)k.row * a.vs[1] + (k.h / a.v_rep) * a.vs[2] + k.tile * DV + col;
    const float *g = a.g + bq * a.gs[0] + (int64_t)k.row * a.gs[1] + k.h * a.gs[2];
    const int cols = (int)(a.dv - k.tile * DV - col);
#pragma unroll 1
    for (int t = 0; t < k.m; ++t) {
        const float f = expf(*g), x = r < a.dk ? __bfloat162float(*kk) : 0.0f;
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (j < cols)
                h[j] = __float_as_uint(fmaf(f, __uint_as_float(h[j]), x * __bfloat162float(v[j])));
        kk += a.ks[1];
        v += a.vs[1];
        g += a.gs[1];
    }
    __syncwarp();
    tmem_st16(taddr, h);
    tmem_wait_st();
}

// STATE: the pass over segments that leaves their states; no Q, no outputs
template <bool STATE>
__global__ void __launch_bounds__(THREADS, 1)
decay_chunk_kernel(const __grid_constant__ CUtensorMap map_q,
                   const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v,
                   const __grid_constant__ CUtensorMap map_o, const __grid_constant__ Args a,
                   uint32_t tiles, uint32_t items) {
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t base = smem_u32(smem);
    float *const colf = reinterpret_cast<float *>(smem + OFF_COLF);
    float *const g2 = reinterpret_cast<float *>(smem + OFF_G2);
    float *const sc = reinterpret_cast<float *>(smem + OFF_SC);
    // e^{G_C}, four deep: the state's warps read it after the outputs of their
    // chunk may already have freed its other decays
    float *const dec = reinterpret_cast<float *>(smem + OFF_DEC);
    // the chunks, four deep for the same reason
    Chunk *const chunks = reinterpret_cast<Chunk *>(smem + OFF_CHUNK);
    uint32_t *const tmem_slot = reinterpret_cast<uint32_t *>(smem + OFF_TMEM);
    auto bar = [&](int i) { return base + OFF_BARS + 8u * i; };
    auto full_q = [&](int s) { return bar(s); };
    auto full_k = [&](int s) { return bar(2 + s); };
    auto full_v = [&](int s) { return bar(4 + s); };
    auto empty_q = [&](int s) { return bar(6 + s); };
    auto empty_k = [&](int s) { return bar(8 + s); };
    auto empty_v = [&](int s) { return bar(10 + s); };
    auto g_full = [&](int s) { return bar(12 + s); };    // a chunk's decays in shared memory
    auto g_free = [&](int s) { return bar(14 + s); };    // ... read
    const uint32_t s_full = bar(16);    // Q K^T in TMEM
    const uint32_t vt_full = bar(17);   // V~ in shared memory
    const uint32_t d_full = bar(18);    // K^T V~ in TMEM, V~ read
    const uint32_t d_free = bar(19);    // ... read
    const uint32_t h_full = bar(20);    // S0 (bf16) in shared memory
    const uint32_t h_free = bar(21);    // ... read
    const uint32_t p_full = bar(22);    // P in TMEM, S read
    const uint32_t o_full = bar(23);    // P V and Q S0 in TMEM, P read
    const uint32_t o_free = bar(24);    // ... read
    const uint32_t drain = bar(25);     // [2] a warp's MMAs complete (once, at the end)
    // V in shared memory with its tail zeroed, V~ made; by stage, since V~ may be a chunk
    // ahead of P V (vt_full would then be in its next phase)
    auto v_full = [&](int s) { return bar(27 + s); };
    auto k_tail = [&](int s) { return bar(29 + s); };    // K's rows behind the end zeroed
    auto q_read = [&](int s) { return bar(31 + s); };    // Q K^T has read Q

    // through a shuffle, so that the compiler knows it to be one value a warp
    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const bool wide = a.dk > 64;                         // two 64-column operand tiles
    if (threadIdx.x == 0) {
        for (int i = 0; i < NBARS; ++i) {
            const int n = (i == 6 || i == 7) ? 4 :       // empty_q
                          (i == 8 || i == 9) ? (STATE ? 1 : 2) :   // empty_k
                          (i == 10 || i == 11) ? (STATE ? 128 : 1) :   // empty_v
                          (i == 12 || i == 13) ? 32 :    // g_full
                          (i == 14 || i == 15) ? (STATE ? 256 : 384) :   // g_free
                          i == 23 ? 2 :                  // o_full
                          (i == 17 || i == 24 || (i >= 27 && i < 31)) ? 128 :   // vt_full, o_free, v_full, k_tail
                          (i == 19 || i == 20 || i == 22) ? 256 : 1;   // d_free, h_full, p_full
            mbar_init(bar(i), n);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == W_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(base + OFF_TMEM), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = uniform(*tmem_slot);

    if (warp == W_TMA) {
        // -------------------------------------------------------- TMA loads
        if (lane == 0) {
            Walk<STATE> k;
            const uint32_t qk = wide ? 2 * SUB : SUB;
            uint32_t nk = 0, nq = 0, nv = 0;             // loads issued
#pragma unroll 1
            for (uint32_t c = 0; k.next(a, tiles, items, [] {}); ++c) {
                const int s = c & 1;
                const uint32_t ph = ((c >> 1) & 1) ^ 1;
                const int tok = k.it.row0 + k.t0, bq = a.cu ? 0 : k.it.seq;
                const int hq = k.it.h / a.q_rep, hk = k.it.h / a.k_rep, hv = k.it.h / a.v_rep;
                const uint32_t dk = base + OFF_K + s * 2 * SUB, dq = base + OFF_Q + s * 2 * SUB;
                if (!wait_one(empty_k(s), ph, 0x401)) break;
                mbar_expect_tx(full_k(s), qk);
                tma_load_4d(dk, &map_k, full_k(s), 0, hk, tok, bq);
                if (wide) tma_load_4d(dk + SUB, &map_k, full_k(s), 64, hk, tok, bq);
                ++nk;
                if (!wait_one(empty_v(s), ph, 0x403)) break;
                mbar_expect_tx(full_v(s), SUB);
                tma_load_4d(base + OFF_V + s * SUB, &map_v, full_v(s), k.it.tile * DV, hv, tok, bq);
                ++nv;
                if (STATE) continue;
                // the stage held output rows (c - 2) and S0 (c - 1)'s second part
                if (!wait_one(empty_q(s), ph, 0x402) || !wait_one(h_free, s ^ 1, 0x402)) break;
                mbar_expect_tx(full_q(s), qk);
                tma_load_4d(dq, &map_q, full_q(s), 0, hq, tok, bq);
                if (wide) tma_load_4d(dq + SUB, &map_q, full_q(s), 64, hq, tok, bq);
                ++nq;
            }
            // no load is in flight when the CTA ends (its consumers may have given up)
            auto land = [&](auto full, uint32_t n) {
                for (uint32_t i = n > 2 ? n - 2 : 0; i < n; ++i) wait_one(full(i & 1), (i >> 1) & 1, 0x404);
            };
            land(full_k, nk);
            land(full_q, nq);
            land(full_v, nv);
        }
        __syncwarp();
    } else if (warp == W_MMA || warp == W_MMA + 1) {
        // -------------------------------------------------------- MMA issue
        // The whole warp walks the chunks and one lane issues: descriptors and loop
        // are then provably one value a warp and stay in uniform registers, where
        // an MMA wants them.
        const uint64_t dq0 = smem_desc(base + OFF_Q), dk0 = smem_desc(base + OFF_K);
        const uint64_t kt0 = smem_desc_mn(base + OFF_K), v0 = smem_desc_mn(base + OFF_V);
        const uint64_t vt0 = smem_desc_mn(base + OFF_VT);
        constexpr uint64_t STAGE = 2 * SUB >> 4, ROWS16 = 2048 >> 4;
        const int steps = wide ? 8 : 4;                  // of 16 columns of q and k
        bool ok = true;
        if (STATE && warp == W_MMA) {
        } else if (warp == W_MMA) {
            // iteration n: P V of chunk n - 1, Q K^T of chunk n
#pragma unroll 1
            for (uint32_t n = 0, more = 1; more && ok; ++n) {
                const uint32_t s = n & 1, ph2 = (n >> 1) & 1;
                ok = wait_warp(g_full(s), ph2, 0x410);
                more = ok ? uniform(chunks[n & 3].m) : 0;
                if (more) {
                    ok = ok && wait_warp(full_k(s), ph2, 0x411);
                    if (more < C) ok = ok && wait_warp(k_tail(s), ph2, 0x41a);
                }
                if (n > 0) {
                    const uint32_t ph = (n - 1) & 1;
                    const uint64_t v = v0 + ph * (SUB >> 4);
                    ok = ok && wait_warp(o_free, ph ^ 1, 0x416) &&
                         wait_warp(v_full(ph), ((n - 1) >> 1) & 1, 0x419) &&
                         wait_warp(p_full, ph, 0x417);
                    fence_after();
                    if (ok && elect_one()) {
#pragma unroll 2
                        for (int i = 0; i < C / 16; ++i) {
                            mma_ts_bf16(tmem + T_PV, tmem + T_S + i * 16 + 8, v + i * ROWS16,
                                        idesc(64, false, true), i != 0);
                            mma_ts_bf16(tmem + T_PV, tmem + T_S + i * 16, v + i * ROWS16,
                                        idesc(64, false, true), 1);
                        }
                        mma_commit(o_full);
                        mma_commit(empty_v(ph));
                    }
                    __syncwarp();
                }
                if (more) {
                    const uint64_t q = dq0 + s * STAGE, k = dk0 + s * STAGE;
                    ok = ok && wait_warp(full_q(s), ph2, 0x412);
                    // the scores' columns hold P until P V has read it
                    if (n > 0) ok = ok && wait_warp(empty_v(s ^ 1), ((n - 1) >> 1) & 1, 0x41c);
                    fence_after();
                    if (ok && elect_one()) {
#pragma unroll 2
                        for (int i = 0; i < steps; ++i) {
                            const uint64_t off = (i >> 2) * (SUB >> 4) + (i & 3) * 2;
                            mma_ss(tmem + T_S, q + off, k + off, idesc(128, false, false), i != 0);
                        }
                        mma_commit(s_full);
                        mma_commit(empty_k(s));
                        mma_commit(q_read(s));
                    }
                    __syncwarp();
                }
            }
        } else {
            // K^T V~, then Q S0 of each chunk
#pragma unroll 1
            for (uint32_t n = 0; ok; ++n) {
                const uint32_t s = n & 1, ph2 = (n >> 1) & 1;
                ok = wait_warp(g_full(s), ph2, 0x410);
                if (!ok || !uniform(chunks[n & 3].m)) break;
                const uint64_t q = dq0 + s * STAGE, kt = kt0 + s * STAGE;
                // S0's second part and, behind it, its first
                const uint64_t h = smem_desc_mn(base + off_h2(s), OFF_H - off_h2(s));
                // (behind Q K^T, which P is waiting for: side by side they take twice as long)
                ok = (STATE || wait_warp(q_read(s), ph2, 0x41d)) && wait_warp(vt_full, s, 0x413) &&
                     wait_warp(full_k(s), ph2, 0x414) && wait_warp(d_free, s ^ 1, 0x414);
                fence_after();
                if (ok && elect_one()) {
                    // V~'s first two parts side by side, the third added to the second's
#pragma unroll 1
                    for (int i = 0; i < C / 16; ++i) {
                        mma_ss(tmem + T_D, kt + i * ROWS16, vt0 + i * ROWS16, idesc(128, true, true),
                               i != 0);
                        mma_ss(tmem + T_D + 64, kt + i * ROWS16, vt0 + (2 * SUB >> 4) + i * ROWS16,
                               idesc(64, true, true), 1);
                    }
                    mma_commit(d_full);
                    mma_commit(empty_k(s));
                }
                __syncwarp();
                if (STATE) continue;
                ok = ok && wait_warp(h_full, s, 0x415) && wait_warp(full_q(s), ph2, 0x412) &&
                     wait_warp(o_free, s ^ 1, 0x416);
                fence_after();
                if (ok && elect_one()) {
#pragma unroll 2
                    for (int i = 0; i < steps; ++i)
                        mma_ss(tmem + T_QH, q + (i >> 2) * (SUB >> 4) + (i & 3) * 2, h + i * ROWS16,
                               idesc(128, false, true), i != 0);
                    mma_commit(h_free);
                    mma_commit(o_full);
                }
                __syncwarp();
            }
        }
        if (elect_one()) {
            const uint32_t mine = drain + 8 * (warp - W_MMA);
            mma_commit(mine);                            // before TMEM is given back
            wait_one(mine, 0, 0x418);
        }
        __syncwarp();
    } else if (warp == W_G) {
        // ----------------------------------------------------------- decays
        // lane l: tokens 4 l .. 4 l + 3; lanes 8 b .. 8 b + 7 are block b
        Walk<STATE> k;
        Chunk now = {};
        float gnow[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        double span_g = 0.0;                             // of the span so far
        bool more = true;
        // iteration c: chunk c's loads, then the decays of chunk c - 1; the end is a
        // chunk without tokens
#pragma unroll 1
        for (uint32_t n = 0;; ++n) {
            const uint32_t c = n - 1;
            const int s = c & 1;
            Chunk next = {};
            float gn[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (more)
                more = k.next(a, tiles, items, [&] {
                    // a span without tokens keeps its state
                    if (STATE || k.it.out < 0) return;
                    const int64_t per = a.heads * a.dk * a.dv, at = k.it.h * a.dk * a.dv;
                    const float *const hin = (a.seg ? a.seg_state : a.h0) + k.it.in * per + at;
                    float *const hout = a.h_last + k.it.out * per + at;
#pragma unroll 1
                    for (int i = lane; i < (int)a.dk * DV; i += 32) {
                        const int col = k.it.tile * DV + i % DV;
                        const int64_t e = (i / DV) * a.dv + col;
                        if (col < a.dv) hout[e] = k.it.in >= 0 ? hin[e] : 0.0f;
                    }
                });
            if (more) {
                const int left = k.it.len - k.t0;
                next.row = k.it.row0 + k.t0;
                next.m = left < C ? left : C;
                next.first = k.t0 == 0;
                next.last = left <= C;
                next.h = k.it.h;
                next.batch = a.cu ? 0 : k.it.seq;
                next.tile = k.it.tile;
                next.in = k.it.in;
                next.out = k.it.out;
#pragma unroll
                for (int e = 0; e < 4; ++e) gn[e] = load_g(a, k.it, k.t0 + 4 * lane + e);
                // its tiles into L2, before their stages are free
                if (lane < (wide ? 2 : 1)) {
                    const int x = 64 * lane;
                    tma_prefetch_4d(&map_k, x, k.it.h / a.k_rep, next.row, next.batch);
                    if (!STATE) tma_prefetch_4d(&map_q, x, k.it.h / a.q_rep, next.row, next.batch);
                    if (lane == 0)
                        tma_prefetch_4d(&map_v, next.tile * DV, next.h / a.v_rep, next.row, next.batch);
                }
            }
            if (n == 0) {
                now = next;
#pragma unroll
                for (int e = 0; e < 4; ++e) gnow[e] = gn[e];
                continue;
            }
            double g[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) g[e] = (double)clamp_g(gnow[e]);
#pragma unroll
            for (int e = 1; e < 4; ++e) g[e] += g[e - 1];
            double sum = g[3];                           // of the block's lanes up to this one
#pragma unroll
            for (int d = 1; d < 8; d <<= 1) {
                const double y = __shfl_up_sync(0xffffffffu, sum, d, 8);
                if ((lane & 7) >= d) sum += y;
            }
            const double last = __shfl_up_sync(0xffffffffu, sum, 1, 8);
            const double before = (lane & 7) ? last : 0.0;
            const double block = __shfl_sync(0xffffffffu, sum, 7, 8);
            // lane l: the blocks whose decays scalar l of OFF_SC multiplies
            constexpr uint64_t sets = 0x462F08CE7310ull;
            const uint32_t set = lane < 12 ? (uint32_t)(sets >> (4 * lane)) & 15u : 0u;
            double all = 0.0;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const double t = __shfl_sync(0xffffffffu, block, 8 * b);
                if (set >> b & 1u) all += t;
            }
            float cf[4], gg[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double x = before + g[e];
                cf[e] = exp_of(block - x);
                gg[e] = (float)(x * 1.4426950408889634);
            }
            const float mine = exp_of(all);
            if (STATE) {
                span_g = now.first ? all : span_g + all;
                if (lane == SC_ALL && now.last && now.tile == 0 && now.out >= 0)
                    a.seg_g[(int64_t)now.out * a.heads + now.h] = span_g;
            }
            if (!wait_warp(g_free(s), ((c >> 1) & 1) ^ 1, 0x451)) break;
            if (lane < 12) sc[s * 16 + lane] = mine;
            if (lane == SC_ALL) {
                dec[c & 3] = mine;                       // chunk c - 4 is long done
                chunks[c & 3] = now;
            }
            *reinterpret_cast<float4 *>(colf + s * C + 4 * lane) = make_float4(cf[0], cf[1], cf[2], cf[3]);
            *reinterpret_cast<float4 *>(g2 + s * C + 4 * lane) = make_float4(gg[0], gg[1], gg[2], gg[3]);
            mbar_arrive(g_full(s));
            if (now.m == 0) break;
            now = next;
#pragma unroll
            for (int e = 0; e < 4; ++e) gnow[e] = gn[e];
        }
    } else if (warp < W_P) {
        // -------------------------------------------------------- the state
        // Row r of the state, 32 columns a warp, 16 at a time: from h0 at a
        // sequence's start (pass 0), and e^{G_C} S0 + K^T V~ behind each chunk
        // (pass 1); to TMEM and (bf16, for Q S0) to shared memory, or to h_last
        // behind the last chunk.
        const int w = warp & 3, half = warp >> 2, r = 32 * w + lane;
        const uint32_t quarter = tmem + ((uint32_t)(32 * w) << 16);
        uint8_t *const hrow = smem + OFF_H + r * 128;
        bool ok = true;
        for (uint32_t c = 0; ok; ++c) {
            if (!wait_warp(g_full(c & 1), (c >> 1) & 1, 0x424)) break;
            const Chunk k = chunks[c & 3];
            if (k.m == 0) break;
            // g_full's next phase of this stage has to wait for this one to be seen here,
            // too: the state of chunk c is handed over a chunk earlier, so that all other
            // roles can be done with the chunk before these warps have looked
            if (!STATE) mbar_arrive(g_free(c & 1));
            const uint64_t dec2 = pair(dec[c & 3]);
            const int c0 = k.tile * DV;
            const int64_t at = ((int64_t)k.h * a.dk + r) * a.dv + c0;
            const int64_t per = a.heads * a.dk * a.dv;
            const float *const hin = (!STATE && a.seg ? a.seg_state : a.h0) + k.in * per + at;
            float *const hout = (STATE ? a.seg_state : a.h_last) + k.out * per + at;
            const bool row = r < a.dk;
#pragma unroll 1
            for (int pass = k.first ? 0 : 1; pass < 2; ++pass) {
                const bool store = pass == 1 && k.last;
                if (pass == 1) {
                    if (!(ok = wait_warp(d_full, c & 1, 0x425))) break;
                    fence_after();
                }
#pragma unroll 1
                for (int i = 32 * half; i < 32 * half + 32; i += 16) {
                    uint32_t h[16];
                    if (pass == 0) {
#pragma unroll
                        for (int j = 0; j < 16; j += 4) {
                            uint4 x = make_uint4(0, 0, 0, 0);
                            if (k.in >= 0 && row && c0 + i + j < a.dv)
                                x = *reinterpret_cast<const uint4 *>(hin + i + j);
                            h[j] = x.x; h[j + 1] = x.y; h[j + 2] = x.z; h[j + 3] = x.w;
                        }
                    } else {
                        uint32_t d0[16], d1[16];
                        tmem_ld16_async(quarter + T_H + i, h);
                        tmem_ld16_async(quarter + T_D + i, d0);
                        tmem_ld16_async(quarter + T_D + 64 + i, d1);
                        tmem_loaded(h);
                        tmem_loaded(d0);
                        tmem_loaded(d1);
                        uint64_t nan = 0;                // 0, or NaN
#pragma unroll
                        for (int j = 0; j < 16; j += 2) {
                            const uint64_t own = add2(pair(d0[j], d0[j + 1]), pair(d1[j], d1[j + 1]));
                            const uint64_t x = fma2(dec2, pair(h[j], h[j + 1]), own);
                            nan = fma2(own, 0, nan);
                            h[j] = lo_of(x);
                            h[j + 1] = hi_of(x);
                        }
                        if (__any_sync(0xffffffffu, row && ((lo_of(nan) | hi_of(nan)) & 0x7fffffffu))) {
                            // an infinity times V~'s parts makes NaN: the chunk's tokens one
                            // by one
                            walk_state(a, chunks[c & 3], r, i, quarter + T_H + i);
                            tmem_ld16_async(quarter + T_H + i, h);
                            tmem_loaded(h);
                        }
                    }
                    if (store) {
#pragma unroll
                        for (int j = 0; j < 16; j += 4)
                            if (k.out >= 0 && row && c0 + i + j < a.dv)
                                *reinterpret_cast<uint4 *>(hout + i + j) =
                                    make_uint4(h[j], h[j + 1], h[j + 2], h[j + 3]);
                    } else {
                        tmem_st16(quarter + T_H + i, h);
                    }
                }
                if (pass == 1) {
                    fence_before();
                    mbar_arrive(d_free);
                    if (STATE) mbar_arrive(g_free(c & 1));   // V~ (c) has read them too
                }
                if (!store) tmem_wait_st();
                if (STATE || store) continue;
                // Q S0 of the chunk before the one this state is for, and all else that
                // reads that chunk's q, where the second part goes
                const uint32_t prev = c + pass - 1;
                if (!(ok = wait_warp(h_free, prev & 1, 0x423) &&
                           wait_warp(q_read(prev & 1), (prev >> 1) & 1, 0x426)))
                    break;
                uint8_t *const hrow2 = smem + off_h2(c + pass) + r * 128;
#pragma unroll 1
                for (int i = 32 * half; i < 32 * half + 32; i += 16) {
                    uint32_t h[16], p[8], p2[8], bad = 0;
                    tmem_ld16_async(quarter + T_H + i, h);
                    tmem_loaded(h);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint64_t x = pair(h[2 * j], h[2 * j + 1]);
                        p[j] = pack_bf16(x);
                        p2[j] = pack_bf16(rest(x, p[j]));
                        poison(bad, p2[j]);
                    }
                    if (__any_sync(0xffffffffu, row && (bad & 0x7fff7fffu))) {
                        // infinities stand in the first part alone
#pragma unroll
                        for (int j = 0; j < 8; ++j) p2[j] = finite(p2[j]);
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t off = ((i / 8 + j) ^ (r & 7)) << 4;
                        *reinterpret_cast<uint4 *>(hrow + off) =
                            make_uint4(p[4 * j], p[4 * j + 1], p[4 * j + 2], p[4 * j + 3]);
                        *reinterpret_cast<uint4 *>(hrow2 + off) =
                            make_uint4(p2[4 * j], p2[4 * j + 1], p2[4 * j + 2], p2[4 * j + 3]);
                    }
                }
                fence_async_smem();
                mbar_arrive(h_full);
            }
        }
    } else if (warp < W_O) {
        // ---------------------------------------------------------------- P
        // rows 32 w + lane; the first four warps take blocks 0 and 2, the others
        // 1 and 3, each in place of its scores; zeros above the diagonal.
        const int w = warp & 3, odd = (warp - W_P) >> 2, r = 32 * w + lane;
        const uint32_t quarter = tmem + ((uint32_t)(32 * w) << 16);
        const uint64_t scale2 = pair(a.scale);
        for (uint32_t c = 0; !STATE; ++c) {
            const int s = c & 1;
            if (!wait_warp(g_full(s), (c >> 1) & 1, 0x431) || chunks[c & 3].m == 0) break;
            const float gr = g2[s * C + r];
            const float rowf = ex2(gr) * a.scale;
            // e^{blocks between}: block b's columns for the rows of block w
            const float f0 = rowf * (w == 2 ? sc[s * 16 + SC_1] : w == 3 ? sc[s * 16 + SC_12] : 1.0f);
            const float f1 = rowf * (w == 3 ? sc[s * 16 + SC_2] : 1.0f);
            if (!wait_warp(s_full, c & 1, 0x432)) break;
            fence_after();
#pragma unroll 1
            for (int n = 2 * odd; n < C / 16; n += (n & 1) ? 3 : 1) {      // 16 columns
                uint32_t x[16], p[16];
                uint64_t f[8];
                if (n >= 2 * w + 2) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) p[i] = 0u;
                    tmem_st16(quarter + T_S + 16 * n, p);
                    continue;
                }
                tmem_ld16_async(quarter + T_S + 16 * n, x);
                const int b = n >> 1;
                if (b < w) {
                    const uint64_t fb = pair(b == 0 ? f0 : b == 1 ? f1 : rowf);
                    const ulonglong2 *cf = reinterpret_cast<const ulonglong2 *>(colf + s * C + 16 * n);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const ulonglong2 y = cf[i];
                        f[2 * i] = mul2(y.x, fb);
                        f[2 * i + 1] = mul2(y.y, fb);
                    }
                } else {
                    // 0 above the diagonal; times an infinity or NaN that makes a
                    // NaN, and the row is done again below
                    const float4 *gj = reinterpret_cast<const float4 *>(g2 + s * C + 16 * n);
                    const int last = lane - 16 * (n & 1);            // the diagonal's column
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float4 y = gj[i];
                        const float e0 = 4 * i <= last ? ex2(gr - y.x) : 0.0f;
                        const float e1 = 4 * i + 1 <= last ? ex2(gr - y.y) : 0.0f;
                        const float e2 = 4 * i + 2 <= last ? ex2(gr - y.z) : 0.0f;
                        const float e3 = 4 * i + 3 <= last ? ex2(gr - y.w) : 0.0f;
                        f[2 * i] = mul2(scale2, pair(__float_as_uint(e0), __float_as_uint(e1)));
                        f[2 * i + 1] = mul2(scale2, pair(__float_as_uint(e2), __float_as_uint(e3)));
                    }
                }
                tmem_loaded(x);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint64_t y = mul2(pair(x[2 * i], x[2 * i + 1]), f[i]);
                    p[i] = pack_bf16(y);
                    p[8 + i] = pack_bf16(rest(y, p[i]));
                }
                tmem_st16(quarter + T_S + 16 * n, p);
            }
            tmem_wait_st();
            fence_before();
            mbar_arrive(p_full);
        }
    } else if (warp >= W_V) {
        // --------------------------------------------------------------- V~
        // the rows of V times e^{G_C - G_j}, in three bf16 parts
        const int w = warp & 3, r = 32 * w + lane;
        uint8_t *const trow = smem + OFF_VT + r * 128;
        for (uint32_t c = 0;; ++c) {
            const uint32_t ph2 = (c >> 1) & 1;
            const int s = c & 1;
            if (!wait_warp(g_full(s), ph2, 0x441)) break;
            const int m = chunks[c & 3].m;
            if (m == 0) break;
            if (m < C) {
                // rows behind the sequence (another one's, or nothing): zero in V and K,
                // whose values a product would otherwise meet; in K before Q K^T
                if (!wait_warp(full_k(s), ph2, 0x443)) break;
                if (r >= m) zero_row(smem + OFF_K + s * 2 * SUB + r * 128, 2);
                fence_async_smem();
            }
            if (!STATE) mbar_arrive(k_tail(s));
            const uint64_t wj2 = pair(colf[s * C + r] * sc[s * 16 + SC_AFTER + w]);
            if (!wait_warp(full_v(s), ph2, 0x442)) break;
            if (!wait_warp(d_full, (c & 1) ^ 1, 0x444)) break;             // V~ (c - 1) read
            uint8_t *const vrow = smem + OFF_V + s * SUB + r * 128;
            if (r >= m) zero_row(vrow, 1);
#pragma unroll 2
            for (int i = 0; i < 8; ++i) {
                const uint32_t off = (uint32_t)((i ^ (r & 7)) << 4);   // free of bank conflicts
                const uint4 x4 = *reinterpret_cast<const uint4 *>(vrow + off);
                const uint32_t x[4] = {x4.x, x4.y, x4.z, x4.w};
                uint32_t p0[4], p1[4], p2[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint64_t y = mul2(unpack_bf16(x[e]), wj2);
                    p0[e] = pack_bf16(y);
                    y = rest(y, p0[e]);
                    p1[e] = pack_bf16(y);
                    p2[e] = pack_bf16(rest(y, p1[e]));
                }
                *reinterpret_cast<uint4 *>(trow + off) = make_uint4(p0[0], p0[1], p0[2], p0[3]);
                *reinterpret_cast<uint4 *>(trow + SUB + off) =
                    make_uint4(p1[0], p1[1], p1[2], p1[3]);
                *reinterpret_cast<uint4 *>(trow + 2 * SUB + off) =
                    make_uint4(p2[0], p2[1], p2[2], p2[3]);
            }
            fence_async_smem();
            mbar_arrive(vt_full);
            mbar_arrive(STATE ? empty_v(s) : v_full(s));
        }
    } else {
        // -------------------------------------------------- the output rows
        const int w = warp & 3, r = 32 * w + lane;
        const uint32_t quarter = tmem + ((uint32_t)(32 * w) << 16);
        for (uint32_t c = 0; !STATE; ++c) {
            const int s = c & 1;
            if (!wait_warp(g_full(s), (c >> 1) & 1, 0x446)) break;
            const Chunk k = chunks[c & 3];
            if (k.m == 0) break;
            const uint64_t ei2 = pair(ex2(g2[s * C + r]) * sc[s * 16 + SC_BEFORE + w] * a.scale);
            const int c0 = k.tile * DV;
            __nv_bfloat16 *const row = static_cast<__nv_bfloat16 *>(a.o) +
                                       k.batch * a.os[0] +
                                       (int64_t)(k.row + r) * a.os[1] + k.h * a.os[2] + c0;
            if (!wait_warp(o_full, c & 1, 0x445)) break;
            mbar_arrive(g_free(s));                      // P (c) has read them too
            fence_after();
            // Q K^T and Q S0 have read the chunk's q: its stage takes the output rows
            uint8_t *const orow = smem + OFF_Q + s * 2 * SUB + r * 128;
            uint32_t bad = 0;                            // 0, or NaN
#pragma unroll 1
            for (int i0 = 0; i0 < DV; i0 += 16) {
                uint32_t pv[16], q2[16], qh[16], y[8];
                tmem_ld16_async(quarter + T_PV + i0, pv);
                tmem_ld16_async(quarter + T_QH + i0, q2);
                tmem_ld16_async(quarter + T_QH + 64 + i0, qh);
                tmem_loaded(pv);
                tmem_loaded(q2);
                tmem_loaded(qh);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    y[i] = pack_bf16(fma2(add2(pair(q2[2 * i], q2[2 * i + 1]),
                                               pair(qh[2 * i], qh[2 * i + 1])),
                                          ei2, pair(pv[2 * i], pv[2 * i + 1])));
                    poison(bad, y[i]);
                }
                const int j = i0 / 8;
                *reinterpret_cast<uint4 *>(orow + ((j ^ (r & 7)) << 4)) =
                    make_uint4(y[0], y[1], y[2], y[3]);
                *reinterpret_cast<uint4 *>(orow + (((j + 1) ^ (r & 7)) << 4)) =
                    make_uint4(y[4], y[5], y[6], y[7]);
            }
            // what P V alone has met (a state that is not finite stays so: its rows are right)
            uint32_t redo = 0;
            if (__any_sync(0xffffffffu, r < k.m && (bad & 0x7fff7fffu))) {
                uint64_t nan = 0;                        // 0, or NaN
#pragma unroll 1
                for (int i0 = 0; i0 < DV; i0 += 16) {
                    uint32_t pv[16];
                    tmem_ld16_async(quarter + T_PV + i0, pv);
                    tmem_loaded(pv);
#pragma unroll
                    for (int i = 0; i < 8; ++i) nan = fma2(pair(pv[2 * i], pv[2 * i + 1]), 0, nan);
                }
                redo = __ballot_sync(0xffffffffu, r < k.m && ((lo_of(nan) | hi_of(nan)) & 0x7fffffffu));
            }
            const bool cold = redo != 0;
            if (!cold) {
                fence_before();
                mbar_arrive(o_free);
                fence_async_smem();
                __syncwarp();
                if (k.m == C) {
                    if (lane == 0) {
                        tma_store_4d(&map_o, base + OFF_Q + s * 2 * SUB + w * 32 * 128, k.tile * DV,
                                     k.h, k.row + 32 * w, k.batch);
                        bulk_commit();
                        bulk_wait_read0();
                    }
                } else if (r < k.m) {
                    // the rows behind a sequence's end may be another one's
#pragma unroll 1
                    for (int i = 0; i < DV / 8 && c0 + 8 * i < a.dv; ++i)
                        *reinterpret_cast<uint4 *>(row + 8 * i) =
                            *reinterpret_cast<const uint4 *>(orow + ((i ^ (r & 7)) << 4));
                }
            } else {
                // infinities or NaN: those rows again, from their own tokens; 16 rows at a
                // time through the warp's part of the stage
                float *const part = reinterpret_cast<float *>(smem + OFF_Q + s * 2 * SUB + w * 32 * 128);
#pragma unroll 1
                for (int n = 0; n < 2; ++n) {
#pragma unroll 1
                    for (int i0 = 0; i0 < DV; i0 += 16) {
                        uint32_t z[16], q2[16], qh[16];
                        tmem_ld16_async(quarter + T_PV + i0, z);
                        tmem_ld16_async(quarter + T_QH + i0, q2);
                        tmem_ld16_async(quarter + T_QH + 64 + i0, qh);
                        tmem_loaded(z);
                        tmem_loaded(q2);
                        tmem_loaded(qh);
                        if (lane >> 4 == n) {
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                // an infinite q meets S0's first part alone: the second's
                                // sign is its own
                                float x = __uint_as_float(qh[i]);
                                if (x - x == 0.0f) x += __uint_as_float(q2[i]);
                                x *= __uint_as_float(lo_of(ei2));
                                part[64 * (lane & 15) + i0 + i] =
                                    redo >> lane & 1 ? x : x + __uint_as_float(z[i]);
                            }
                        }
                        __syncwarp();
                    }
                    masked_rows(a, chunks[c & 3], 32 * w + 16 * n, redo >> 16 * n, part);
                    __syncwarp();
                }
                fence_async_smem();                      // the stage is a TMA load's next
                fence_before();
                mbar_arrive(o_free);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty_q(s));
            __syncwarp();
        }
        if (lane == 0) bulk_wait0();                     // the stores are complete
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == W_MMA) {
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

// (batch, tokens, heads, width) bf16 as a 4D map of `rows`-token x 64-column boxes;
// *ok = false when TMA cannot address it
static int token_map(CUtensorMap *map, const void *p, const int64_t (&s)[3], int64_t batch,
                     int64_t tokens, int64_t heads, int64_t width, int rows, bool *ok) {
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
    cuuint32_t box[4] = {64, 1, (cuuint32_t)rows, 1};
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
    return !a.recurrent && a.dtype == MB2_BF16 && a.dk <= 128 && a.dk % 8 == 0 && a.dv % 8 == 0 &&
           a.seqlen > 0 && aligned(a.o, 16) && a.os[0] % 8 == 0 && a.os[1] % 8 == 0 && a.os[2] % 8 == 0 &&
           (!a.h0 || aligned(a.h0, 16)) && (!a.h_last || aligned(a.h_last, 16));
}

bool chunked_fits(const Args &a) { return fits(a); }

int chunked(const Args &a, bool state_only, cudaStream_t st, bool *used) {
    *used = false;
    if (!fits(a)) return MB2_OK;
    MB2_TRY(get_encode());
    CUtensorMap mq, mk, mv, mo;
    const int64_t batch = a.cu ? 1 : a.seqs;
    bool ok[4];
    MB2_TRY(token_map(&mq, a.q, a.qs, batch, a.seqlen, a.heads / a.q_rep, a.dk, C, &ok[0]));
    MB2_TRY(token_map(&mk, a.k, a.ks, batch, a.seqlen, a.heads / a.k_rep, a.dk, C, &ok[1]));
    MB2_TRY(token_map(&mv, a.v, a.vs, batch, a.seqlen, a.heads / a.v_rep, a.dv, C, &ok[2]));
    MB2_TRY(token_map(&mo, a.o, a.os, batch, a.seqlen, a.heads, a.dv, 32, &ok[3]));
    if (!ok[0] || !ok[1] || !ok[2] || !ok[3]) return MB2_OK;
    *used = true;
    const int sms = num_sms();
    auto kern = state_only ? decay_chunk_kernel<true> : decay_chunk_kernel<false>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)SMEM_BYTES);
    if (e != cudaSuccess) return fail(MB2_ERR_CUDA, "decay_attention: %s", cudaGetErrorString(e));
    const int tiles = (int)ceil_div(a.dv, DV);
    const int64_t items = (int64_t)tiles * a.heads * spans(a);
    MB2_REQUIRE(items < (1ll << 31), MB2_ERR_SHAPE, "decay_attention: too many sequences x heads");
    const unsigned grid = (unsigned)(items < sms ? items : sms);
    kern<<<grid, THREADS, SMEM_BYTES, st>>>(mq, mk, mv, mo, a, (uint32_t)tiles, (uint32_t)items);
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
