// Gated linear recurrence: r = sigmoid(decay_gate), i = sigmoid(input_gate),
//   a_t = exp(-sharpness softplus(decay) r_t),
//   h_t = a_t h_{t-1} + sqrt(1 - a_t^2) i_t x_t,
// over whole prompts, its gradients, and one token at a time.
//
// A prompt is cut into tiles of tokens x 64 channels; persistent CTAs take them in
// order.  A run of tokens acts on the state as h -> A h + H: the CTA's warps compute their
// tokens' a and b = sqrt(1 - a^2) i x once, one warp composes the warps' (A, H), publishes
// the tile's, and looks back over the tiles before it for the nearest known state, so that
// the inputs are read once and h written once whatever the sequences' lengths.  A state
// found at a distance is carried through the published (A, H) in order, with the operations
// that the tiles themselves use: the bits do not depend on where it was found.
// The gradients run the same way from the end: with C_t = a_t G_t,
//   G_t = dh_t + C_{t+1},
//   dx = G m i,  dinput_gate = G m i x (1 - i),  m = sqrt(1 - a^2),
//   d log a = G (a h_{t-1} - a^2 i x / m),
// the states h from those that the forward pass left before every tile of the backward's.
// Sequences end inside tiles: at a first token the state is started anew (never
// multiplied by zero, which would let an infinity through).
//
// Measured (B200; a value: one channel of one token), with the rate that HBM allows:
//   forward  fp32, 151 x 180 x 1536     124 us   103  HBM, 83 % of the copy rate
//            bf16, 8 x 8192 x 1536      195      124  issue slots 52 %, MUFU 42 %, 28 warps an
//                                                     SM that wait for one another's tiles
//            bf16, 5 of 6500 x 1024     116       41  16 chains of tiles for 296 CTAs
//            bf16, 65536 x 64            44        5  one chain
//            bf16, 8 x 8192 x 1535      473      124  one CTA an SM (slots of twice the bytes)
//   backward bf16, 8 x 4096 x 1536      230      108  issue 40 %, MUFU 29 %, 16 warps an SM
// What it took for the bf16 forward at 8 x 8192: a thread a channel 6710 us, tiles 593,
// rare paths out of the unrolled loops 401, one barrier a tile and 16-byte fetches 293, a
// carrying warp 263, a and b through shared memory and more warps 235, tiles without marks
// 219, of 104 tokens 210, nothing fenced 202.
#include "gated_rec.cuh"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace mb2 {
namespace rec {
namespace {

constexpr int STRIP = 64;                     // channels of a tile
// Warps that hold a tile's tokens, tokens of each, of a tile; CTAs of an SM.  One more
// warp of the CTA carries the states.  As many warps as registers (bf16) or shared memory
// (fp32: twice the bytes a token) let two CTAs have; bf16 rows off 16 bytes come through
// fp32's slots in bf16's shape, of which one CTA fits an SM.  Forward, 8 x 8192 bf16: 13 warps 202
// us, 11 210, 9 (three CTAs) 215, 14 212 (spills); 151 x 180 fp32: 10 warps 139, 8 134.  The
// backward pass keeps more of a token in registers, and there fewer warps of longer runs
// win, for less is composed and carried a token; 8 x 4096 with gradients, bf16: 12 warps of
// 4 tokens 385 us, 7 of 8 346, 6 of 8 359, 5 of 8 (three CTAs) 379; fp32: 8 of 4 454, 5 of 8
// 429 (at an odd width 190 and 211); with 1 - sigmoid kept by itself 353 and 431.
template <typename T> struct Forward {
    static constexpr int WARPS = sizeof(T) == 2 ? 13 : 8, RUN = 8, THREADS = 32 * WARPS;
    static constexpr int TILE = WARPS * RUN, CTAS = 2;
};
template <typename T> struct Backward {
    static constexpr int WARPS = sizeof(T) == 2 ? 7 : 5, RUN = 8, THREADS = 32 * WARPS;
    static constexpr int TILE = WARPS * RUN, CTAS = 2;
};
static_assert(Backward<float>::TILE % Forward<float>::RUN == 0 &&
              Backward<__nv_bfloat16>::TILE % Forward<__nv_bfloat16>::RUN == 0,
              "states are left between warps' runs");
constexpr uint64_t WAIT_NS = 2000000000ull;   // 2 s bound on any wait

// 0 = ok, else a wait expired; part of mb2_device_status
__device__ int g_error = 0;

__device__ __forceinline__ uint64_t globaltimer() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

// How a call is cut up.  Dense batches of short sequences are one axis of
// batch x seqlen tokens (flat), so that a tile can hold several; otherwise a tile
// holds tokens of one sequence.
struct Plan {
    int64_t tokens;                           // of the axis that tiles cut
    int period;                               // dense: tokens of a sequence
    int axes;                                 // batch rows of the tiles, 1 when flat or packed
    int per_axis, rows, strips;               // tiles along an axis, all of them, across
    unsigned *ticket;                         // and whether a wait ran out
    ulonglong2 *state, *agg;                  // (rows, strips, 32): what tiles publish
    float *log2a;                             // (strips x 64): log2 of a at an open gate
    float *parts;                             // backward: (rows, width)
    int stride[4];                            // bytes from token to token: gates, x, dh
    bool lean;                                // they fit, and rows are 16-byte chunks
    bool alone;                               // no tile needs another's state, all run at once:
                                              // CTA k has tile k, and nothing is set up first
};

Plan plan_of(const Args &a, int tile, int ctas) {
    Plan p{};
    const bool flat = !a.cu && a.seqlen <= 32;
    p.period = (int)a.seqlen;
    p.axes = a.cu || flat ? 1 : (int)a.batch;
    p.tokens = flat ? a.batch * a.seqlen : a.seqlen;
    p.per_axis = (int)ceil_div(p.tokens, tile);
    p.rows = p.axes * p.per_axis;
    p.strips = (int)ceil_div(a.width, STRIP);
    // (148: a B200's SMs; the workspace's size depends on it, which is asked for on the host)
    p.alone = p.per_axis == 1 && (int64_t)p.rows * p.strips <= 148 * ctas;
    return p;
}

template <template <typename> class Shape> Plan plan_of(const Args &a, int dtype) {
    return dtype == MB2_F32 ? plan_of(a, Shape<float>::TILE, Shape<float>::CTAS)
                            : plan_of(a, Shape<__nv_bfloat16>::TILE, Shape<__nv_bfloat16>::CTAS);
}

// the workspace's parts; returns its size
size_t lay_out(Plan &p, void *ws, int64_t width, bool backward) {
    char *at = static_cast<char *>(ws);
    const size_t tiles = (size_t)p.rows * p.strips;
    size_t n = 0;
    if (p.alone) {
        p.parts = static_cast<float *>(ws);
        return backward ? (size_t)p.rows * width * 4 : 0;
    }
    auto part = [&](size_t bytes) {
        char *q = at ? at + n : nullptr;
        n += (size_t)round_up((int64_t)bytes, 256);
        return q;
    };
    p.state = reinterpret_cast<ulonglong2 *>(part(tiles * 512));
    p.agg = reinterpret_cast<ulonglong2 *>(part(tiles * 512));
    p.ticket = reinterpret_cast<unsigned *>(part(16));     // behind them: zeroed with them
    p.log2a = reinterpret_cast<float *>(part((size_t)p.strips * STRIP * 4));
    p.parts = backward ? reinterpret_cast<float *>(part((size_t)p.rows * width * 4)) : nullptr;
    return n;
}

// ---------------------------------------------------------- rows and channels
// A lane has two channels: neighbours, fetched by its warp in chunks of 16 bytes (WIDE:
// all rows aligned to those), or channels lane and lane + 32 of the strip, one by one.
template <typename T, bool WIDE> struct Lane;
template <> struct Lane<__nv_bfloat16, true> {
    using Slot = uint32_t;
    static __device__ __forceinline__ uint64_t get(Slot s, int) {
        return pair(s << 16, s & 0xffff0000u);
    }
    static __device__ __forceinline__ void put(__nv_bfloat16 *p, uint64_t v, bool, bool) {
        const __nv_bfloat162 w = __floats2bfloat162_rn(lo(v), hi(v));
        *reinterpret_cast<__nv_bfloat162 *>(p) = w;
    }
};
template <> struct Lane<float, true> {
    using Slot = uint64_t;
    static __device__ __forceinline__ uint64_t get(Slot s, int) { return s; }
    static __device__ __forceinline__ void put(float *p, uint64_t v, bool, bool) {
        *reinterpret_cast<float2 *>(p) = make_float2(lo(v), hi(v));
    }
};
template <> struct Lane<__nv_bfloat16, false> {
    using Slot = uint64_t;
    // the aligned words that hold the two values (inside the allocation: words are
    // smaller than what any allocator aligns to)
    static __device__ __forceinline__ void fetch(Slot *s, const __nv_bfloat16 *p, bool in0,
                                                 bool in1) {
        const char *w = reinterpret_cast<const char *>(reinterpret_cast<uintptr_t>(p) & ~3ull);
        uint32_t *d = reinterpret_cast<uint32_t *>(s);
        if (in0) cp_async4(d, w);
        if (in1) cp_async4(d + 1, w + 64);
    }
    static __device__ __forceinline__ uint64_t get(Slot s, int odd) {
        const uint32_t a = lo_of(s), b = hi_of(s);
        return odd ? pair(a & 0xffff0000u, b & 0xffff0000u) : pair(a << 16, b << 16);
    }
    static __device__ __forceinline__ void put(__nv_bfloat16 *p, uint64_t v, bool in0, bool in1) {
        if (in0) p[0] = __float2bfloat16_rn(lo(v));
        if (in1) p[32] = __float2bfloat16_rn(hi(v));
    }
};
template <> struct Lane<float, false> {
    using Slot = uint64_t;
    static __device__ __forceinline__ void fetch(Slot *s, const float *p, bool in0, bool in1) {
        uint32_t *d = reinterpret_cast<uint32_t *>(s);
        if (in0) cp_async4(d, p);
        if (in1) cp_async4(d + 1, p + 32);
    }
    static __device__ __forceinline__ uint64_t get(Slot s, int) { return s; }
    static __device__ __forceinline__ void put(float *p, uint64_t v, bool in0, bool in1) {
        if (in0) p[0] = lo(v);
        if (in1) p[32] = hi(v);
    }
};

// the channels of a lane: c and c + (WIDE ? 1 : 32), in range or not
template <bool WIDE> struct Channels {
    int64_t c;
    bool in0, in1;
    __device__ __forceinline__ Channels(int strip, int lane, int64_t width) {
        c = (int64_t)strip * STRIP + (WIDE ? 2 * lane : lane);
        in0 = c < width;
        in1 = c + (WIDE ? 1 : 32) < width;
    }
    __device__ __forceinline__ uint64_t load(const float *p) const {
        constexpr int step = WIDE ? 1 : 32;
        return pack(in0 ? p[c] : 0.0f, in1 ? p[c + step] : 0.0f);
    }
    // of an array that goes on to the strip's end
    __device__ __forceinline__ uint64_t load_all(const float *p) const {
        return pack(p[c], p[c + (WIDE ? 1 : 32)]);
    }
    __device__ __forceinline__ void store(float *p, uint64_t v) const {
        constexpr int step = WIDE ? 1 : 32;
        if (in0) p[c] = lo(v);
        if (in1) p[c + step] = hi(v);
    }
};

// A tensor's rows.  Where a flat batch is not one run of tokens, token g of the axis
// is row (g / period, g % period).
struct Rows {
    const void *p;
    int64_t sb, st;
    bool run;
    __device__ __forceinline__ Rows(const void *at, const int64_t (&s)[2], const Args &a,
                                    const Plan &q)
        : p(at), sb(s[0]), st(s[1]), run(q.axes > 1 || a.batch == 1 || s[0] == s[1] * a.seqlen) {}
    __device__ __forceinline__ int64_t of(int axis, int g) const { return axis * sb + g * st; }
    __device__ __forceinline__ int64_t far(const Plan &q, int g) const {
        return (g / q.period) * sb + (g % q.period) * st;
    }
};

struct Tile {
    int row, strip, axis, first, count;       // tokens first .. first + count of the axis
    int plain;                                // full, and no sequence starts or ends in it
};
// where a tile's rows are: of decay gate, input gate, x and dh, and the outputs' offset
struct Places {
    const char *in[4];
    int64_t out;
};
constexpr unsigned NO_TILE = 0xffffffffu;     // behind the last
__device__ __forceinline__ Tile tile_at(const Plan &p, unsigned k, int tile, bool backward) {
    Tile t;
    const unsigned q = k / p.strips;
    t.strip = (int)(k - q * p.strips);
    int c = (int)(q / p.axes);
    t.axis = (int)(q - (unsigned)c * p.axes);
    if (backward) c = p.per_axis - 1 - c;
    t.row = c < 0 || c >= p.per_axis ? -1 : t.axis * p.per_axis + c;
    t.first = c * tile;
    t.count = (int)min((int64_t)tile, p.tokens - t.first);
    t.plain = 0;
    return t;
}
// Whether a tile needs none of the marks of its tokens: most do not, and the warps that
// hold tokens save a quarter of their instructions.
__device__ __forceinline__ bool is_plain(const Args &a, const Plan &p, const Tile &t, int tile) {
    if (!p.lean || t.row < 0 || t.count < tile || (int64_t)(t.strip + 1) * STRIP > a.width)
        return false;
    if (!a.cu) return (p.axes > 1 || a.batch == 1) && t.first > 0 && t.first + tile < p.period;
    int lo = 0, hi = (int)a.seqs + 1;                      // offsets <= first: lo .. hi
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (a.cu[mid] <= t.first) lo = mid + 1;
        else hi = mid;
    }
    return lo > 0 && lo <= a.seqs && a.cu[lo - 1] < t.first && t.first > 0 &&
           (int64_t)a.cu[lo] > t.first + tile && t.first + tile < a.seqlen;
}
// By the carrying warp: the k-th tile and its places, for the CTA.
template <typename T>
__device__ __forceinline__ void next_tile(const Args &a, const Plan &p, unsigned k, int tile,
                                          bool backward, Tile *to, Places *places) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) {
        Tile t = tile_at(p, k, tile, backward);
        t.plain = is_plain(a, p, t, tile);
        *to = t;
    }
    __syncwarp();
    const Tile t = *to;
    if (!t.plain) return;
    const int64_t c = (int64_t)t.strip * STRIP;
    auto place = [&](int k, const void *from, const int64_t (&stride)[2]) {
        const int64_t at = (p.axes > 1 ? t.axis * stride[0] : 0) + t.first * stride[1] + c;
        if (lane == k)
            places->in[k] = static_cast<const char *>(from) + at * (int64_t)sizeof(T);
    };
    place(0, a.rg, a.rs);
    place(1, a.ig, a.is);
    place(2, a.x, a.xs);
    place(3, a.dh, a.ds);
    if (lane == 4)
        places->out = (((p.axes > 1 ? t.axis * a.seqlen : 0) + t.first) * a.width + c) *
                      (int64_t)sizeof(T);
}

// Where sequences start and end among a warp's tokens (bit j: its token j); the same in
// all lanes, but for seq, which in lane j is token j's sequence if that starts or ends there.
struct Marks {
    unsigned first, last, none;               // none: tokens of no sequence
    int seq;
};
// g: the axis' token, n of them
__device__ __forceinline__ Marks marks_of(const Args &a, const Plan &p, const Tile &t, int g,
                                          int n) {
    const int lane = threadIdx.x & 31;
    Marks m{};
    if (p.axes > 1 || (!a.cu && a.batch == 1)) {          // a tile of one sequence
        m.seq = t.axis;
        m.first = g == 0 && n > 0;
        m.last = n > 0 && g + n == p.period ? 1u << (n - 1) : 0u;
        return m;
    }
    bool first = false, last = false, none = false;
    if (lane < n) {
        const int at = g + lane;
        if (a.cu) {
            int lo = 0, hi = (int)a.seqs + 1;              // offsets <= at: lo .. hi
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (a.cu[mid] <= at) lo = mid + 1;
                else hi = mid;
            }
            m.seq = lo - 1;
            none = m.seq < 0 || m.seq >= a.seqs;
            if (!none) {
                first = max(a.cu[m.seq], 0) == at;
                last = min((int64_t)a.cu[m.seq + 1], a.seqlen) == at + 1;
            }
        } else {
            m.seq = at / p.period;
            first = at == m.seq * p.period;
            last = at + 1 == (m.seq + 1) * p.period;
        }
    }
    m.first = __ballot_sync(0xffffffffu, first);
    m.last = __ballot_sync(0xffffffffu, last);
    m.none = __ballot_sync(0xffffffffu, none);
    return m;
}
__device__ __forceinline__ int64_t seq_of(const Marks &m, int j) {
    return __shfl_sync(0xffffffffu, m.seq, j);
}

// cp.async of a warp's tokens; slots: the warp's of token 0, [token][THREADS]
template <typename T, bool WIDE, typename Shape>
__device__ __forceinline__ void fetch(const Rows &r, typename Lane<T, WIDE>::Slot *slots,
                                      const Plan &p, const Tile &t, int g, int n, int64_t width) {
    const int lane = threadIdx.x & 31;
    n = min(n, Shape::RUN);
    if constexpr (WIDE) {
        constexpr int CHUNK = 16 / (int)sizeof(T), CHUNKS = STRIP / CHUNK, MANY = 32 / CHUNKS;
        const int64_t c = (int64_t)t.strip * STRIP + lane % CHUNKS * CHUNK;
        if (c >= width) return;
        const T *base = static_cast<const T *>(r.p) + c;
        const int j0 = lane / CHUNKS;
        char *s = reinterpret_cast<char *>(slots + j0 * Shape::THREADS) + lane % CHUNKS * 16;
        static_assert(Shape::RUN % MANY == 0, "a warp fetches MANY rows at a time");
        constexpr int64_t kStep = (int64_t)MANY * Shape::THREADS * sizeof(*slots);
        if (n == Shape::RUN && r.run) {
            const T *q = base + r.of(t.axis, g + j0);
#pragma unroll
            for (int k = 0; k < Shape::RUN / MANY; ++k)
                cp_async16(s + k * kStep, q + k * MANY * r.st);
        } else {
#pragma unroll 1
            for (int j = j0; j < n; j += MANY, s += kStep)
                cp_async16(s, base + (r.run ? r.of(t.axis, g + j) : r.far(p, g + j)));
        }
    } else {
        const Channels<WIDE> ch(t.strip, lane, width);
        if (!ch.in0) return;
        const T *base = static_cast<const T *>(r.p) + ch.c, *q = base + r.of(t.axis, g);
        slots += lane;
        if (n == Shape::RUN && r.run) {
#pragma unroll
            for (int j = 0; j < Shape::RUN; ++j)
                Lane<T, WIDE>::fetch(slots + j * Shape::THREADS, q + j * r.st, ch.in0, ch.in1);
        } else {
#pragma unroll 1
            for (int j = 0; j < n; ++j)
                Lane<T, WIDE>::fetch(slots + j * Shape::THREADS,
                                     r.run ? q + j * r.st : base + r.far(p, g + j), ch.in0, ch.in1);
        }
    }
}
// the same for a plain tile; from: its first token's row
template <typename Slot, typename Shape>
__device__ __forceinline__ void fetch_plain(const char *from, int stride, Slot *slots) {
    constexpr int CHUNKS = 32 * (int)sizeof(Slot) / 16, MANY = 32 / CHUNKS;
    static_assert(Shape::RUN % MANY == 0, "a warp fetches MANY rows at a time");
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, j0 = lane / CHUNKS;
    const char *q = from + (w * Shape::RUN + j0) * stride + lane % CHUNKS * 16;
    char *s = reinterpret_cast<char *>(slots + j0 * Shape::THREADS) + lane % CHUNKS * 16;
#pragma unroll
    for (int k = 0; k < Shape::RUN / MANY; ++k)
        cp_async16(s + k * MANY * Shape::THREADS * (int)sizeof(Slot), q + k * MANY * stride);
}
// a warp's rows of an output from its lanes' values; to: where its first token's go
template <typename T, int RUN>
__device__ __forceinline__ void put_plain(void *to, int64_t offset, int64_t width,
                                          const uint64_t (&v)[RUN]) {
    char *q = static_cast<char *>(to) + offset;
    const int step = (int)width * (int)sizeof(T);
#pragma unroll
    for (int j = 0; j < RUN; ++j)
        Lane<T, true>::put(reinterpret_cast<T *>(q + j * step), v[j], true, true);
}
// bit j: token j's values are in the upper halves of their words
template <typename T, bool WIDE, typename Shape>
__device__ __forceinline__ unsigned odd_of(const Rows &r, const Plan &p, int axis, int g,
                                           int64_t c) {
    if (WIDE || sizeof(T) == 4) return 0;
    const unsigned at = (unsigned)(reinterpret_cast<uintptr_t>(r.p) >> 1) + (unsigned)c;
    if (r.run) {
        const unsigned odd = (at + (unsigned)r.of(axis, g)) & 1u ? ~0u : 0u;
        return r.st & 1 ? odd ^ 0xaaaaaaaau : odd;
    }
    unsigned odd = 0;
#pragma unroll 1
    for (int j = 0; j < Shape::RUN; ++j) odd |= ((at + (unsigned)r.far(p, g + j)) & 1u) << j;
    return odd;
}
// what a lane has fetched, token j
template <typename T, bool WIDE>
__device__ __forceinline__ uint64_t value(typename Lane<T, WIDE>::Slot s, unsigned odd, int j) {
    return Lane<T, WIDE>::get(s, odd >> j & 1);
}
// Whether a warp met input gates below -43.6 (where near_input_factor does not hold) that are
// not closed (1 + e^-v infinite): the least distance of their bits from the first such value's,
// which wraps around for all others.
template <typename T, bool WIDE> struct FarGates {
    static constexpr unsigned kFirst = 0x5f000001u, kMany = 0x7f800000u - kFirst;  // of 1 + e^-v
    unsigned least = ~0u;
    __device__ __forceinline__ void note(typename Lane<T, WIDE>::Slot, uint64_t d) {
        least = __viaddmin_u32(lo_of(d), 0u - kFirst, __viaddmin_u32(hi_of(d), 0u - kFirst, least));
    }
    __device__ __forceinline__ bool some() const {
        return __any_sync(0xffffffffu, least < kMany);
    }
};
template <> struct FarGates<__nv_bfloat16, true> {     // both gates at once: -43 .. -88.5
    static constexpr unsigned kFirst = 0xc22cu, kMany = 0xc2b2u - kFirst;
    unsigned least = ~0u;
    __device__ __forceinline__ void note(uint32_t gates, uint64_t) {
        least = __viaddmin_u16x2(gates, (0x10000u - kFirst) * 0x10001u, least);
    }
    __device__ __forceinline__ bool some() const {
        return __any_sync(0xffffffffu, (least & 0xffffu) < kMany || least >> 16 < kMany);
    }
};
// rows of an output from a lane's values: token j of n
template <typename T, bool WIDE, int RUN>
__device__ __forceinline__ void put_rows(void *to, int64_t token, int64_t width, int n,
                                         const Channels<WIDE> &ch, const uint64_t (&v)[RUN]) {
    if (!ch.in0) return;
    T *q = static_cast<T *>(to) + token * width + ch.c;
    if (n == RUN) {
#pragma unroll
        for (int j = 0; j < RUN; ++j) Lane<T, WIDE>::put(q + j * width, v[j], ch.in0, ch.in1);
    } else {
#pragma unroll
        for (int j = 0; j < RUN; ++j)
            if (j < n) Lane<T, WIDE>::put(q + j * width, v[j], ch.in0, ch.in1);
    }
}

// ------------------------------------------------------------------ look-back
// What a tile publishes, for a lane's two channels: two words of 64 bits with its (A, H),
// and two with the states behind it and a tag.  A word is read and written in one piece
// and says itself whether it is there (the tag, or an A that is not 0), so that nothing
// needs a fence and a look takes one trip to L2.
constexpr unsigned KNOWN = 2;
// Looks for the state of the tile before once a tile's (A, H) are out, in which it mostly
// has come (8 x 8192, 192 chains of tiles for 296 CTAs); more of them, or some while the
// tile is computed, cost where it has not (5 sequences of 6500 tokens, 16 chains: 121 us,
// with four early looks 128).
constexpr int LOOKS = 2;

__device__ __forceinline__ ulonglong2 words_load(const ulonglong2 *p) {
    ulonglong2 v;
    asm volatile("ld.relaxed.gpu.global.v2.u64 {%0, %1}, [%2];"
                 : "=l"(v.x), "=l"(v.y) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void words_store(ulonglong2 *p, uint64_t x, uint64_t y) {
    asm volatile("st.relaxed.gpu.global.v2.u64 [%0], {%1, %2};" ::"l"(p), "l"(x), "l"(y) : "memory");
}
__device__ __forceinline__ void state_store(ulonglong2 *p, uint64_t h) {
    words_store(p, pair(lo_of(h), KNOWN), pair(hi_of(h), KNOWN));
}
__device__ __forceinline__ bool known(const ulonglong2 &v) {
    return hi_of(v.x) == KNOWN && hi_of(v.y) == KNOWN;
}
__device__ __forceinline__ uint64_t state_of(const ulonglong2 &v) {
    return pair(lo_of(v.x), lo_of(v.y));
}
__device__ __forceinline__ bool there(const ulonglong2 &v) {       // (A below, H above)
    return lo_of(v.x) != 0 && lo_of(v.y) != 0;
}

// Bounds a warp's wait; true, in all lanes, once it is over.  After one wait of the call
// ran out the others do not wait as long again.
struct Patience {
    unsigned *gave_up;                        // of the call
    uint64_t since = 0;
    unsigned polls = 0;
    __device__ __forceinline__ explicit Patience(const Plan &p) : gave_up(p.ticket + 1) {}
    __device__ __forceinline__ bool over() {
        if ((++polls & 63) != 0) return false;
        const uint64_t now = globaltimer();
        if (since == 0) since = now;
        const bool out = now - since > WAIT_NS || *(volatile unsigned *)gave_up != 0;
        if (!__any_sync(0xffffffffu, out)) return false;
        if ((threadIdx.x & 31) == 0) {
            *(volatile unsigned *)gave_up = 1;
            atomicCAS(&g_error, 0, 901);
        }
        return true;
    }
};

// the tile's lane of p.state and p.agg
__device__ __forceinline__ int64_t record(const Plan &p, int row, int strip) {
    return ((int64_t)row * p.strips + strip) * 32 + (threadIdx.x & 31);
}
// A product of decays that underflowed still passes an infinity on, and is never 0
__device__ __forceinline__ uint64_t keep(uint64_t a) {
    constexpr float kLeast = 1.17549435e-38f;
    return pack(fmaxf(lo(a), kLeast), fmaxf(hi(a), kLeast));
}

// The state that enters tile (row, strip): that behind the nearest tile whose state is
// known, carried through the (A, H) of those between.  STEP: -1 towards earlier rows, +1
// towards later ones.  Tiles are taken in order, so the tiles looked at are done or held
// by CTAs that run and publish (A, H) without waiting.
template <int STEP>
__device__ __forceinline__ uint64_t look_back(const Plan &p, int row, int strip) {
    const int lane = threadIdx.x & 31;
    constexpr int MANY = 8;
    Patience patience(p);
    for (;;) {
        // the nearest: each lane looks at another tile, at the word of its first channel
        int found = 0;
        for (int base = 0; !found; base += 32) {
            const int q = row + STEP * (base + lane + 1);
            const bool in = q >= 0 && q < p.rows;
            bool has = false;
            if (in) has = known(words_load(p.state + ((int64_t)q * p.strips + strip) * 32));
            const unsigned have = __ballot_sync(0xffffffffu, has);
            if (have) {
                found = base + __ffs(have);
            } else if (!__all_sync(0xffffffffu, in)) {     // none so far
                if (patience.over()) return 0;
                base = -32;
            }
        }
        // the lane's own channels.  Where a word between is missing, the nearest is looked
        // for again: a tile that knew its state at once has no (A, H)
        const ulonglong2 s = words_load(p.state + record(p, row + STEP * found, strip));
        bool all = known(s);
        uint64_t h = state_of(s);
        for (int d = found - 1; d > 0; d -= MANY) {
            ulonglong2 v[MANY];
#pragma unroll
            for (int i = 0; i < MANY; ++i)
                if (d - i > 0) v[i] = words_load(p.agg + record(p, row + STEP * (d - i), strip));
#pragma unroll
            for (int i = 0; i < MANY; ++i)
                if (d - i > 0) {
                    all = all && there(v[i]);
                    h = fma2(pair(lo_of(v[i].x), lo_of(v[i].y)), h,
                             pair(hi_of(v[i].x), hi_of(v[i].y)));
                }
            if (!__all_sync(0xffffffffu, all)) break;
        }
        if (__all_sync(0xffffffffu, all)) return h;
        if (patience.over()) return 0;
    }
}

// By the carrying warp, from the composition (all, sum) of a tile's tokens: publishes the
// state behind the tile and returns the one that enters it.  reset: a sequence starts
// inside, and `sum` is the state whatever enters; entered: whether one does.
template <int STEP>
__device__ __forceinline__ uint64_t pass_on(const Plan &p, int row, int strip, uint64_t all,
                                            uint64_t sum, bool reset, bool entered,
                                            const ulonglong2 &early) {
    if (p.alone) return 0;
    ulonglong2 *to = p.state + record(p, row, strip);
    if (reset || !entered) state_store(to, sum);
    if (!entered) return 0;
    ulonglong2 v = early;
    uint64_t h;
    if (!__all_sync(0xffffffffu, known(v))) {
        if (!reset)
            words_store(p.agg + record(p, row, strip), pair(lo_of(all), lo_of(sum)),
                        pair(hi_of(all), hi_of(sum)));
        for (int i = 0; i < LOOKS && !__all_sync(0xffffffffu, known(v)); ++i)
            v = words_load(p.state + record(p, row + STEP, strip));
    }
    if (__all_sync(0xffffffffu, known(v))) h = state_of(v);
    else h = look_back<STEP>(p, row, strip);
    if (!reset) state_store(to, fma2(all, h, sum));
    return h;
}

// before the tiles: no states known, no ticket given, the channels' logs of a
__global__ void __launch_bounds__(256) prepare_kernel(const Args a, const Plan p, int64_t vectors) {
    const int64_t step = (int64_t)gridDim.x * blockDim.x;
    const int64_t i0 = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    uint4 *state = reinterpret_cast<uint4 *>(p.state);
    for (int64_t i = i0; i < vectors; i += step) state[i] = make_uint4(0, 0, 0, 0);
    for (int64_t c = i0; c < (int64_t)p.strips * STRIP; c += step)
        p.log2a[c] = c < a.width ? log2_decay(a.decay[c], a.sharpness) : 0.0f;
}
template <bool WIDE>
__device__ __forceinline__ uint64_t log2_decays(const Args &a, const Plan &p,
                                                const Channels<WIDE> &ch) {
    if (!p.alone) return ch.load_all(p.log2a);
    const uint64_t v = ch.load(a.decay);
    return pack(log2_decay(lo(v), a.sharpness), log2_decay(hi(v), a.sharpness));
}
__device__ __forceinline__ float4 four(uint64_t a, uint64_t b) {
    return make_float4(lo(a), hi(a), lo(b), hi(b));
}
__device__ __forceinline__ float2 two(uint64_t a) { return make_float2(lo(a), hi(a)); }

// an empty sequence has no token to write its final state (its gradient): the CTAs of
// a strip share those
template <typename Shape, bool WIDE>
__device__ __forceinline__ void empty_sequences(const Args &a, const Plan &p, const Tile &t,
                                                const Channels<WIDE> &ch, const float *from,
                                                float *to) {
    const int w = threadIdx.x >> 5;
    for (int64_t s = t.row + (int64_t)p.rows * w; s < a.seqs; s += (int64_t)p.rows * Shape::WARPS)
        if (min(max((int64_t)a.cu[s], (int64_t)0), a.seqlen) >=
            min((int64_t)a.cu[s + 1], a.seqlen))
            ch.store(to + s * a.width, from ? ch.load(from + s * a.width) : 0);
}

// -------------------------------------------------------------------- forward
// The warps that hold tokens compute their a and b and put them aside in shared memory;
// the carrying warp composes the warps, publishes the tile's state and says which state
// enters each warp; then those write their rows.  The other CTAs of the SM work meanwhile.
template <typename T, typename Slot> struct ForwardSmem {
    using Shape = Forward<T>;
    Slot in[3][Shape::RUN][Shape::THREADS];
    float4 ab[Shape::RUN][Shape::THREADS];
    float4 agg[Shape::WARPS][32];
    float2 enter[Shape::WARPS][32];         // the states before the warps' tokens
    int reset[Shape::WARPS];                // bit 0: a first token, bit 1: the warp's own first
    Tile next;
    Places places;
};

__device__ __forceinline__ void barrier() { asm volatile("bar.sync 0;" ::: "memory"); }

template <typename T, bool WIDE>
__global__ void __launch_bounds__(Forward<T>::THREADS + 32, Forward<T>::CTAS)
forward_kernel(const Args a, const Plan p) {
    using Shape = Forward<T>;
    constexpr int RUN = Shape::RUN, WARPS = Shape::WARPS;
    using L = Lane<T, WIDE>;
    using Smem = ForwardSmem<T, typename L::Slot>;
    extern __shared__ __align__(16) char raw_smem[];
    Smem &sm = *reinterpret_cast<Smem *>(raw_smem);
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    auto ticket = [&] {
        return __shfl_sync(0xffffffffu, lane ? 0u : atomicAdd(p.ticket, 1u), 0);
    };
    if (w == WARPS)
        next_tile<T>(a, p, p.alone ? blockIdx.x : ticket(), Shape::TILE, false, &sm.next, &sm.places);
    barrier();
    Tile t = sm.next;
    if (t.row < 0) return;

    if (w == WARPS) {                         // carries the states
        barrier();
        for (;;) {
            next_tile<T>(a, p, p.alone ? NO_TILE : ticket(), Shape::TILE, false, &sm.next, &sm.places);
            const bool first_row = p.alone || t.row == 0 || (!a.cu && t.first == 0);
            ulonglong2 early{};
            if (!first_row) early = words_load(p.state + record(p, t.row - 1, t.strip));
            barrier();
            const int seen = lane < WARPS ? sm.reset[lane] : 0;
            const unsigned resets = __ballot_sync(0xffffffffu, seen & 1);
            uint64_t P = pair(1.0f), S = 0;
#pragma unroll
            for (int j = 0; j < WARPS; ++j) {
                const float4 v = sm.agg[j][lane];
                const uint64_t A = pack(v.x, v.y), H = pack(v.z, v.w);
                P = mul2(P, A);
                S = resets >> j & 1 ? H : fma2(A, S, H);
            }
            // (a sequence that starts with the tile takes no state from before)
            const bool entered = !first_row && !(__shfl_sync(0xffffffffu, seen, 0) & 2);
            uint64_t h = pass_on<-1>(p, t.row, t.strip, keep(P), S, resets != 0, entered, early);
#pragma unroll
            for (int j = 0; j < WARPS; ++j) {
                sm.enter[j][lane] = two(h);
                const float4 v = sm.agg[j][lane];
                h = resets >> j & 1 ? pack(v.z, v.w) : fma2(pack(v.x, v.y), h, pack(v.z, v.w));
            }
            t = sm.next;
            barrier();
            if (t.row < 0) return;
        }
    }

    const Factors k = Factors::set();
    const Rows rx(a.x, a.xs, a, p), ri(a.ig, a.is, a, p), rr(a.rg, a.rs, a, p);
    auto issue = [&](const Tile &t) {
        if (WIDE && t.plain) {
            using Slot = typename L::Slot;
            fetch_plain<Slot, Shape>(sm.places.in[0], p.stride[0], &sm.in[0][0][w * 32]);
            fetch_plain<Slot, Shape>(sm.places.in[1], p.stride[1], &sm.in[1][0][w * 32]);
            fetch_plain<Slot, Shape>(sm.places.in[2], p.stride[2], &sm.in[2][0][w * 32]);
            cp_async_commit();
            return;
        }
        const int g = t.first + w * RUN, n = t.count - w * RUN;
        fetch<T, WIDE, Shape>(rr, &sm.in[0][0][w * 32], p, t, g, n, a.width);
        fetch<T, WIDE, Shape>(ri, &sm.in[1][0][w * 32], p, t, g, n, a.width);
        fetch<T, WIDE, Shape>(rx, &sm.in[2][0][w * 32], p, t, g, n, a.width);
        cp_async_commit();
    };
    // bytes from a tile's first value of an output to the lane's
    const int64_t mine = (w * RUN * a.width + 2 * lane) * (int64_t)sizeof(T);
    issue(t);
    int64_t out = sm.places.out + mine;       // a plain tile's rows of the output
    barrier();
    for (;;) {
        const bool plain = WIDE && t.plain;
        const Channels<WIDE> ch(t.strip, lane, a.width);
        const int g = t.first + w * RUN, n = plain ? RUN : min(max(t.count - w * RUN, 0), RUN);
        Marks mk{};
        if (!plain) mk = marks_of(a, p, t, g, n);
        const uint64_t log2a = log2_decays(a, p, ch);
        // the warp's tokens: h -> A h + H, or to H alone from a first token on
        uint64_t A = pair(1.0f), H = 0;
        cp_async_wait<0>();
        __syncwarp();
        const unsigned or_ = odd_of<T, WIDE, Shape>(rr, p, t.axis, g, ch.c);
        const unsigned oi = odd_of<T, WIDE, Shape>(ri, p, t.axis, g, ch.c);
        const unsigned ox = odd_of<T, WIDE, Shape>(rx, p, t.axis, g, ch.c);
        FarGates<T, WIDE> far;
        auto compute = [&](auto is_mild, auto is_near, int j, uint64_t &da, uint64_t &db) {
            const uint64_t dr = one_plus_exp(value<T, WIDE>(sm.in[0][j][tid], or_, j), k);
            const uint64_t di = one_plus_exp(value<T, WIDE>(sm.in[1][j][tid], oi, j), k);
            const Decay e = decay_of<decltype(is_mild)::value>(
                mul2(log2a, pack(rcp(lo(dr)), rcp(hi(dr)))), k);
            da = e.a;
            if constexpr (decltype(is_near)::value) far.note(sm.in[1][j][tid], di);
            const uint64_t mi = decltype(is_near)::value ? near_input_factor(e.y, di)
                                                         : input_factor(e.y, di);
            db = mul2(mi, value<T, WIDE>(sm.in[2][j][tid], ox, j));
        };
        auto all = [&](auto is_mild) {
#pragma unroll
            for (int j = 0; j < RUN; ++j) {
                uint64_t da, db;
                compute(is_mild, std::true_type(), j, da, db);
                H = fma2(da, H, db);
                A = mul2(A, da);
                sm.ab[j][tid] = four(da, db);
            }
        };
        bool done = plain || (n == RUN && !(mk.first | mk.none));
        if (done) {
            if (mild(log2a)) all(std::true_type());
            else all(std::false_type());
            done = !far.some();
        }
        if (!done) {                          // a sequence's start, tokens of none, input
            A = pair(1.0f), H = 0;            // gates between -89 and -43
#pragma unroll 2
            for (int j = 0; j < RUN; ++j) {
                uint64_t da = pair(1.0f), db = 0;
                if (j < n && !(mk.none >> j & 1))
                    compute(std::false_type(), std::false_type(), j, da, db);
                if (mk.first >> j & 1) {
                    if (a.h0) db = fma2(da, ch.load(a.h0 + seq_of(mk, j) * a.width), db);
                    H = db;
                } else {
                    H = fma2(da, H, db);
                }
                A = mul2(A, da);
                sm.ab[j][tid] = four(da, db);
            }
        }
        sm.agg[w][lane] = four(keep(A), H);
        if (lane == 0) sm.reset[w] = (mk.first ? 1 : 0) | (mk.first & 1) << 1;
        barrier();
        const Tile next = sm.next;
        if (next.row >= 0) issue(next);
        const int64_t next_out = sm.places.out + mine;
        barrier();
        if (plain) {
            const float2 e = sm.enter[w][lane];
            uint64_t h = pack(e.x, e.y), v[RUN];
            if (a.saved && g % Backward<T>::TILE == 0)
                ch.store(a.saved + (t.axis * ceil_div(p.tokens, Backward<T>::TILE) +
                                    g / Backward<T>::TILE) * a.width, h);
#pragma unroll
            for (int j = 0; j < RUN; ++j) {
                const float4 ab = sm.ab[j][tid];
                v[j] = h = fma2(pack(ab.x, ab.y), h, pack(ab.z, ab.w));
            }
            put_plain<T>(a.h, out, a.width, v);
        } else if (n > 0) {
            const float2 e = sm.enter[w][lane];
            uint64_t h = pack(e.x, e.y), v[RUN];
            if (a.saved && g % Backward<T>::TILE == 0)
                ch.store(a.saved + (t.axis * ceil_div(p.tokens, Backward<T>::TILE) +
                                    g / Backward<T>::TILE) * a.width, h);
#pragma unroll
            for (int j = 0; j < RUN; ++j) {
                const float4 ab = sm.ab[j][tid];
                h = mk.first >> j & 1 ? pack(ab.z, ab.w)
                                      : fma2(pack(ab.x, ab.y), h, pack(ab.z, ab.w));
                v[j] = mk.none >> j & 1 ? 0 : h;
            }
            put_rows<T, WIDE>(a.h, (p.axes > 1 ? t.axis * a.seqlen : 0) + g, a.width, n, ch, v);
            if (mk.last && a.h_last) {
#pragma unroll
                for (int j = 0; j < RUN; ++j)
                    if (mk.last >> j & 1) ch.store(a.h_last + seq_of(mk, j) * a.width, v[j]);
            }
        }
        if (a.cu && a.h_last) empty_sequences<Shape>(a, p, t, ch, a.h0, a.h_last);
        t = next, out = next_out;
        if (t.row < 0) break;
    }
}

// ------------------------------------------------------------------- backward
template <typename T, typename Slot> struct BackwardSmem {
    using Shape = Backward<T>;
    Slot gates[2][Shape::RUN][Shape::THREADS];
    Slot xd[2][2][Shape::RUN][Shape::THREADS];       // x, dh; two tiles'
    // a, m i; m (1 - i), e^-v of the decay gate, and once the states are known 1 - i, 1 - r
    float4 kept[2][Shape::RUN][Shape::THREADS];
    float4 agg[Shape::WARPS][32];          // A, A and the states' H, H
    float2 back[Shape::WARPS][32];         // the gradients' H, H
    float4 enter[Shape::WARPS][32];        // h before the warps' tokens, C behind them
    float2 sums[Shape::WARPS][32];         // of d log a at an open gate
    int reset[Shape::WARPS];               // bit 0: a first token, 1: a last, 2: the last one's
    Tile next;
    Places places;
};

template <typename T, bool WIDE>
__global__ void __launch_bounds__(Backward<T>::THREADS + 32, Backward<T>::CTAS)
backward_kernel(const Args a, const Plan p) {
    using Shape = Backward<T>;
    constexpr int RUN = Shape::RUN, WARPS = Shape::WARPS;
    using L = Lane<T, WIDE>;
    using Smem = BackwardSmem<T, typename L::Slot>;
    extern __shared__ __align__(16) char raw_smem[];
    Smem &sm = *reinterpret_cast<Smem *>(raw_smem);
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    auto ticket = [&] {
        return __shfl_sync(0xffffffffu, lane ? 0u : atomicAdd(p.ticket, 1u), 0);
    };
    if (w == WARPS)
        next_tile<T>(a, p, p.alone ? blockIdx.x : ticket(), Shape::TILE, true, &sm.next, &sm.places);
    barrier();
    Tile t = sm.next;
    if (t.row < 0) return;

    if (w == WARPS) {                         // carries the gradients' C, adds up d log a
        barrier();
        auto add_up = [&](int row, int strip) {
            if (!a.ddecay) return;
            uint64_t s = 0;
#pragma unroll
            for (int j = 0; j < WARPS; ++j) {
                const float2 v = sm.sums[j][lane];
                s = add2(s, pack(v.x, v.y));
            }
            Channels<WIDE>(strip, lane, a.width).store(p.parts + (int64_t)row * a.width, s);
        };
        int done_row = -1, done_strip = 0;
        for (;;) {
            next_tile<T>(a, p, p.alone ? NO_TILE : ticket(), Shape::TILE, true, &sm.next, &sm.places);
            const bool last_row = p.alone || t.row + 1 == p.rows ||
                                  (!a.cu && t.first + t.count == p.tokens);
            const Channels<WIDE> ch(t.strip, lane, a.width);
            uint64_t h = ch.load(a.saved + (int64_t)t.row * a.width);  // before the tile
            ulonglong2 early{};
            if (!last_row) early = words_load(p.state + record(p, t.row + 1, t.strip));
            barrier();
            const int seen = lane < WARPS ? sm.reset[lane] : 0;
            const unsigned firsts = __ballot_sync(0xffffffffu, seen & 1);
            const unsigned lasts = __ballot_sync(0xffffffffu, seen & 2);
            uint64_t P = pair(1.0f), S = 0;
#pragma unroll
            for (int j = WARPS - 1; j >= 0; --j) {
                const float4 v = sm.agg[j][lane];
                const float2 b = sm.back[j][lane];
                const uint64_t A = pack(v.x, v.y), B = pack(b.x, b.y);
                P = mul2(P, A);
                S = lasts >> j & 1 ? B : fma2(A, S, B);
            }
            // (none comes from behind where a sequence ends with the tile)
            const bool entered = !last_row && !__any_sync(0xffffffffu, seen & 4);
            uint64_t c = pass_on<1>(p, t.row, t.strip, keep(P), S, lasts != 0, entered, early);
            float2 *enter = reinterpret_cast<float2 *>(&sm.enter[0][lane]);
#pragma unroll
            for (int j = 0; j < WARPS; ++j) {
                enter[j * 64] = two(h);
                const float4 v = sm.agg[j][lane];
                h = firsts >> j & 1 ? pack(v.z, v.w) : fma2(pack(v.x, v.y), h, pack(v.z, v.w));
            }
#pragma unroll
            for (int j = WARPS - 1; j >= 0; --j) {
                enter[j * 64 + 1] = two(c);
                const float4 v = sm.agg[j][lane];
                const float2 b = sm.back[j][lane];
                c = lasts >> j & 1 ? pack(b.x, b.y) : fma2(pack(v.x, v.y), c, pack(b.x, b.y));
            }
            if (done_row >= 0) add_up(done_row, done_strip);           // of the tile before
            done_row = t.row, done_strip = t.strip;
            t = sm.next;
            barrier();
            if (t.row < 0) break;
        }
        barrier();
        add_up(done_row, done_strip);
        return;
    }

    const Factors k = Factors::set();
    const Rows rx(a.x, a.xs, a, p), ri(a.ig, a.is, a, p), rr(a.rg, a.rs, a, p);
    const Rows rd(a.dh, a.ds, a, p);
    auto issue = [&](const Tile &t, int par) {
        if (WIDE && t.plain) {
            using Slot = typename L::Slot;
            fetch_plain<Slot, Shape>(sm.places.in[0], p.stride[0], &sm.gates[0][0][w * 32]);
            fetch_plain<Slot, Shape>(sm.places.in[1], p.stride[1], &sm.gates[1][0][w * 32]);
            fetch_plain<Slot, Shape>(sm.places.in[2], p.stride[2], &sm.xd[par][0][0][w * 32]);
            if (a.dh)
                fetch_plain<Slot, Shape>(sm.places.in[3], p.stride[3], &sm.xd[par][1][0][w * 32]);
            cp_async_commit();
            return;
        }
        const int g = t.first + w * RUN, n = t.count - w * RUN;
        fetch<T, WIDE, Shape>(rr, &sm.gates[0][0][w * 32], p, t, g, n, a.width);
        fetch<T, WIDE, Shape>(ri, &sm.gates[1][0][w * 32], p, t, g, n, a.width);
        fetch<T, WIDE, Shape>(rx, &sm.xd[par][0][0][w * 32], p, t, g, n, a.width);
        if (a.dh) fetch<T, WIDE, Shape>(rd, &sm.xd[par][1][0][w * 32], p, t, g, n, a.width);
        cp_async_commit();
    };
    // bytes from a tile's first value of an output to the lane's
    const int64_t mine = (w * RUN * a.width + 2 * lane) * (int64_t)sizeof(T);
    issue(t, 0);
    int64_t out = sm.places.out + mine;       // a plain tile's rows of the outputs
    barrier();
    for (int par = 0;; par ^= 1) {
        const Channels<WIDE> ch(t.strip, lane, a.width);
        const bool whole = WIDE && t.plain;
        const int g = t.first + w * RUN, n = whole ? RUN : min(max(t.count - w * RUN, 0), RUN);
        Marks mk{};
        if (!whole) mk = marks_of(a, p, t, g, n);
        const uint64_t log2a = log2_decays(a, p, ch);
        const unsigned ox = odd_of<T, WIDE, Shape>(rx, p, t.axis, g, ch.c);
        const unsigned od = odd_of<T, WIDE, Shape>(rd, p, t.axis, g, ch.c);
        const unsigned or_ = odd_of<T, WIDE, Shape>(rr, p, t.axis, g, ch.c);
        const unsigned oi = odd_of<T, WIDE, Shape>(ri, p, t.axis, g, ch.c);
        typename L::Slot (&xs)[RUN][Shape::THREADS] = sm.xd[par][0];
        typename L::Slot (&ds)[RUN][Shape::THREADS] = sm.xd[par][1];
        cp_async_wait<0>();
        __syncwarp();
        // the states: h -> A h + H, or to H alone; the gradients' C from the later tokens:
        // C -> A C + B, or to B alone before a last one
        uint64_t A = pair(1.0f), H = 0, B = 0, da[RUN];
        // a, m i, m (1 - i) and e^-v of the decay gate of a token
        auto compute = [&](auto is_mild, int j, uint64_t &mi, uint64_t &mo, uint64_t &er) {
            er = exp_neg(value<T, WIDE>(sm.gates[0][j][tid], or_, j), k);
            const uint64_t ei = exp_neg(value<T, WIDE>(sm.gates[1][j][tid], oi, j), k);
            const Decay e = decay_of<decltype(is_mild)::value>(
                mul2(log2a, rcp2(add2(er, k.one))), k);
            // m, or 0 where it is below 1e-18: nothing comes back through a closed gate (an
            // m^2 that is not normal would be 0 to the root, and 1 / m infinite)
            const uint64_t m = mul2(e.y, pack(lo(e.y) < kTiny ? 0.0f : rsq(lo(e.y)),
                                              hi(e.y) < kTiny ? 0.0f : rsq(hi(e.y))));
            const uint64_t i = rcp2(add2(ei, k.one));
            mi = mul2(m, i);
            mo = mul2(m, rest_of(ei, i));
            return e.a;
        };
        const bool plain = whole || (n == RUN && !(mk.first | mk.last | mk.none));
        auto all = [&](auto is_mild) {
#pragma unroll
            for (int j = 0; j < RUN; ++j) {
                uint64_t mi, mo, er;
                da[j] = compute(is_mild, j, mi, mo, er);
                H = fma2(da[j], H, mul2(mi, value<T, WIDE>(xs[j][tid], ox, j)));
                A = mul2(A, da[j]);
                sm.kept[0][j][tid] = four(da[j], mi);
                sm.kept[1][j][tid] = four(mo, er);
            }
#pragma unroll
            for (int j = RUN - 1; j >= 0; --j)
                B = mul2(da[j], add2(B, value<T, WIDE>(ds[j][tid], od, j)));
        };
        if (plain && a.dh) {
            if (mild(log2a)) all(std::true_type());
            else all(std::false_type());
        } else {
#pragma unroll 2
            for (int j = 0; j < RUN; ++j) {
                uint64_t a1 = pair(1.0f), mi = 0, mo = 0, er = 0;
                if (j >= n || (mk.none >> j & 1)) xs[j][tid] = ds[j][tid] = 0;
                else a1 = compute(std::false_type(), j, mi, mo, er);
                if (!a.dh) ds[j][tid] = 0;
                const uint64_t b = mul2(mi, value<T, WIDE>(xs[j][tid], ox, j));
                if (mk.first >> j & 1) {
                    H = b;
                    if (a.h0) H = fma2(a1, ch.load(a.h0 + seq_of(mk, j) * a.width), H);
                } else {
                    H = fma2(a1, H, b);
                }
                A = mul2(A, a1);
                sm.kept[0][j][tid] = four(a1, mi);
                sm.kept[1][j][tid] = four(mo, er);
            }
#pragma unroll 2
            for (int j = RUN - 1; j >= 0; --j) {
                if (mk.last >> j & 1) B = a.dlast ? ch.load(a.dlast + seq_of(mk, j) * a.width) : 0;
                const float2 a1 = *reinterpret_cast<const float2 *>(&sm.kept[0][j][tid]);
                B = mul2(pack(a1.x, a1.y), add2(B, value<T, WIDE>(ds[j][tid], od, j)));
            }
        }
        sm.agg[w][lane] = four(keep(A), H);
        sm.back[w][lane] = two(B);
        if (lane == 0)
            sm.reset[w] = (mk.first ? 1 : 0) | (mk.last ? 2 : 0) |
                          (n && t.count <= (w + 1) * RUN && (mk.last >> (n - 1) & 1) ? 4 : 0);
        barrier();
        const Tile next = sm.next;
        if (next.row >= 0) issue(next, par ^ 1);
        const int64_t next_out = sm.places.out + mine;
        barrier();
        uint64_t total = 0;
        if (n > 0) {
            const float4 e = sm.enter[w][lane];
            const uint64_t g1 = mul2(log2a, pair(0.6931471824645996f));
            uint64_t h = pack(e.x, e.y), C = pack(e.z, e.w);
            // beside G the outputs need m i, x (1 - i), q = r (a h_{t-1} - a^2 i x / m) and
            // g1 (1 - r); m is the sum of its two parts
            uint64_t q[RUN];
            auto take = [&](int j) {
                const float4 am = sm.kept[0][j][tid], mr = sm.kept[1][j][tid];
                const uint64_t a1 = pack(am.x, am.y), mi = pack(am.z, am.w);
                const uint64_t mo = pack(mr.x, mr.y), er = pack(mr.z, mr.w);
                const uint64_t b = mul2(mi, value<T, WIDE>(xs[j][tid], ox, j));
                const uint64_t rm = rcp2(add2(add2(mi, mo), pair(kFloor)));
                const uint64_t r = rcp2(add2(er, k.one));
                // h - a i x / m
                const uint64_t less = fma2(mul2(a1, mul2(mul2(b, rm), rm)), k.neg_one, h);
                q[j] = mul2(mul2(r, a1), less);
                sm.kept[1][j][tid] = four(mul2(mo, rm), rest_of(er, r));
                h = fma2(a1, h, b);
            };
            uint64_t dx[RUN], di[RUN], dr[RUN];
            auto give = [&](int j) {
                const float4 am = sm.kept[0][j][tid], rest = sm.kept[1][j][tid];
                const uint64_t x = value<T, WIDE>(xs[j][tid], ox, j);
                const uint64_t G = add2(C, value<T, WIDE>(ds[j][tid], od, j));
                const uint64_t dl = mul2(G, q[j]);
                dx[j] = mul2(G, pack(am.z, am.w));
                di[j] = mul2(dx[j], mul2(x, pack(rest.x, rest.y)));
                dr[j] = mul2(dl, mul2(g1, pack(rest.z, rest.w)));
                total = add2(total, dl);
                C = mul2(pack(am.x, am.y), G);
            };
            if (plain) {
#pragma unroll
                for (int j = 0; j < RUN; ++j) take(j);
#pragma unroll
                for (int j = RUN - 1; j >= 0; --j) give(j);
            } else {
#pragma unroll
                for (int j = 0; j < RUN; ++j) {
                    if (mk.first >> j & 1) h = a.h0 ? ch.load(a.h0 + seq_of(mk, j) * a.width) : 0;
                    take(j);
                }
#pragma unroll
                for (int j = RUN - 1; j >= 0; --j) {
                    if (mk.last >> j & 1)
                        C = a.dlast ? ch.load(a.dlast + seq_of(mk, j) * a.width) : 0;
                    dx[j] = di[j] = dr[j] = 0;
                    if (j < n && !(mk.none >> j & 1)) give(j);
                    if ((mk.first >> j & 1) && a.dh0)
                        ch.store(a.dh0 + seq_of(mk, j) * a.width, C);
                }
            }
            if (whole) {
                if (a.dx) put_plain<T>(a.dx, out, a.width, dx);
                if (a.dig) put_plain<T>(a.dig, out, a.width, di);
                if (a.drg) put_plain<T>(a.drg, out, a.width, dr);
            } else {
                const int64_t token = (p.axes > 1 ? t.axis * a.seqlen : 0) + g;
                if (a.dx) put_rows<T, WIDE>(a.dx, token, a.width, n, ch, dx);
                if (a.dig) put_rows<T, WIDE>(a.dig, token, a.width, n, ch, di);
                if (a.drg) put_rows<T, WIDE>(a.drg, token, a.width, n, ch, dr);
            }
        }
        sm.sums[w][lane] = two(total);
        if (a.cu && a.dh0) empty_sequences<Shape>(a, p, t, ch, a.dlast, a.dh0);
        t = next, out = next_out;
        if (t.row < 0) break;
    }
    barrier();
}

// ddecay = -sharpness sigmoid(decay) sum of the tiles' parts, in 64 bits and in order:
// 32 channels x 32 runs of rows a CTA
__global__ void __launch_bounds__(1024) decay_grad_kernel(const Args a, const float *parts,
                                                          int rows) {
    __shared__ double sums[32][33];
    const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
    double s = 0.0;
    if (c < a.width) {
#pragma unroll 8
        for (int r = threadIdx.y; r < rows; r += 32) s += parts[(int64_t)r * a.width + c];
    }
    sums[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y || c >= a.width) return;
    for (int y = 1; y < 32; ++y) s += sums[y][threadIdx.x];
    a.ddecay[c] = (float)(-(double)a.sharpness * s / (1.0 + exp(-(double)a.decay[c])));
}

// ------------------------------------------------------------------- one token
// One token.  A thread has V channels (4, moved together, where all rows allow it) of
// every gridDim.y-th sequence, whose decays it works out once; the next sequence's
// values are on their way while one is computed.  Bound by HBM.
template <typename T, int V> struct Few;
template <typename T> struct Few<T, 1> {
    float v[1];
    __device__ __forceinline__ void load(const T *p) { v[0] = io<T>::to_f(*p); }
    __device__ __forceinline__ void store(T *p) const { *p = io<T>::from_f(v[0]); }
};
template <> struct Few<float, 4> {
    float v[4];
    __device__ __forceinline__ void load(const float *p) {
        const float4 f = *reinterpret_cast<const float4 *>(p);
        v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    }
    __device__ __forceinline__ void store(float *p) const {
        *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    }
};
template <> struct Few<__nv_bfloat16, 4> {
    float v[4];
    __device__ __forceinline__ void load(const __nv_bfloat16 *p) {
        const uint2 f = *reinterpret_cast<const uint2 *>(p);
        v[0] = __uint_as_float(f.x << 16), v[1] = __uint_as_float(f.x & 0xffff0000u);
        v[2] = __uint_as_float(f.y << 16), v[3] = __uint_as_float(f.y & 0xffff0000u);
    }
    __device__ __forceinline__ void store(__nv_bfloat16 *p) const {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]);
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2], v[3]);
        *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a),
                                                   *reinterpret_cast<const uint32_t *>(&b));
    }
};

constexpr int STEP_THREADS = 128;
template <typename T, int V>
__global__ void __launch_bounds__(STEP_THREADS) step_kernel(const Args a, float *state) {
    const int64_t c = ((int64_t)blockIdx.x * STEP_THREADS + threadIdx.x) * V;
    if (c >= a.width) return;
    struct Token {
        Few<T, V> x, i, r;
        Few<float, V> h;
    };
    auto load = [&](int64_t b) {
        Token q;
        q.r.load(static_cast<const T *>(a.rg) + b * a.rs[0] + c);
        q.i.load(static_cast<const T *>(a.ig) + b * a.is[0] + c);
        q.x.load(static_cast<const T *>(a.x) + b * a.xs[0] + c);
        q.h.load(state + b * a.width + c);
        return q;
    };
    int64_t b = blockIdx.y;
    Token q = load(b);
    float u[V];
#pragma unroll
    for (int e = 0; e < V; ++e) u[e] = log2_decay(a.decay[c + e], a.sharpness);
    const Factors k = Factors::set();
    for (;;) {
        const int64_t next = b + gridDim.y;
        Token ahead;
        if (next < a.batch) ahead = load(next);
        Few<T, V> out;
#pragma unroll
        for (int e = 0; e < V; e += 2) {
            constexpr int o = V > 1;            // the second of two channels, or the same one
            const uint64_t dr = one_plus_exp(pack(q.r.v[e], q.r.v[e + o]), k);
            const uint64_t di = one_plus_exp(pack(q.i.v[e], q.i.v[e + o]), k);
            const Decay d = decay_of<false>(mul2(pack(u[e], u[e + o]),
                                                 pack(rcp(lo(dr)), rcp(hi(dr)))), k);
            const uint64_t h = fma2(d.a, pack(q.h.v[e], q.h.v[e + o]),
                                    mul2(input_factor(d.y, di), pack(q.x.v[e], q.x.v[e + o])));
            q.h.v[e] = out.v[e] = lo(h);
            q.h.v[e + o] = out.v[e + o] = o ? hi(h) : lo(h);
        }
        q.h.store(state + b * a.width + c);
        out.store(static_cast<T *>(a.h) + b * a.width + c);
        if (next >= a.batch) break;
        b = next, q = ahead;
    }
}

int check(const char *what, const mb2_gated_rec *d, bool tokens, Args &a) {
    MB2_REQUIRE(d, MB2_ERR_ARG, "%s: null descriptor", what);
    MB2_REQUIRE(d->dtype == MB2_F32 || d->dtype == MB2_BF16, MB2_ERR_ARG, "%s: bad dtype", what);
    MB2_REQUIRE(d->batch >= 0 && (!tokens || d->seqlen >= 0) && d->width > 0, MB2_ERR_SHAPE,
                "%s: bad size", what);
    MB2_REQUIRE(d->sharpness > 0.0f && d->sharpness < 1e30f, MB2_ERR_ARG,
                "%s: sharpness must be positive and finite", what);
    MB2_REQUIRE(!tokens || !d->cu_seqlens || (d->batch == 1 && d->n_seqs >= 0), MB2_ERR_SHAPE,
                "%s: cu_seqlens needs a batch of 1", what);
    constexpr int64_t kMost = (1ll << 31) - 4096;
    MB2_REQUIRE(d->batch < kMost && d->width < kMost && (!tokens || (d->seqlen < kMost &&
                (d->batch == 0 || d->seqlen < kMost / d->batch) && d->n_seqs < kMost)),
                MB2_ERR_SHAPE, "%s: more than 2^31 tokens, channels or sequences", what);
    a = Args{};
    a.x = d->x, a.ig = d->input_gate, a.rg = d->decay_gate, a.decay = d->decay;
    a.sharpness = d->sharpness;
    for (int i = 0; i < 2; ++i) {
        a.xs[i] = d->x_stride[i], a.is[i] = d->input_gate_stride[i];
        a.rs[i] = d->decay_gate_stride[i], a.ds[i] = d->dh_stride[i];
    }
    a.h0 = d->h0, a.cu = tokens ? d->cu_seqlens : nullptr;
    a.batch = d->batch, a.seqlen = tokens ? d->seqlen : 1, a.width = d->width;
    a.seqs = a.cu ? d->n_seqs : d->batch;
    a.h = d->h, a.h_last = d->h_last, a.saved = d->saved;
    a.dh = d->dh, a.dlast = d->dh_last, a.dx = d->dx, a.dig = d->dinput_gate;
    a.drg = d->ddecay_gate, a.ddecay = d->ddecay, a.dh0 = d->dh0;
    return MB2_OK;
}

// whether a tensor's rows are multiples of 16 bytes
bool wide(const void *p, const int64_t (&s)[2], int dtype) {
    const int64_t n = 16 / (int64_t)dtype_size(dtype);
    return !p || (aligned(p, 16) && s[0] % n == 0 && s[1] % n == 0);
}
bool all_wide(const Args &a, int dtype) {
    const int64_t own[2] = {a.width, a.width};
    return wide(a.x, a.xs, dtype) && wide(a.ig, a.is, dtype) && wide(a.rg, a.rs, dtype) &&
           wide(a.dh, a.ds, dtype) && a.width % (16 / (int64_t)dtype_size(dtype)) == 0 &&
           wide(a.h, own, dtype) && wide(a.dx, own, dtype) && wide(a.dig, own, dtype) &&
           wide(a.drg, own, dtype);
}

// the current device's SMs, asked for once a device
int sms_of(int dev, int &sms) {
    static std::atomic<int> seen[64];
    sms = dev < 64 ? seen[dev].load(std::memory_order_relaxed) : 0;
    if (sms) return MB2_OK;
    const cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    MB2_REQUIRE(e == cudaSuccess, MB2_ERR_CUDA, "gated_recurrence: %s", cudaGetErrorString(e));
    if (dev < 64) seen[dev].store(sms, std::memory_order_relaxed);
    return MB2_OK;
}

// The kernel's launch on as many CTAs as the device holds, or as there are tiles.
template <typename Shape, void (*KERN)(Args, Plan)>
int launch(const char *what, size_t smem, const Args &a, const Plan &p, cudaStream_t st) {
    static std::atomic<uint64_t> ready;       // devices that know of its shared memory
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    MB2_REQUIRE(e == cudaSuccess, MB2_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
    MB2_TRY(sms_of(dev, sms));
    if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
        e = cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        MB2_REQUIRE(e == cudaSuccess, MB2_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
        if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    const int64_t tiles = (int64_t)p.rows * p.strips;
    if (!p.alone) {
        const int64_t vectors = (reinterpret_cast<char *>(p.ticket + 4) -
                                 reinterpret_cast<char *>(p.state)) / 16;
        const int64_t blocks = ceil_div(vectors, 1024) + p.strips / 16;
        prepare_kernel<<<(unsigned)std::min<int64_t>(blocks, sms * 8), 256, 0, st>>>(a, p, vectors);
        MB2_TRY(check_launch(what));
    }
    const int64_t ctas = p.alone ? tiles : std::min<int64_t>(tiles, (int64_t)sms * Shape::CTAS);
    KERN<<<(unsigned)ctas, Shape::THREADS + 32, smem, st>>>(a, p);
    return check_launch(what);
}
// a tile's offsets fit 32 bits
template <typename T> void set_lean(const Args &a, Plan &p, bool wide) {
    const int64_t strides[4] = {a.rs[1], a.is[1], a.xs[1], a.ds[1]};
    constexpr int64_t kMost = (1ll << 30) / 128 / sizeof(T);          // tiles are up to 104 tokens
    p.lean = wide && a.width < kMost;
    for (int k = 0; k < 4; ++k) {
        p.lean = p.lean && strides[k] < kMost && strides[k] > -kMost;
        p.stride[k] = p.lean ? (int)(strides[k] * (int64_t)sizeof(T)) : 0;
    }
}
template <typename T, bool WIDE> int run_forward(const Args &a, Plan p, cudaStream_t st) {
    set_lean<T>(a, p, WIDE);
    return launch<Forward<T>, forward_kernel<T, WIDE>>(
        "gated_recurrence", sizeof(ForwardSmem<T, typename Lane<T, WIDE>::Slot>), a, p, st);
}
template <typename T, bool WIDE> int run_backward(const Args &a, Plan p, cudaStream_t st) {
    set_lean<T>(a, p, WIDE);
    return launch<Backward<T>, backward_kernel<T, WIDE>>(
        "gated_recurrence_backward", sizeof(BackwardSmem<T, typename Lane<T, WIDE>::Slot>), a, p, st);
}

// Final states (their gradients) of a call without tokens: the initial ones.
int no_tokens(const char *what, const Args &a, const float *from, float *to, cudaStream_t st) {
    const size_t n = (size_t)(a.seqs * a.width) * 4;
    cudaError_t e = cudaSuccess;
    if (to && n)
        e = from ? cudaMemcpyAsync(to, from, n, cudaMemcpyDeviceToDevice, st)
                 : cudaMemsetAsync(to, 0, n, st);
    MB2_REQUIRE(e == cudaSuccess, MB2_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
    return MB2_OK;
}

}  // namespace

// this file's part of mb2_device_status
int rec_status(int *code, int clear) {
    cudaError_t e = cudaMemcpyFromSymbol(code, g_error, sizeof(int));
    if (e == cudaSuccess && clear) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_error, &zero, sizeof(int));
    }
    MB2_REQUIRE(e == cudaSuccess, MB2_ERR_CUDA, "device_status: %s", cudaGetErrorString(e));
    return MB2_OK;
}

}  // namespace rec
}  // namespace mb2

using namespace mb2;
using namespace mb2::rec;

extern "C" size_t mb2_gated_recurrence_saved_bytes(const mb2_gated_rec *d) {
    Args a;
    if (check("gated_recurrence_saved_bytes", d, true, a) != MB2_OK) return 0;
    return (size_t)plan_of<Backward>(a, d->dtype).rows * a.width * 4;
}

extern "C" size_t mb2_gated_recurrence_workspace_bytes(const mb2_gated_rec *d, int backward) {
    Args a;
    if (check("gated_recurrence_workspace_bytes", d, true, a) != MB2_OK) return 0;
    Plan p = backward ? plan_of<Backward>(a, d->dtype) : plan_of<Forward>(a, d->dtype);
    return p.rows ? lay_out(p, nullptr, a.width, backward) : 0;
}

extern "C" int mb2_gated_recurrence(const mb2_gated_rec *d, void *ws, size_t ws_bytes,
                                    mb2_stream_t stream) {
    const char *what = "gated_recurrence";
    Args a;
    MB2_TRY(check(what, d, true, a));
    cudaStream_t st = (cudaStream_t)stream;
    Plan p = plan_of<Forward>(a, d->dtype);
    if (p.rows == 0) return no_tokens(what, a, a.h0, a.h_last, st);
    MB2_REQUIRE(a.x && a.ig && a.rg && a.decay && a.h, MB2_ERR_ARG, "%s: null pointer", what);
    MB2_REQUIRE((int64_t)p.rows * p.strips < (1ll << 31), MB2_ERR_SHAPE, "%s: too many tiles", what);
    const size_t need = lay_out(p, ws, a.width, false);
    MB2_REQUIRE((ws || !need) && ws_bytes >= need, MB2_ERR_WORKSPACE, "%s: workspace of %zu bytes, needs %zu",
                what, ws_bytes, need);
    MB2_REQUIRE(aligned(ws, 256), MB2_ERR_ALIGN, "%s: workspace not 256-byte aligned", what);
    const bool whole = all_wide(a, d->dtype);
    if (d->dtype == MB2_F32)
        return whole ? run_forward<float, true>(a, p, st) : run_forward<float, false>(a, p, st);
    return whole ? run_forward<__nv_bfloat16, true>(a, p, st)
                 : run_forward<__nv_bfloat16, false>(a, p, st);
}

extern "C" int mb2_gated_recurrence_backward(const mb2_gated_rec *d, void *ws, size_t ws_bytes,
                                             mb2_stream_t stream) {
    const char *what = "gated_recurrence_backward";
    Args a;
    MB2_TRY(check(what, d, true, a));
    cudaStream_t st = (cudaStream_t)stream;
    Plan p = plan_of<Backward>(a, d->dtype);
    if (p.rows == 0) {
        if (a.ddecay) {
            const cudaError_t e = cudaMemsetAsync(a.ddecay, 0, a.width * 4, st);
            MB2_REQUIRE(e == cudaSuccess, MB2_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
        }
        return no_tokens(what, a, a.dlast, a.dh0, st);
    }
    MB2_REQUIRE(a.x && a.ig && a.rg && a.decay && a.saved, MB2_ERR_ARG, "%s: null pointer", what);
    MB2_REQUIRE((int64_t)p.rows * p.strips < (1ll << 31), MB2_ERR_SHAPE, "%s: too many tiles", what);
    const size_t need = lay_out(p, ws, a.width, true);
    MB2_REQUIRE((ws || !need) && ws_bytes >= need, MB2_ERR_WORKSPACE, "%s: workspace of %zu bytes, needs %zu",
                what, ws_bytes, need);
    MB2_REQUIRE(aligned(ws, 256), MB2_ERR_ALIGN, "%s: workspace not 256-byte aligned", what);
    const bool whole = all_wide(a, d->dtype);
    if (d->dtype == MB2_F32)
        MB2_TRY((whole ? run_backward<float, true> : run_backward<float, false>)(a, p, st));
    else
        MB2_TRY((whole ? run_backward<__nv_bfloat16, true>
                       : run_backward<__nv_bfloat16, false>)(a, p, st));
    if (!a.ddecay) return MB2_OK;
    decay_grad_kernel<<<(unsigned)ceil_div(a.width, 32), dim3(32, 32), 0, st>>>(a, p.parts, p.rows);
    return check_launch(what);
}

extern "C" int mb2_gated_recurrence_step(const mb2_gated_rec *d, float *state,
                                         mb2_stream_t stream) {
    Args a;
    MB2_TRY(check("gated_recurrence_step", d, false, a));
    if (a.batch == 0) return MB2_OK;
    MB2_REQUIRE(a.x && a.ig && a.rg && a.decay && a.h && state, MB2_ERR_ARG,
                "gated_recurrence_step: null pointer");
    cudaStream_t st = (cudaStream_t)stream;
    // rows of 4 channels at 4 elements' alignment
    const int64_t bytes = 4 * (int64_t)dtype_size(d->dtype);
    auto fours = [&](const void *p, int64_t ld) { return aligned(p, bytes) && ld % 4 == 0; };
    const bool wide = a.width % 4 == 0 && fours(a.x, a.xs[0]) && fours(a.ig, a.is[0]) &&
                      fours(a.rg, a.rs[0]) && fours(a.h, 0) && aligned(state, 16);
    // as many sequences side by side as fill the SMs (2048 threads each)
    const int64_t across = ceil_div(a.width, STEP_THREADS * (wide ? 4 : 1));
    const int64_t down = std::max<int64_t>(1, 148 * 16 / across);
    const dim3 grid((unsigned)across, (unsigned)std::min<int64_t>({a.batch, down, 65535}));
    if (d->dtype == MB2_F32) {
        if (wide) step_kernel<float, 4><<<grid, STEP_THREADS, 0, st>>>(a, state);
        else step_kernel<float, 1><<<grid, STEP_THREADS, 0, st>>>(a, state);
    } else {
        if (wide) step_kernel<__nv_bfloat16, 4><<<grid, STEP_THREADS, 0, st>>>(a, state);
        else step_kernel<__nv_bfloat16, 1><<<grid, STEP_THREADS, 0, st>>>(a, state);
    }
    return check_launch("gated_recurrence_step");
}
