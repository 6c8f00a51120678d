// Decay attention, shared by its kernels: the arguments of a call and the rows
// of a sequence.
#pragma once

#include "common.cuh"
#include "pair.cuh"

namespace mb2 {
namespace decay {

struct Args {
    int dtype;
    int64_t seqs, seqlen;                 // sequences; tokens (packed: of all of them)
    int64_t heads, dk, dv;
    int q_rep, k_rep, v_rep;              // heads per q, k and v head
    const void *q, *k, *v;
    const float *g;
    void *o;
    int64_t qs[3], ks[3], vs[3], gs[3], os[3];   // strides: batch, token, head
    const float *h0;                      // (seqs, heads, dk, dv) or null
    float *h_last;                        // same, or null
    const int32_t *cu;                    // seqs + 1 offsets of packed sequences, or null
    float scale;
    int recurrent;                        // not for the tensor cores
    int narrow;                           // recurrent: a state spread over more lanes
    // A sequence may be walked in segments of `seg` tokens (0: whole) side by side:
    // a first pass leaves every segment's own final state (from 0) and the sum of
    // its log decays, seg_states turns them into the segments' initial states, and
    // a second pass computes the outputs.  A segment has a slot in the workspace.
    int64_t seg;
    int64_t slots;                        // segments of all sequences (packed: at most)
    const int32_t *slot0;                 // packed: seqs + 1, a sequence's first slot
    float *seg_state;                     // (slots, heads, dk, dv)
    double *seg_g;                        // (slots, heads)
};

// one walk of a kernel: a sequence, or a segment of it
struct Span {
    int64_t seq, row0, len;
    int64_t in, out;                      // state to start from (-1: 0) and to leave (-1: none)
};

__device__ __forceinline__ int64_t clamp_row(int64_t r, int64_t n) {
    return r < 0 ? 0 : (r > n ? n : r);
}
// first row and length of sequence `seq`; offsets outside [0, seqlen] or in
// the wrong order give rows inside the tensors
__device__ __forceinline__ void bounds(const Args &a, int64_t seq, int64_t &row0, int64_t &len) {
    if (a.cu) {
        row0 = clamp_row(a.cu[seq], a.seqlen);
        const int64_t end = clamp_row(a.cu[seq + 1], a.seqlen);
        len = end > row0 ? end - row0 : 0;
    } else {
        row0 = 0;
        len = a.seqlen;
    }
}
// segments of a sequence of len tokens (1 when it is empty)
__host__ __device__ __forceinline__ int64_t segments(int64_t len, int64_t seg) {
    return len > seg ? (len + seg - 1) / seg : 1;
}
// span `id` (a sequence, or a slot when there are segments).  STATE: the pass
// that leaves the segments' own states; a sequence's last one is not asked for.
template <bool STATE>
__device__ __forceinline__ Span span_of(const Args &a, int64_t id) {
    Span p;
    if (a.seg == 0) {
        p.seq = id;
        bounds(a, id, p.row0, p.len);
        p.in = a.h0 ? id : -1;
        p.out = a.h_last ? id : -1;
        return p;
    }
    int64_t j, n;
    if (a.cu) {
        int64_t lo = 0, hi = a.seqs;      // the last sequence whose first slot is <= id
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) >> 1;
            if (a.slot0[mid] <= id) lo = mid;
            else hi = mid;
        }
        p.seq = lo;
        j = id - a.slot0[lo];
        n = a.slot0[lo + 1] - a.slot0[lo];
    } else {
        n = segments(a.seqlen, a.seg);
        p.seq = id / n;
        j = id - p.seq * n;
    }
    bounds(a, p.seq, p.row0, p.len);
    const bool last = j == n - 1, valid = j < n && (!STATE || !last);
    p.row0 += j * a.seg;
    p.len -= j * a.seg;
    if (p.len > a.seg) p.len = a.seg;
    if (!valid) p.len = 0;
    p.in = STATE ? -1 : id;
    p.out = !valid ? -1 : STATE ? id : last && a.h_last ? p.seq : -1;
    return p;
}
inline int64_t spans(const Args &a) { return a.seg ? a.slots : a.seqs; }

// decay_tc.cu: the tensor-core prompt kernel; *used = false (and nothing
// launched) when it does not take the call
int chunked(const Args &a, bool state_only, cudaStream_t st, bool *used);
// whether it takes calls like this one (as far as the strides tell)
bool chunked_fits(const Args &a);
int num_sms();

}  // namespace decay
}  // namespace mb2
