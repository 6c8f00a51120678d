// Decay attention, shared by its kernels: the arguments of a call and the rows
// of a sequence.
#pragma once

#include "common.cuh"

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

// decay_tc.cu: the tensor-core prompt kernel; *used = false (and nothing
// launched) when it does not take the call
int chunked(const Args &a, cudaStream_t st, bool *used);

}  // namespace decay
}  // namespace mb2
