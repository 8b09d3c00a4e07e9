// paged.cuh - what the kernels over the paged cache share: a step's sequences, and packing.
#pragma once
#include "common.cuh"
#include "kernels.h"

namespace mgpu_dev {

// Contents that a kernel skipped.  An expired wait, already recorded or still to come, has the word: its
// output is invalid, and its tickets are not all counted.
__device__ __forceinline__ void report_contents(int* status) { atomicCAS(status, 0, (int)MGPU_ERR_INVALID_ARG); }

template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The sequence that activation row t belongs to: the last b with cu_q[b] <= t, if t < cu_q[b+1];
// else -1.  All 32 lanes of a warp call it with the same t; each round tests 32 splits of the
// remaining range, so 1024 sequences take two dependent loads.
__device__ __forceinline__ int seq_of_token(const mgpu_k::PagedBatch& b, int t) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = b.n_seqs;  // the answer, if any, is in [lo, lo + n)
    while (n > 0) {
        const int step = (n + 31) / 32;
        const int i = lo + lane * step;
        const unsigned le = __ballot_sync(0xffffffffu, lane * step < n && b.cu_q[i] <= t);
        if (!le) return -1;
        const int k = 31 - __clz(le);
        const int end = lo + n;
        lo += k * step;
        n = min(step, end - lo);
        if (step == 1) break;
    }
    return t < b.cu_q[lo + 1] ? lo : -1;
}

// One sequence of a step, as far as its contents fit the batch's bounds.
struct SeqView {
    int q0, n, kv;  // first activation row, new tokens, length (new tokens included)
};
// n = 0 where nothing can be computed; *bad is set where the contents do not fit.
__device__ __forceinline__ SeqView seq_view(const mgpu_k::PagedBatch& b, int seq, int page_size, bool* bad) {
    SeqView s;
    s.q0 = b.cu_q[seq];
    s.n = b.cu_q[seq + 1] - s.q0;
    s.kv = b.kv_lens[seq];
    if (s.q0 < 0 || s.n < 0 || s.n > b.max_q_len || s.q0 > b.n_tokens - s.n || s.kv < 0 ||
        s.kv > (int64_t)b.max_pages * page_size) {
        *bad = true;
        s.n = 0;
    }
    return s;
}

}  // namespace mgpu_dev
