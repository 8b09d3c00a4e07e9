// attention.cu - attention of a step's new tokens over the paged cache.
#include "common.cuh"
#include "kernels.h"
#include "paged.cuh"

using namespace mgpu_dev;

namespace {

// One warp per (token, query head): one pass over the visible keys with a running maximum and sum.
template <typename T>
__global__ void __launch_bounds__(128) attend_kernel(const mgpu_k::AttendArgs a) {
    const int lane = threadIdx.x & 31, h = blockIdx.y * 4 + (threadIdx.x >> 5), t = blockIdx.x;
    if (h >= a.hq) return;
    const int seq = seq_of_token(a.batch, t);
    if (seq < 0) return;
    bool bad = false;
    const SeqView s = seq_view(a.batch, seq, a.page_size, &bad);
    if (bad) {
        if (lane == 0) atomicExch(a.status, (int)MGPU_ERR_INVALID_ARG);
        return;
    }
    const int p = s.kv - s.n + (t - s.q0), kvh = h / (a.hq / a.hkv);
    const int end = a.causal ? min(p + 1, s.kv) : s.kv;
    const int begin = a.window > 0 ? max(0, p - a.window + 1) : 0;
    const T* q = reinterpret_cast<const T*>(a.q) + (int64_t)t * a.ldq + (int64_t)h * a.D;
    float qv[4], o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) qv[i] = lane + 32 * i < a.D ? to_f32<T>(q[lane + 32 * i]) : 0.0f;
    for (int j = begin; j < end; ++j) {
        const int page = a.batch.page_table[(int64_t)seq * a.batch.max_pages + j / a.page_size];
        if (page < 0 || page >= a.num_pages) {
            if (lane == 0) atomicExch(a.status, (int)MGPU_ERR_INVALID_ARG);
            return;
        }
        const int64_t row = (((int64_t)page * a.hkv + kvh) * a.page_size + j % a.page_size) * a.D;
        float x = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (lane + 32 * i < a.D) x += qv[i] * to_f32<T>(reinterpret_cast<const T*>(a.kc)[row + lane + 32 * i]);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
        x *= a.scale;
        const float mn = fmaxf(m, x), r = expf(m - mn), w = expf(x - mn);
        m = mn;
        l = l * r + w;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (lane + 32 * i < a.D) o[i] = o[i] * r + w * to_f32<T>(reinterpret_cast<const T*>(a.vc)[row + lane + 32 * i]);
    }
    T* out = reinterpret_cast<T*>(a.out) + (int64_t)t * a.ldo + (int64_t)h * a.D;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (lane + 32 * i < a.D) out[lane + 32 * i] = from_f32<T>(end > begin ? o[i] / l : 0.0f);
}

}  // namespace

namespace mgpu_k {

cudaError_t paged_attention(const LaunchCtx& c, const AttendArgs& a) {
    const dim3 grid((unsigned)a.batch.n_tokens, (unsigned)((a.hq + 3) / 4));
    if (a.type == MGPU_F16) attend_kernel<__half><<<grid, 128, 0, c.stream>>>(a);
    else attend_kernel<__nv_bfloat16><<<grid, 128, 0, c.stream>>>(a);
    return cudaGetLastError();
}

}  // namespace mgpu_k
