// logits.cu - penalties, biases and grammar masks on rows of logits, and the first maximum of
// what they leave, in one pass.
//
// A cluster of CTAs shares a row; each CTA owns a contiguous range of the vocabulary and keeps one
// word per token of it in shared memory (how often the history holds the token).  It scans the
// row's history for tokens of its range, then streams its logits once.  Bound: the logits in and
// out at HBM rate.  Counts are integers and a bias is picked by its entry's index, so the order in
// which threads reach a word cannot change a result.
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "paged.cuh"

using namespace mgpu_dev;

namespace {

constexpr int kRulesThreads = 512;
constexpr uint32_t kUsed = 1u << 31, kBiased = 1u << 30, kCount = kBiased - 1;

// A logit as mgpu_argmax compares it: exponent field zero -> 0, all ones -> +-1e30 by the sign.
template <typename T> __device__ __forceinline__ float compared(T v) {
    constexpr int kExp = sizeof(T) == 2 && std::is_same<T, __half>::value ? 0x7C00 : 0;
    if constexpr (kExp != 0) {
        const uint32_t h = __half_as_ushort(v);
        if ((h & 0x7C00u) == 0) return 0.0f;
        if ((h & 0x7C00u) == 0x7C00u) return (h & 0x8000u) ? -1e30f : 1e30f;
        return __half2float(v);
    } else {
        const uint32_t b = __float_as_uint(to_f32<T>(v));
        if ((b & 0x7F800000u) == 0) return 0.0f;
        if ((b & 0x7F800000u) == 0x7F800000u) return (b & 0x80000000u) ? -1e30f : 1e30f;
        return __uint_as_float(b);
    }
}

struct Best {
    float v;
    int i;
    __device__ __forceinline__ void take(float w, int j) {
        if (w > v || (w == v && j < i)) {
            v = w;
            i = j;
        }
    }
};

template <typename T, int VEC> struct alignas(16) Pack {
    T v[VEC];
};

template <typename T>
__global__ void __launch_bounds__(kRulesThreads) rules_kernel(const mgpu_k::RulesArgs a, int ctas, int range, int piece, int slots) {
    constexpr int VEC = 16 / (int)sizeof(T);
    extern __shared__ uint32_t words[];  // [slots] counts, then [slots] bias entry + 1 where there are biases
    uint32_t* entry = words + slots;
    __shared__ Best warp_best[kRulesThreads / 32];
    __shared__ Best cta_best;
    const int tid = threadIdx.x, row = blockIdx.x / ctas, rank = blockIdx.x % ctas;
    const T* x = reinterpret_cast<const T*>(a.x) + (int64_t)row * a.ldx;
    T* out = a.out ? reinterpret_cast<T*>(a.out) + (int64_t)row * a.ldo : nullptr;
    const int first = min((int64_t)a.n, (int64_t)rank * range), last = min((int64_t)a.n, (int64_t)first + range);
    int hist = 0, prompt = 0, b0 = 0, b1 = 0;
    float again = 1.0f, often = 0.0f, present = 0.0f;
    const int* ids = nullptr;
    if (a.history) {
        ids = a.history + (int64_t)row * a.history_ld;
        hist = min(max(a.history_lens[row], 0), a.history_ld);
        prompt = a.prompt_lens ? a.prompt_lens[row] : 0;
        again = a.penalties[3 * row];
        often = a.penalties[3 * row + 1];
        present = a.penalties[3 * row + 2];
    }
    if (a.bias_offsets) {
        b0 = min(max(a.bias_offsets[row], 0), a.bias_entries);
        b1 = min(a.bias_offsets[row + 1], a.bias_entries);
    }
    const bool marks = hist > 0 || b1 > b0;
    const uint32_t* allowed = a.allowed ? a.allowed + (int64_t)row * ((a.n + 31) / 32) : nullptr;
    Best best{-1e30f, 0x7FFFFFFF};

    for (int p0 = first; p0 < last; p0 += piece) {
        const int p1 = min(p0 + piece, last);
        // Vectors start where the row is 16-byte aligned; the words are shifted by as much, so that
        // a vector's words are one aligned vector too.
        const int lead = (int)((((uintptr_t)(x + p0) + 15) & ~(uintptr_t)15) - (uintptr_t)(x + p0)) / (int)sizeof(T);
        const int shift = (VEC - lead) % VEC;
        const bool vec_out = !out || (((uintptr_t)(out + p0) ^ (uintptr_t)(x + p0)) & 15) == 0;
        if (marks) {
            const int used = p1 - p0 + shift;
            for (int i = tid; i < used; i += kRulesThreads) words[i] = 0;
            if (b1 > b0)
                for (int i = tid; i < used; i += kRulesThreads) entry[i] = 0;
            __syncthreads();
            for (int i = tid; i < hist; i += kRulesThreads) {
                const int t = ids[i];
                if (t < p0 || t >= p1) continue;
                // a token of the prompt is used but not counted
                if (i < prompt) atomicOr(&words[t - p0 + shift], kUsed);
                else atomicAdd(&words[t - p0 + shift], 1u);
            }
            for (int i = b0 + tid; i < b1; i += kRulesThreads) {
                const int t = a.bias_tokens[i];
                if (t < p0 || t >= p1) continue;
                atomicOr(&words[t - p0 + shift], kBiased);
                atomicMax(&entry[t - p0 + shift], (uint32_t)(i - b0) + 1u);
            }
            __syncthreads();
        }
        // multiplication, division and subtraction each rounded once, in the documented order
        auto rule = [&](float v, uint32_t w, int t, bool ok) {
            if (w) {
                const float c = (float)(w & kCount);
                if (w & (kUsed | kCount)) v = v > 0.0f ? __fdiv_rn(v, again) : __fmul_rn(v, again);
                if (w & kCount) v = __fsub_rn(__fsub_rn(v, __fmul_rn(often, c)), present);
                if (w & kBiased) v = __fadd_rn(v, a.bias_values[b0 + (int)entry[t - p0 + shift] - 1]);
            }
            return ok ? v : -INFINITY;
        };
        auto single = [&](int t) {
            const uint32_t w = marks ? words[t - p0 + shift] : 0u;
            const bool ok = !allowed || ((allowed[t >> 5] >> (t & 31)) & 1u);
            const T y = from_f32<T>(rule(to_f32<T>(x[t]), w, t, ok));
            if (out) out[t] = y;
            if (a.best) {
                const float c = compared<T>(y);
                if (c > best.v) best = Best{c, t};
            }
        };
        if (!vec_out) {
            for (int t = p0 + tid; t < p1; t += kRulesThreads) single(t);
        } else {
            const int head = min(p0 + lead, p1), vecs = (p1 - head) / VEC;
            if (tid < head - p0) single(p0 + tid);
            for (int i = tid; i < vecs; i += kRulesThreads) {
                const int t = head + i * VEC;
                const uint4 raw = *reinterpret_cast<const uint4*>(x + t);
                Pack<T, VEC> v = *reinterpret_cast<const Pack<T, VEC>*>(&raw);
                uint32_t w[VEC], bits = 0xFFFFFFFFu;
#pragma unroll
                for (int k = 0; k < VEC; ++k) w[k] = 0;
                if (marks) {
#pragma unroll
                    for (int k = 0; k < VEC / 4; ++k) {
                        const uint4 q = *reinterpret_cast<const uint4*>(&words[t - p0 + shift + 4 * k]);
                        w[4 * k] = q.x; w[4 * k + 1] = q.y; w[4 * k + 2] = q.z; w[4 * k + 3] = q.w;
                    }
                }
                if (allowed) bits = __funnelshift_r(allowed[t >> 5], allowed[(t + VEC - 1) >> 5], t & 31);
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const T y = from_f32<T>(rule(to_f32<T>(v.v[k]), w[k], t + k, (bits >> k) & 1u));
                    v.v[k] = y;
                    if (a.best) {
                        const float c = compared<T>(y);
                        if (c > best.v) best = Best{c, t + k};
                    }
                }
                if (out) *reinterpret_cast<uint4*>(out + t) = *reinterpret_cast<const uint4*>(&v);
            }
            const int tail = head + vecs * VEC;
            if (tid < p1 - tail) single(tail + tid);
        }
        __syncthreads();
    }
    if (!a.best) return;
    // each thread met its tokens in index order and kept its first maximum; equal values of two
    // threads go to the smaller index
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
        best.take(__shfl_xor_sync(0xffffffffu, best.v, off), __shfl_xor_sync(0xffffffffu, best.i, off));
    if ((tid & 31) == 0) warp_best[tid >> 5] = best;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kRulesThreads / 32; ++w) best.take(warp_best[w].v, warp_best[w].i);
        cta_best = best;
    }
    cluster_sync_all();
    if (rank == 0 && tid == 0) {
        for (uint32_t r = 1; r < (uint32_t)ctas; ++r) {
            const uint32_t p = cluster_addr(&cta_best, r);
            float v;
            int i;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(p) : "memory");
            asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(i) : "r"(p + 4) : "memory");
            best.take(v, i);
        }
        // nothing above -1e30: index 0, as mgpu_argmax starts
        a.best[2 * row] = best.v > -1e30f ? best.i : 0;
        a.best[2 * row + 1] = __float_as_int(best.v);
    }
    cluster_sync_all();  // no CTA leaves while another reads its result
}

template <typename T>
cudaError_t launch_rules(const mgpu_k::LaunchCtx& c, const mgpu_k::RulesArgs& a) {
    auto kern = rules_kernel<T>;
    constexpr int kMost = 12 * 1024;  // tokens of a CTA's piece: 48 KB of counts, as much of bias entries
    static std::atomic<uint64_t> configured{0};
    int ordinal = 0;
    cudaError_t e = cudaGetDevice(&ordinal);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (ordinal & 63);
    if (ordinal >= 64 || !(configured.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 8 * (kMost + 8));
        if (e != cudaSuccess) return e;
        configured.fetch_or(bit, std::memory_order_acq_rel);
    }
    // CTAs to a row: enough of them to fill the device, and no more than a cluster holds
    int ctas = 1;
    while (ctas < 8 && ((int64_t)a.rows * ctas < 4 * c.sm_count || (a.n + ctas - 1) / ctas > kMost)) ctas *= 2;
    const int range = ((a.n + ctas - 1) / ctas + 31) / 32 * 32;
    const int piece = range < kMost ? range : kMost;
    const int slots = piece + 8;
    const bool marks = a.history || a.bias_offsets;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas * (unsigned)a.rows);
    cfg.blockDim = dim3(kRulesThreads);
    cfg.dynamicSmemBytes = marks ? (size_t)slots * 4 * (a.bias_offsets ? 2 : 1) : 0;
    cfg.stream = c.stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, a, ctas, range, piece, slots);
}

}  // namespace

namespace mgpu_k {

cudaError_t logits_process(const LaunchCtx& c, const RulesArgs& a) {
    if (a.type == MGPU_F32) return launch_rules<float>(c, a);
    if (a.type == MGPU_F16) return launch_rules<__half>(c, a);
    return launch_rules<__nv_bfloat16>(c, a);
}

}  // namespace mgpu_k
