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
constexpr int kPiece = 8192;  // tokens of a CTA's round: 32 KB of logits and 32 KB of words
constexpr uint32_t kUsed = 1u << 31, kCount = kUsed - 1;

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

__device__ __forceinline__ float max_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

template <typename T, int VEC> struct alignas(16) Pack {
    T v[VEC];
};

template <typename T>
__global__ void __launch_bounds__(kRulesThreads, 3) rules_kernel(const mgpu_k::RulesArgs a, int ctas, int range, int slots) {
    constexpr int VEC = 16 / (int)sizeof(T), U = kPiece / (kRulesThreads * VEC);
    extern __shared__ __align__(16) uint8_t smem[];
    float* vals = reinterpret_cast<float*>(smem);                 // [slots] the piece's logits
    uint32_t* words = reinterpret_cast<uint32_t*>(vals + slots);  // [slots] counts, then bias entries
    __shared__ Best warp_best[kRulesThreads / 32];
    __shared__ Best cta_best;
    const int tid = threadIdx.x, row = blockIdx.x / ctas, rank = blockIdx.x % ctas;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const T* x = reinterpret_cast<const T*>(a.x) + (int64_t)row * a.ldx;
    T* out = a.out ? reinterpret_cast<T*>(a.out) + (int64_t)row * a.ldo : nullptr;
    const int first = (int)min((int64_t)a.n, (int64_t)rank * range), last = (int)min((int64_t)a.n, (int64_t)first + range);
    const uint32_t* allowed = a.allowed ? a.allowed + (int64_t)row * ((a.n + 31) / 32) : nullptr;
    Best best{-1e30f, 0x7FFFFFFF};

    for (int p0 = first; p0 < last; p0 += kPiece) {
        const int p1 = min(p0 + kPiece, last);
        // Vectors start where the row is 16-byte aligned; places in shared memory are shifted by as much,
        // so that a vector there is aligned too: token t is at t - base.
        const int lead = (int)((((uintptr_t)(x + p0) + 15) & ~(uintptr_t)15) - (uintptr_t)(x + p0)) / (int)sizeof(T);
        const int shift = (VEC - lead) % VEC, base = p0 - shift, head = min(p0 + lead, p1), vecs = (p1 - head) / VEC;
        const int tail = head + vecs * VEC, ends = (head - p0) + (p1 - tail);  // single tokens, before and after
        auto end_token = [&](int i) { return i < head - p0 ? p0 + i : tail + i - (head - p0); };
        const bool vec_out = (((uintptr_t)(out + p0) ^ (uintptr_t)(x + p0)) & 15) == 0;
        // the piece's logits are on their way while its words are cleared
        uint4 raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (tid + u * kRulesThreads < vecs) raw[u] = *reinterpret_cast<const uint4*>(x + head + (tid + u * kRulesThreads) * VEC);
        if (tid < ends) vals[end_token(tid) - base] = to_f32<T>(x[end_token(tid)]);
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
        if (marks) {
            const int used = (p1 - base + 3) / 4;  // slots are a multiple of 4
            for (int i = tid; i < used; i += kRulesThreads) reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
            __syncthreads();
#pragma unroll 4
            for (int i = tid; i < hist; i += kRulesThreads) {
                const int t = ids[i];
                if (t < p0 || t >= p1) continue;
                // a token of the prompt is used but not counted
                if (i < prompt) atomicOr(&words[t - base], kUsed);
                else atomicAdd(&words[t - base], 1u);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = tid + u * kRulesThreads;
            if (i >= vecs) break;
            const Pack<T, VEC> in = *reinterpret_cast<const Pack<T, VEC>*>(&raw[u]);
            float4* to = reinterpret_cast<float4*>(vals + head - base + i * VEC);
#pragma unroll
            for (int k = 0; k < VEC; k += 4)
                to[k / 4] = make_float4(to_f32<T>(in.v[k]), to_f32<T>(in.v[k + 1]), to_f32<T>(in.v[k + 2]), to_f32<T>(in.v[k + 3]));
        }
        __syncthreads();
        // The few tokens that have a mark are changed where they lie, each by the one entry that takes its
        // word: the pass over all tokens then knows nothing of penalties and biases.  Multiplication,
        // division, subtraction and addition are each rounded once, in the documented order.
        if (hist > 0) {
#pragma unroll 2
            for (int i = tid; i < hist; i += kRulesThreads) {
                const int t = ids[i];
                if (t < p0 || t >= p1) continue;
                const uint32_t w = atomicExch(&words[t - base], 0u);
                if (w == 0) continue;
                float v = vals[t - base];
                v = v > 0.0f ? __fdiv_rn(v, again) : __fmul_rn(v, again);
                if (w & kCount) v = __fsub_rn(__fsub_rn(v, __fmul_rn(often, (float)(w & kCount))), present);
                vals[t - base] = v;
            }
            __syncthreads();
        }
        if (b1 > b0) {  // of entries with one token, the last: the words are clear again and take its index
            for (int i = b0 + tid; i < b1; i += kRulesThreads) {
                const int t = a.bias_tokens[i];
                if (t >= p0 && t < p1) atomicMax(&words[t - base], (uint32_t)(i - b0) + 1u);
            }
            __syncthreads();
            for (int i = b0 + tid; i < b1; i += kRulesThreads) {
                const int t = a.bias_tokens[i];
                if (t >= p0 && t < p1 && words[t - base] == (uint32_t)(i - b0) + 1u)
                    vals[t - base] = __fadd_rn(vals[t - base], a.bias_values[i]);
            }
            __syncthreads();
        }
        auto consider = [&](T y, int t) {
            const float c = compared<T>(y);
            if (c > best.v || (c == best.v && t < best.i && c > -1e30f)) best = Best{c, t};
        };
        if (tid < ends) {
            const int t = end_token(tid);
            const bool ok = !allowed || ((allowed[t >> 5] >> (t & 31)) & 1u);
            const T y = from_f32<T>(ok ? vals[t - base] : -INFINITY);
            if (out) out[t] = y;
            if (a.best) consider(y, t);
        }
        for (int i = tid; i < vecs; i += kRulesThreads) {
            const int t = head + i * VEC;
            float v[VEC];
#pragma unroll
            for (int k = 0; k < VEC; k += 4) {
                const float4 q = *reinterpret_cast<const float4*>(vals + t - base + k);
                v[k] = q.x; v[k + 1] = q.y; v[k + 2] = q.z; v[k + 3] = q.w;
            }
            if (allowed) {
                const uint32_t bits = __funnelshift_r(allowed[t >> 5], allowed[(t + VEC - 1) >> 5], t & 31);
#pragma unroll
                for (int k = 0; k < VEC; ++k) v[k] = (bits >> k) & 1u ? v[k] : -INFINITY;
            }
            Pack<T, VEC> y;
#pragma unroll
            for (int k = 0; k < VEC; ++k) y.v[k] = from_f32<T>(v[k]);
            if (out) {
                if (vec_out) {
                    *reinterpret_cast<uint4*>(out + t) = *reinterpret_cast<const uint4*>(&y);
                } else {
#pragma unroll
                    for (int k = 0; k < VEC; ++k) out[t + k] = y.v[k];
                }
            }
            if (a.best) {
                // A value that beats the best in the comparison's own terms is above it, or NaN, as it
                // stands: only then are the vector's values looked at one by one.
                float top = to_f32<T>(y.v[0]);
#pragma unroll
                for (int k = 1; k < VEC; ++k) top = max_nan(top, to_f32<T>(y.v[k]));
                if (!(top <= best.v)) {
#pragma unroll 1
                    for (int k = 0; k < VEC; ++k) consider(y.v[k], t + k);
                }
            }
        }
        if (p1 < last) __syncthreads();  // the next piece takes the places
    }
    if (!a.best) return;
    // equal values of two threads go to the smaller index, as they did within one
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
        best.take(__shfl_xor_sync(0xffffffffu, best.v, off), __shfl_xor_sync(0xffffffffu, best.i, off));
    if ((tid & 31) == 0) warp_best[tid >> 5] = best;
    __syncthreads();
    if (tid < 32) {
        best = tid < kRulesThreads / 32 ? warp_best[tid] : Best{-1e30f, 0x7FFFFFFF};
#pragma unroll
        for (int off = 8; off > 0; off >>= 1)
            best.take(__shfl_xor_sync(0xffffffffu, best.v, off), __shfl_xor_sync(0xffffffffu, best.i, off));
        if (tid == 0) cta_best = best;
    }
    if (ctas > 1) cluster_sync_all();
    if (rank == 0 && tid < 32) {
        Best other{-1e30f, 0x7FFFFFFF};
        if (tid > 0 && tid < ctas) {
            const uint32_t p = cluster_addr(&cta_best, (uint32_t)tid);
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(other.v) : "r"(p) : "memory");
            asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(other.i) : "r"(p + 4) : "memory");
        }
        if (tid == 0) other = best;
#pragma unroll
        for (int off = 4; off > 0; off >>= 1)
            other.take(__shfl_xor_sync(0xffffffffu, other.v, off), __shfl_xor_sync(0xffffffffu, other.i, off));
        if (tid == 0) {
            // nothing above -1e30: index 0, as mgpu_argmax starts
            a.best[2 * row] = other.v > -1e30f ? other.i : 0;
            a.best[2 * row + 1] = __float_as_int(other.v);
        }
    }
    if (ctas > 1) cluster_sync_all();  // no CTA leaves while another reads its result
}

template <typename T>
cudaError_t launch_rules(const mgpu_k::LaunchCtx& c, const mgpu_k::RulesArgs& a) {
    auto kern = rules_kernel<T>;
    static std::atomic<uint64_t> configured{0};
    int ordinal = 0;
    cudaError_t e = cudaGetDevice(&ordinal);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (ordinal & 63);
    if (ordinal >= 64 || !(configured.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 8 * (kPiece + 8));
        if (e != cudaSuccess) return e;
        configured.fetch_or(bit, std::memory_order_acq_rel);
    }
    // CTAs to a row: enough of them to fill the device, and no more than a cluster holds
    int ctas = 1;
    while (ctas < 8 && ((int64_t)a.rows * ctas < 4 * c.sm_count || (a.n + ctas - 1) / ctas > kPiece)) ctas *= 2;
    const int range = ((a.n + ctas - 1) / ctas + 31) / 32 * 32;
    const int slots = (range < kPiece ? range : kPiece) + 8;  // a multiple of 4, with room for the shift
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas * (unsigned)a.rows);
    cfg.blockDim = dim3(kRulesThreads);
    cfg.dynamicSmemBytes = (size_t)slots * 8;
    cfg.stream = c.stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)ctas;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, a, ctas, range, slots);
}

}  // namespace

namespace mgpu_k {

cudaError_t logits_process(const LaunchCtx& c, const RulesArgs& a) {
    if (a.type == MGPU_F32) return launch_rules<float>(c, a);
    if (a.type == MGPU_F16) return launch_rules<__half>(c, a);
    return launch_rules<__nv_bfloat16>(c, a);
}

}  // namespace mgpu_k
