// logits.cu - penalties, biases and grammar masks on rows of logits, and the first maximum of
// what they leave, in one pass.
//
// Up to eight CTAs share a row; each owns a contiguous range of the vocabulary and keeps one word per
// token of it in shared memory (how often the history holds the token, which bias it has).  It scans
// the row's history and biases for tokens of its range, then streams its logits once.  Bound: the
// logits in and out at HBM rate.  Measured: 256 rows of 51200 fp32 logits, 108 MB, with histories of
// up to 2048 tokens, 16 biases, masks and the maximum in 37 us (44 % of a copy's rate), 17.5 us without
// any of them: the history costs 6.6, the maximum 5.5, the biases 4 to 5, the masks 1.5, nearly all of it
// waits one after another in a CTA (lengths, ids, words, logits), with four CTAs to an SM to fill them.
// Counts are integers and a bias is picked by its entry's index, so
// the order in which threads reach a word cannot change a result.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "paged.cuh"

using namespace mgpu_dev;

namespace {

constexpr int kRulesThreads = 256;
constexpr int kPiece = 8192;  // tokens of a CTA's round: at most 32 KB of logits, 32 KB of words, 2 KB of places
constexpr int kIds = 8;        // entries of the history that a thread keeps
constexpr int kListed = 1024;  // marked tokens that a round lists
// A token's word: how often the history after the prompt holds it, whether the prompt does, and its
// last bias entry + 1.
constexpr int kBiasShift = 21, kBiases = (1 << (32 - kBiasShift)) - 1;
constexpr uint32_t kUsed = 1u << 20, kCount = kUsed - 1;

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

// Values below the type's smallest normal one as 0.
template <typename T> __device__ __forceinline__ float flush(float v) {
    if constexpr (std::is_same<T, __half>::value) {
        return fabsf(v) < 6.103515625e-5f ? 0.0f : v;
    } else {
        float r;
        asm("add.ftz.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(v));
        return r;
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

// The warp's best, in every lane: the largest value by an integer that orders as it does, then the
// smallest of its indexes.
__device__ __forceinline__ Best warp_best_of(Best b) {
    const uint32_t bits = __float_as_uint(b.v + 0.0f);  // one zero
    const uint32_t key = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
    const uint32_t top = __reduce_max_sync(0xffffffffu, key);
    Best r;
    r.i = __reduce_min_sync(0xffffffffu, key == top ? b.i : 0x7FFFFFFF);
    r.v = __uint_as_float(top & 0x80000000u ? top & 0x7FFFFFFFu : ~top);
    return r;
}

__device__ __forceinline__ float max_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

template <typename T, int VEC> struct alignas(16) Pack {
    T v[VEC];
};

template <typename T>
__global__ void __launch_bounds__(kRulesThreads) rules_kernel(const mgpu_k::RulesArgs a, int ctas, int range, int slots) {
    constexpr int VEC = 16 / (int)sizeof(T);
    extern __shared__ __align__(16) uint8_t smem[];
    T* vals = reinterpret_cast<T*>(smem);                                                // [slots] the piece's logits
    uint32_t* words = reinterpret_cast<uint32_t*>(smem + (size_t)slots * sizeof(T));     // [slots] marks and counts
    uint32_t* mask = words + slots;                                                      // [kPiece / 32 + 2] allowed tokens
    uint16_t* marked = reinterpret_cast<uint16_t*>(mask + kPiece / 32 + 2);              // [kListed] places of marked tokens
    __shared__ Best warp_best[kRulesThreads / 32];
    __shared__ int n_marked;
    const int tid = threadIdx.x, row = blockIdx.x / ctas, rank = blockIdx.x % ctas;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // not before: what came before us is then over
    const T* x = reinterpret_cast<const T*>(a.x) + (int64_t)row * a.ldx;
    T* out = a.out ? reinterpret_cast<T*>(a.out) + (int64_t)row * a.ldo : nullptr;
    const int first = (int)min((int64_t)a.n, (int64_t)rank * range), last = (int)min((int64_t)a.n, (int64_t)first + range);
    const uint32_t* allowed = a.allowed ? a.allowed + (int64_t)row * ((a.n + 31) / 32) : nullptr;
    const int* ids = a.history ? a.history + (int64_t)row * a.history_ld : nullptr;
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
        // Everything that does not hang on something else is asked for at once: a CTA's time is the
        // number of reads it waits for one after another, not their bytes.
        const uint32_t to = smem_u32(vals + head - base);
        for (int i = tid; i < vecs; i += kRulesThreads)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 16 * i), "l"(x + head + i * VEC) : "memory");
        if (allowed)
            for (int i = (p0 >> 5) + tid; i <= (p1 - 1) >> 5; i += kRulesThreads)
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(mask + i - (p0 >> 5))), "l"(allowed + i) : "memory");
        int id[kIds];
#pragma unroll
        for (int k = 0; k < kIds; ++k) id[k] = ids && tid + k * kRulesThreads < a.history_ld ? __ldg(ids + tid + k * kRulesThreads) : -1;
        if (tid < ends) vals[end_token(tid) - base] = x[end_token(tid)];
        int hist = 0, prompt = 0, b0 = 0, b1 = 0;
        float again = 1.0f, often = 0.0f, present = 0.0f;
        if (a.history) {
            hist = min(max(a.history_lens[row], 0), a.history_ld);
            prompt = a.prompt_lens ? a.prompt_lens[row] : 0;
            again = a.penalties[3 * row];
            often = a.penalties[3 * row + 1];
            present = a.penalties[3 * row + 2];
        }
        int bias_t = -1;
        if (a.bias_offsets) {
            b0 = min(max(a.bias_offsets[row], 0), a.bias_entries);
            b1 = max(b0, min(a.bias_offsets[row + 1], a.bias_entries));  // not below: the difference must hold
            if (b1 - b0 > kBiases) {
                if (tid == 0) report_contents(a.status);
                b1 = b0 + kBiases;
            }
            if (b0 + tid < b1) bias_t = __ldg(a.bias_tokens + b0 + tid);
        }
        if (a.history || a.bias_offsets) {
            const int used = (p1 - base + 3) / 4;  // slots are a multiple of 4
            for (int i = tid; i < used; i += kRulesThreads) reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
            if (tid == 0) n_marked = 0;
            __syncthreads();
            // The few tokens that have a mark: the first to mark one lists it, and then each is changed once
            // where it lies, so that the pass over all tokens knows nothing of penalties and biases.
            auto listed = [&](int at) {
                const int k = atomicAdd(&n_marked, 1);
                if (k < kListed) marked[k] = (uint16_t)at;
            };
            auto in = [&](int t) { return (unsigned)(t - p0) < (unsigned)(p1 - p0); };
            if (b1 > b0) {  // of entries with one token, the last
                auto bias = [&](int i, int t) {
                    if (in(t) && atomicMax(&words[t - base], (uint32_t)i << kBiasShift) == 0) listed(t - base);
                };
                if (tid < b1 - b0) bias(tid + 1, bias_t);
                for (int i = tid + kRulesThreads; i < b1 - b0; i += kRulesThreads) bias(i + 1, __ldg(a.bias_tokens + b0 + i));
                __syncthreads();
            }
            // a token of the prompt is used but not counted
            auto mark = [&](int i, int t) {
                if (!in(t)) return;
                uint32_t* w = &words[t - base];
                if ((i < prompt ? atomicOr(w, kUsed) : atomicAdd(w, 1u)) == 0) listed(t - base);
            };
#pragma unroll
            for (int k = 0; k < kIds; ++k)
                if (tid + k * kRulesThreads < hist) mark(tid + k * kRulesThreads, id[k]);
            for (int i = tid + kIds * kRulesThreads; i < hist; i += kRulesThreads) mark(i, __ldg(ids + i));
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();
        if (a.history || a.bias_offsets) {
            // multiplication, division, subtraction and addition each rounded once, in the documented order
            auto change = [&](int at) {
                const uint32_t w = words[at], entry = w >> kBiasShift;
                const float bias = entry ? __ldg(a.bias_values + b0 + entry - 1) : 0.0f;
                float v = to_f32<T>(vals[at]);
                if (w & (kUsed | kCount)) v = v > 0.0f ? __fdiv_rn(v, again) : __fmul_rn(v, again);
                if (w & kCount) v = __fsub_rn(__fsub_rn(v, __fmul_rn(often, (float)(w & kCount))), present);
                if (entry) v = __fadd_rn(v, bias);
                vals[at] = from_f32<T>(v);
            };
            if (n_marked <= kListed) {
                for (int i = tid; i < n_marked; i += kRulesThreads) change(marked[i]);
            } else {  // more than the list holds
                for (int at = tid; at < p1 - base; at += kRulesThreads)
                    if (words[at]) change(at);
            }
            __syncthreads();
        }
        // The maximum: a thread keeps its first greatest vector, and looks for the token in it at the end.
        // Values compare as they stand but for three kinds that mgpu_argmax reads otherwise: subnormal ones
        // are 0, and Inf and NaN, which a vector's maximum shows, go the long way.
        const T none = from_f32<T>(-INFINITY);
        auto value = [&](int t) {
            return !allowed || (mask[(t >> 5) - (p0 >> 5)] >> (t & 31) & 1u) ? vals[t - base] : none;
        };
        float top = -1e30f;
        int top_i = -1;
#pragma unroll 4
        for (int i = tid; i < vecs; i += kRulesThreads) {
            const int t = head + i * VEC;
            const uint4 q = *reinterpret_cast<const uint4*>(vals + t - base);
            Pack<T, VEC> y = *reinterpret_cast<const Pack<T, VEC>*>(&q);
            if (allowed) {
                const uint32_t* m = mask + (t >> 5) - (p0 >> 5);
                const uint32_t bits = __funnelshift_r(m[0], m[1], t & 31);  // m[1] may be beyond: its bits are then not used
#pragma unroll
                for (int k = 0; k < VEC; ++k) y.v[k] = (bits >> k) & 1u ? y.v[k] : none;
            }
            if (out) {
                if (vec_out) {
                    *reinterpret_cast<uint4*>(out + t) = *reinterpret_cast<const uint4*>(&y);
                } else {
#pragma unroll
                    for (int k = 0; k < VEC; ++k) out[t + k] = y.v[k];
                }
            }
            if (a.best) {
                float m = to_f32<T>(y.v[0]);
#pragma unroll
                for (int k = 1; k < VEC; ++k) m = max_nan(m, to_f32<T>(y.v[k]));
                m = flush<T>(m);
                if (!(m < 1e30f)) {
                    m = compared<T>(y.v[0]);
#pragma unroll
                    for (int k = 1; k < VEC; ++k) m = fmaxf(m, compared<T>(y.v[k]));
                }
                if (m > top) {
                    top = m;
                    top_i = i;
                }
            }
        }
        if (a.best && top > best.v) {
            const int t = head + top_i * VEC;
            for (int k = VEC - 1; k >= 0; --k)
                if (compared<T>(value(t + k)) == top) best.i = t + k;
            best.v = top;
        }
        if (tid < ends) {
            const int t = end_token(tid);
            const T y = value(t);
            if (out) out[t] = y;
            const float c = compared<T>(y);
            if (c > best.v || (c == best.v && t < best.i && c > -1e30f)) best = Best{c, t};
        }
        if (p1 < last) __syncthreads();  // the next piece takes the places
    }
    if (!a.best) return;
    // equal values of two threads go to the smaller index, as they did within one
    best = warp_best_of(best);
    if ((tid & 31) == 0) warp_best[tid >> 5] = best;
    __syncthreads();
    if (tid < 32) best = warp_best_of(tid < kRulesThreads / 32 ? warp_best[tid] : Best{-1e30f, 0x7FFFFFFF});
    if (tid != 0) return;
    // The row's last CTA to come joins their results.  (A cluster would hold its CTAs until the slowest:
    // 11 us more for 256 rows of 51200.)
    if (ctas > 1) {
        __stcg(a.partials + (int64_t)row * 8 + rank, make_int2(best.i, __float_as_int(best.v)));
        __threadfence();
        if (atomicAdd(a.tickets + row, 1u) != (unsigned)(ctas - 1)) return;
        a.tickets[row] = 0;
        __threadfence();
        int2 other[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) other[r] = r < ctas ? __ldcg(a.partials + (int64_t)row * 8 + r) : make_int2(0x7FFFFFFF, __float_as_int(-1e30f));
#pragma unroll
        for (int r = 0; r < 8; ++r) best.take(__int_as_float(other[r].y), other[r].x);
    }
    // nothing above -1e30: index 0, as mgpu_argmax starts
    a.best[2 * (int64_t)row] = best.v > -1e30f ? best.i : 0;
    a.best[2 * (int64_t)row + 1] = __float_as_int(best.v);
}

template <typename T> constexpr int rules_smem(int slots) { return slots * ((int)sizeof(T) + 4) + 4 * (kPiece / 32 + 2) + 2 * kListed; }

template <typename T>
cudaError_t launch_rules(const mgpu_k::LaunchCtx& c, const mgpu_k::RulesArgs& a) {
    auto kern = rules_kernel<T>;
    static std::atomic<uint64_t> configured{0};
    int ordinal = 0;
    cudaError_t e = cudaGetDevice(&ordinal);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (ordinal & 63);
    if (ordinal >= 64 || !(configured.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, rules_smem<T>(kPiece + 8));
        if (e != cudaSuccess) return e;
        configured.fetch_or(bit, std::memory_order_acq_rel);
    }
    // CTAs to a row: enough of them to fill the device, and short ranges (a range's waits come one after
    // another).  One row of 51200: 20 us by one CTA, 13 by 2, 8.6 by 4, 6.6 by 8; 256 rows: 48, 48, 42, 37.  More
    // than 8 were measured in a copy whose join reads 32 results in place of 8, which alone costs 2 to 5 us: 256
    // rows 58 us by 16 and 93 by 32, one row of 51200 9.0 and 9.2.  One row of 200,000 is the exception: 13.1 us
    // by 8, 8.6 by 16 and 6.7 by 32.
    int ctas = 1;
    while (ctas < 8 && ((int64_t)a.rows * ctas < 4 * c.sm_count || (a.n + ctas - 1) / ctas > kPiece)) ctas *= 2;
    const int range = ((a.n + ctas - 1) / ctas + 31) / 32 * 32;
    const int slots = (range < kPiece ? range : kPiece) + 8;  // a multiple of 4, with room for the shift
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas * (unsigned)a.rows);
    cfg.blockDim = dim3(kRulesThreads);
    cfg.dynamicSmemBytes = rules_smem<T>(slots);
    cfg.stream = c.stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, a, ctas, range, slots);
}

}  // namespace

namespace mgpu_k {

cudaError_t logits_process(const LaunchCtx& c, const RulesArgs& in) {
    // launches of at most rules_max_rows() rows, for which there are tickets
    for (int64_t r0 = 0; r0 < in.rows; r0 += rules_max_rows()) {
        RulesArgs a = in;
        a.rows = (int)std::min<int64_t>(in.rows - r0, rules_max_rows());
        const size_t es = a.type == MGPU_F32 ? 4 : 2;
        a.x = static_cast<const char*>(in.x) + r0 * in.ldx * es;
        if (in.out) a.out = static_cast<char*>(in.out) + r0 * in.ldo * es;
        if (in.best) a.best = in.best + 2 * r0;
        if (in.history) {
            a.history = in.history + r0 * in.history_ld;
            a.history_lens = in.history_lens + r0;
            if (in.prompt_lens) a.prompt_lens = in.prompt_lens + r0;
            a.penalties = in.penalties + 3 * r0;
        }
        if (in.bias_offsets) a.bias_offsets = in.bias_offsets + r0;
        if (in.allowed) a.allowed = in.allowed + r0 * ((in.n + 31) / 32);
        const cudaError_t e = a.type == MGPU_F32 ? launch_rules<float>(c, a)
                              : a.type == MGPU_F16 ? launch_rules<__half>(c, a) : launch_rules<__nv_bfloat16>(c, a);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

int rules_max_rows() { return 8192; }
size_t rules_scratch_bytes() { return (size_t)rules_max_rows() * 8 * sizeof(int2); }

}  // namespace mgpu_k
