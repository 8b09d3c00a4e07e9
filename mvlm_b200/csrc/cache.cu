// cache.cu - a step's keys and values into the paged cache, with the position rotation on the
// way (and the queries rotated beside them), and the rotation's table.
//
// The reference rotates q and k in place and copies k and v into a contiguous cache
// (dispatch_rope_apply and kv_cache_append, src/models/moondream2.cpp:406-420): three passes over
// the activations.  Here each value is read once and written once: the bound is
// T (Hq + 2 Hkv) D (source + cache bytes) and 4 T rot_dim of the rotation's table at HBM rate.  Measured: 12,814
// tokens of 32 + 16 heads of 128, bf16, 322 MB, in 60 us, 5.4 TB/s, 82 % of a copy's; the same from fp32, 479 MB, in
// 75 us, 98 %; 761 tokens of 96 heads of 64 in 4.9 us.
#include <climits>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "paged.cuh"

using namespace mgpu_dev;

namespace {

constexpr int kAppendThreads = 128;

__global__ void rope_table_kernel(float2* __restrict__ table, int64_t n, int pairs, double log_theta) {
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t p = i / pairs;
        const int k = (int)(i - p * pairs);
        // fp64: at position 1e5 an fp32 angle is already off by 4e-3
        double s, c;
        sincos((double)p * exp(-log_theta * (double)k / (double)pairs), &s, &c);
        table[i] = make_float2((float)c, (float)s);
    }
}

// Where token t of a step goes and by what angles it turns; false where it goes nowhere.  Every warp
// of the CTA calls it with the same t.
struct Place {
    int64_t slot;  // first element of its place in key head 0 of its page
    int pos[3];
};
__device__ __forceinline__ bool place_of(const mgpu_k::AppendArgs& a, int t, Place& p) {
    const int seq = seq_of_token(a.batch, t);
    if (seq < 0) return false;
    const int q0 = a.batch.cu_q[seq], q1 = a.batch.cu_q[seq + 1], kv = a.batch.kv_lens[seq];
    const int index = max(kv, 0) - (q1 - t);  // of this token in its sequence
    int page = -1;
    if (index >= 0 && index / a.page_size < a.batch.max_pages)
        page = a.batch.page_table[(int64_t)seq * a.batch.max_pages + index / a.page_size];
    bool bad = page < 0 || page >= a.num_pages || q0 < 0 || q1 > a.batch.n_tokens || q1 - q0 > a.batch.max_q_len;
#pragma unroll
    for (int x = 0; x < 3; ++x) {
        p.pos[x] = index;
        if (a.table && x < a.n_axes) {
            if (a.positions) p.pos[x] = a.positions[(int64_t)x * a.batch.n_tokens + t];
            bad |= p.pos[x] < 0 || p.pos[x] >= a.max_pos;
        }
    }
    if (bad) {
        if (threadIdx.x == 0) report_contents(a.status);
        return false;
    }
    p.slot = ((int64_t)page * a.hkv * a.page_size + index % a.page_size) * a.D;
    return true;
}
__device__ __forceinline__ float2 angle_of(const mgpu_k::AppendArgs& a, const Place& p, int pair) {
    const int pos = pair < a.end0 ? p.pos[0] : pair < a.end1 ? p.pos[1] : p.pos[2];
    return __ldg(reinterpret_cast<const float2*>(a.table) + (int64_t)pos * (a.rot / 2) + pair);
}

// A head of the step's q, k, v (in this order): where it is read and written.  A place in the cache
// counts from the token's slot.
struct Head {
    const void* src;
    void* dst;
    int stype, dtype;
    int64_t in, out;
    bool turns;
};
__device__ __forceinline__ Head head_of(const mgpu_k::AppendArgs& a, int t, int h) {
    const int g = h - a.hq;  // >= 0: a key head, >= hkv: a value head
    const bool value = g >= a.hkv;
    Head r;
    r.turns = !value;
    if (g < 0) {
        r = {a.q, a.qo, a.qt, a.qot, (int64_t)t * a.ldq + (int64_t)h * a.D, (int64_t)t * a.ldqo + (int64_t)h * a.D, true};
    } else if (!value) {
        r = {a.k, a.kc, a.kt, a.ctype, (int64_t)t * a.ldk + (int64_t)g * a.D, (int64_t)g * a.page_size * a.D, true};
    } else {
        r = {a.v, a.vc, a.vt, a.ctype, (int64_t)t * a.ldv + (int64_t)(g - a.hkv) * a.D, (int64_t)(g - a.hkv) * a.page_size * a.D, false};
    }
    return r;
}

// Eight consecutive values as loaded: 16 bytes, or 32 of fp32.
struct Raw8 {
    uint4 a, b;
};
__device__ __forceinline__ Raw8 load_raw(const void* p, int type, int64_t i) {
    Raw8 r;
    if (type == MGPU_F32) {
        const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(p) + i);
        r.a = q[0];
        r.b = q[1];
    } else {
        r.a = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i);
        r.b = r.a;
    }
    return r;
}
__device__ __forceinline__ void values_of(const Raw8& r, int type, float (&o)[8]) {
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
    if (type == MGPU_F32) {
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = __uint_as_float(w[k]);
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 f = type == MGPU_F16 ? unpack2<__half>(w[k]) : unpack2<__nv_bfloat16>(w[k]);
        o[2 * k] = f.x;
        o[2 * k + 1] = f.y;
    }
}
__device__ __forceinline__ void store8(void* p, int type, int64_t i, const float (&v)[8]) {
    if (type == MGPU_F32) {
        float4* q = reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i);
        q[0] = make_float4(v[0], v[1], v[2], v[3]);
        q[1] = make_float4(v[4], v[5], v[6], v[7]);
        return;
    }
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
        w[k] = type == MGPU_F16 ? pack2<__half>(v[2 * k], v[2 * k + 1]) : pack2<__nv_bfloat16>(v[2 * k], v[2 * k + 1]);
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
}

// One CTA per (token, share of its heads), rows and halves of pairs on 16-byte boundaries.  A head is
// cut into units of one thread: 8 dims and their partners rot/2 further on, or, with adjacent pairs,
// 8 dims that hold their own partners; and 8 dims of the rest.  A thread keeps its unit over its
// heads, so that it reads its angles once, and asks for its first heads of q, k and v before it looks
// up where they go: five dependent reads (sequence, length, page, position, angle) that would
// otherwise come before the first byte of data.
// ST, DT: the type of q, k and v, and that of q_out and the cache; -1 where they are not one.
template <bool ADJ, int ST, int DT>
__global__ void __launch_bounds__(kAppendThreads, ADJ ? 7 : ST == MGPU_F32 || ST < 0 ? 4 : 6) kv_append_kernel(const mgpu_k::AppendArgs a) {
    constexpr int NP = ADJ ? 4 : 8;  // pairs of a unit
    constexpr int AHEAD = ADJ && ST != MGPU_F32 && ST >= 0 ? 4 : 2;  // heads of q on their way: 16 to 64 registers
    const int t = blockIdx.x, half = a.rot / 2;
    const int pair_units = a.rot / (ADJ ? 8 : 16), units = pair_units + (a.D - a.rot) / 8, abreast = kAppendThreads / units;
    const int u = threadIdx.x % units, h0 = threadIdx.x / units;
    const bool paired = u < pair_units;
    const int d = paired ? u * 8 : a.rot + (u - pair_units) * 8;
    const int first = h0 < abreast ? (int)blockIdx.y * abreast + h0 : INT_MAX, step = (int)gridDim.y * abreast;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // not before: what came before us is then over
    struct Unit {
        Raw8 x, y;
    };
    auto load = [&](Unit& r, const void* src, int type, int64_t at) {
        const int st = ST >= 0 ? ST : type;
        r.x = load_raw(src, st, at);
        if (!ADJ && paired) r.y = load_raw(src, st, at + half);
    };
    Unit q[AHEAD], k, v;
    const int64_t row_q = (int64_t)t * a.ldq + d, row_k = (int64_t)t * a.ldk + d, row_v = (int64_t)t * a.ldv + d;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
        if (first < a.hq - i * step) load(q[i], a.q, a.qt, row_q + (int64_t)(first + i * step) * a.D);
    if (first < a.hkv) {
        load(k, a.k, a.kt, row_k + (int64_t)first * a.D);
        load(v, a.v, a.vt, row_v + (int64_t)first * a.D);
    }
    Place place;
    if (!place_of(a, t, place)) return;
    float2 cs[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) cs[i] = paired ? angle_of(a, place, (ADJ ? d / 2 : d) + i) : make_float2(1.0f, 0.0f);
    auto store = [&](const Unit& r, int src_type, void* dst, int dst_type, int64_t at, bool turns) {
        const int st = ST >= 0 ? ST : src_type, dt = DT >= 0 ? DT : dst_type;
        float x[8];
        values_of(r.x, st, x);
        if constexpr (ADJ) {
            if (paired && turns) {
#pragma unroll
                for (int p = 0; p < NP; ++p) {
                    const float b = x[2 * p];
                    x[2 * p] = b * cs[p].x - x[2 * p + 1] * cs[p].y;
                    x[2 * p + 1] = b * cs[p].y + x[2 * p + 1] * cs[p].x;
                }
            }
        } else if (paired) {
            float y[8];
            values_of(r.y, st, y);
            if (turns) {
#pragma unroll
                for (int p = 0; p < NP; ++p) {
                    const float b = x[p];
                    x[p] = b * cs[p].x - y[p] * cs[p].y;
                    y[p] = b * cs[p].y + y[p] * cs[p].x;
                }
            }
            store8(dst, dt, at + half, y);
        }
        store8(dst, dt, at, x);
    };
    const int64_t row_qo = (int64_t)t * a.ldqo + d, slot = place.slot + d, head = (int64_t)a.page_size * a.D;
    for (int h = first; h < a.hkv; h += step) {
        store(k, a.kt, a.kc, a.ctype, slot + h * head, true);
        store(v, a.vt, a.vc, a.ctype, slot + h * head, false);
        if (h + step < a.hkv) {
            load(k, a.k, a.kt, row_k + (int64_t)(h + step) * a.D);
            load(v, a.v, a.vt, row_v + (int64_t)(h + step) * a.D);
        }
    }
    for (int h = first; h < a.hq; h += AHEAD * step) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (h < a.hq - i * step) store(q[i], a.qt, a.qo, a.qot, row_qo + (int64_t)(h + i * step) * a.D, true);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (h < a.hq - (AHEAD + i) * step) load(q[i], a.q, a.qt, row_q + (int64_t)(h + (AHEAD + i) * step) * a.D);
    }
}

__device__ __forceinline__ void store1(void* p, int type, int64_t i, float v) {
    if (type == MGPU_F32) reinterpret_cast<float*>(p)[i] = v;
    else if (type == MGPU_F16) reinterpret_cast<__half*>(p)[i] = from_f32<__half>(v);
    else reinterpret_cast<__nv_bfloat16*>(p)[i] = from_f32<__nv_bfloat16>(v);
}

// The same where rows, pitches or the halves of the rotation (rot_dim not a multiple of 16, of 8 for adjacent
// pairs) do not fall on 16-byte boundaries: a thread to a pair, or to a value that does not turn.
__global__ void __launch_bounds__(kAppendThreads) kv_append_single_kernel(const mgpu_k::AppendArgs a) {
    const int t = blockIdx.x, half = a.rot / 2, units = half + a.D - a.rot, heads = a.hq + 2 * a.hkv;
    Place place;
    if (!place_of(a, t, place)) return;
    for (int i = blockIdx.y * kAppendThreads + threadIdx.x; i < heads * units; i += gridDim.y * kAppendThreads) {
        const int h = i / units, u = i % units;
        const Head s = head_of(a, t, h);
        const int64_t out = s.out + (h < a.hq ? 0 : place.slot);
        if (u >= half) {
            const int d = a.rot + u - half;
            store1(s.dst, s.dtype, out + d, load_float(s.src, s.stype, (size_t)(s.in + d)));
            continue;
        }
        const int d0 = a.interleaved ? 2 * u : u, d1 = a.interleaved ? 2 * u + 1 : u + half;
        float x = load_float(s.src, s.stype, (size_t)(s.in + d0)), y = load_float(s.src, s.stype, (size_t)(s.in + d1));
        if (s.turns) {
            const float2 cs = angle_of(a, place, u);
            const float b = x;
            x = b * cs.x - y * cs.y;
            y = b * cs.y + y * cs.x;
        }
        store1(s.dst, s.dtype, out + d0, x);
        store1(s.dst, s.dtype, out + d1, y);
    }
}

}  // namespace

namespace mgpu_k {

cudaError_t rope_table(const LaunchCtx& c, float* table, int max_pos, int rot, double theta) {
    const int64_t n = (int64_t)max_pos * (rot / 2);
    const int64_t grid = (n + 255) / 256;
    rope_table_kernel<<<(unsigned)(grid < c.sm_count * 16 ? grid : c.sm_count * 16), 256, 0, c.stream>>>(
        reinterpret_cast<float2*>(table), n, rot / 2, log(theta));
    return cudaGetLastError();
}

cudaError_t kv_append(const LaunchCtx& c, const AppendArgs& a) {
    // 16-byte accesses need every row, and the two halves of a pair unit, on 16-byte boundaries: split halves of
    // rot_dim 20, 24 or 40 do not have them, whatever the rows.  The kernel for the others takes 200 us where they
    // take 60, and 18 us where they take 5; 12,814 tokens of heads of 80 take 209 us with rot_dim 40, 51 with 80.
    auto ok = [](const void* p, int type, int64_t ld) {
        return !p || (((uintptr_t)p & 15) == 0 && (ld * (type == MGPU_F32 ? 4 : 2)) % 16 == 0);
    };
    const bool vec = ok(a.q, a.qt, a.ldq) && ok(a.k, a.kt, a.ldk) && ok(a.v, a.vt, a.ldv) && ok(a.qo, a.qot, a.ldqo) &&
                     a.rot % (a.interleaved ? 8 : 16) == 0;
    int passes;  // of a CTA over a token's heads
    if (vec) {
        const int units = a.rot / (a.interleaved ? 8 : 16) + (a.D - a.rot) / 8, abreast = kAppendThreads / units;
        passes = ((a.hq > a.hkv ? a.hq : a.hkv) + abreast - 1) / abreast;
    } else {
        passes = (int)(((int64_t)(a.hq + 2 * a.hkv) * (a.D - a.rot / 2) + kAppendThreads - 1) / kAppendThreads);
    }
    // Few tokens: one pass of heads per CTA, so that a decode step's launch is one round of loads (64
    // tokens of 144 heads: 6.2 us cold, 9.4 with a CTA to a token).  Many: a CTA keeps its token's heads,
    // so that the look-ups are paid once (5 prompts, 12,814 tokens: 59 us, 126 with a pass per CTA).
    int gy = 1;
    while (gy < passes && gy < 65535 && (int64_t)a.batch.n_tokens * gy < 4 * c.sm_count) ++gy;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.batch.n_tokens, (unsigned)gy);
    cfg.blockDim = dim3(kAppendThreads);
    cfg.stream = c.stream;
    if (!vec) return cudaLaunchKernelEx(&cfg, kv_append_single_kernel, a);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    auto launch = [&](auto st, auto dt) {
        constexpr int ST = decltype(st)::value, DT = decltype(dt)::value;
        return cudaLaunchKernelEx(&cfg, a.interleaved ? kv_append_kernel<true, ST, DT> : kv_append_kernel<false, ST, DT>, a);
    };
    // The usual types are compiled in (5 prompts, 12,814 tokens of 48 heads of 128, in 59 us, one of 761 in
    // 4.9); types that differ between q, k and v, or q_out's from the cache's, are looked at value by value
    // (75 and 8 us for the same).
    using F32 = std::integral_constant<int, MGPU_F32>;
    using F16 = std::integral_constant<int, MGPU_F16>;
    using BF16 = std::integral_constant<int, MGPU_BF16>;
    using Any = std::integral_constant<int, -1>;
    if (a.kt == a.vt && (!a.q || (a.qt == a.kt && a.qot == a.ctype))) {
        if (a.kt == MGPU_F32) return a.ctype == MGPU_F16 ? launch(F32(), F16()) : launch(F32(), BF16());
        if (a.kt == MGPU_F16 && a.ctype == MGPU_F16) return launch(F16(), F16());
        if (a.kt == MGPU_BF16 && a.ctype == MGPU_BF16) return launch(BF16(), BF16());
    }
    return launch(Any(), Any());
}

}  // namespace mgpu_k
