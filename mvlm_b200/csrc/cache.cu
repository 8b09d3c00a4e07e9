// cache.cu - a step's keys and values into the paged cache, with the position rotation on the
// way (and the queries rotated beside them), and the rotation's table.
//
// The reference rotates q and k in place and copies k and v into a contiguous cache
// (dispatch_rope_apply and kv_cache_append, src/models/moondream2.cpp:406-420): three passes over
// the activations.  Here each value is read once and written once: the bound is
// T (Hq + 2 Hkv) D (source + cache bytes) at HBM rate.
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

// VEC consecutive values at p[i], of a type known at run time.
template <int VEC>
__device__ __forceinline__ void load_vec(const void* p, int type, int64_t i, float (&o)[VEC]) {
    if constexpr (VEC == 8) {
        if (type == MGPU_F32) {
            const float4* q = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
            const float4 a = q[0], b = q[1];
            o[0] = a.x; o[1] = a.y; o[2] = a.z; o[3] = a.w; o[4] = b.x; o[5] = b.y; o[6] = b.z; o[7] = b.w;
            return;
        }
        const uint4 t = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i);
        const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 f = type == MGPU_F16 ? unpack2<__half>(w[k]) : unpack2<__nv_bfloat16>(w[k]);
            o[2 * k] = f.x;
            o[2 * k + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) o[k] = load_float(p, type, (size_t)(i + k));
    }
}
template <int VEC>
__device__ __forceinline__ void store_vec(void* p, int type, int64_t i, const float (&v)[VEC]) {
    if constexpr (VEC == 8) {
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
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            if (type == MGPU_F32) reinterpret_cast<float*>(p)[i + k] = v[k];
            else if (type == MGPU_F16) reinterpret_cast<__half*>(p)[i + k] = from_f32<__half>(v[k]);
            else reinterpret_cast<__nv_bfloat16*>(p)[i + k] = from_f32<__nv_bfloat16>(v[k]);
        }
    }
}

// One CTA per (token, share of its heads).  A head is cut into units, one per thread: a unit of
// the rotated part holds whole pairs (VEC dims and their partners rot/2 further on, or, with
// adjacent pairs, VEC dims that are their own partners), a unit of the rest VEC dims.  A thread
// keeps its unit over all its heads, so the angles are read once per token and thread.
template <int VEC, bool ADJ>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const mgpu_k::AppendArgs a) {
    constexpr int PW = ADJ ? (VEC == 1 ? 2 : VEC) : VEC;  // dims of the first (or only) vector of a pair unit
    constexpr int NP = ADJ ? PW / 2 : VEC;                // pairs of a unit
    const int t = blockIdx.x;
    const int seq = seq_of_token(a.batch, t);
    if (seq < 0) return;
    const int q0 = a.batch.cu_q[seq], q1 = a.batch.cu_q[seq + 1];
    const int index = a.batch.kv_lens[seq] - (q1 - t);  // of this token in its sequence
    int page = -1;
    if (index >= 0 && index / a.page_size < a.batch.max_pages)
        page = a.batch.page_table[(int64_t)seq * a.batch.max_pages + index / a.page_size];
    bool bad = page < 0 || page >= a.num_pages || q1 > a.batch.n_tokens || q1 - q0 > a.batch.max_q_len;
    int pos[3] = {index, index, index};
    if (a.table) {
#pragma unroll
        for (int x = 0; x < 3; ++x) {
            if (x >= a.n_axes) break;
            if (a.positions) pos[x] = a.positions[(int64_t)x * a.batch.n_tokens + t];
            bad |= pos[x] < 0 || pos[x] >= a.max_pos;
        }
    }
    if (bad) {
        if (threadIdx.x == 0) atomicExch(a.status, (int)MGPU_ERR_INVALID_ARG);
        return;
    }
    const int pair_units = a.rot / (ADJ ? PW : 2 * VEC);
    const int units = pair_units + (a.D - a.rot) / VEC;
    // a head of more units than threads (single-element units of a wide head) takes several passes
    const int abreast = max(1, (int)blockDim.x / units);
    for (int u = threadIdx.x % units, h0 = threadIdx.x / units; h0 < abreast && u < units;
         u += (units > (int)blockDim.x ? (int)blockDim.x : units)) {
        const bool paired = u < pair_units;
        const int d = paired ? u * PW : a.rot + (u - pair_units) * VEC;
        float2 cs[NP];
#pragma unroll
        for (int i = 0; i < NP; ++i) cs[i] = make_float2(1.0f, 0.0f);
        if (paired) {
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int pair = (ADJ ? d / 2 : d) + i;
                const int p = pair < a.end0 ? pos[0] : pair < a.end1 ? pos[1] : pos[2];
                cs[i] = __ldg(reinterpret_cast<const float2*>(a.table) + (int64_t)p * (a.rot / 2) + pair);
            }
        }
        const int heads = a.hq + 2 * a.hkv;
        for (int h = blockIdx.y * abreast + h0; h < heads; h += gridDim.y * abreast) {
            const int g = h - a.hq;  // >= 0: a key head, >= hkv: a value head
            const bool value = g >= a.hkv;
            const void* src = g < 0 ? a.q : value ? a.v : a.k;
            const int st = g < 0 ? a.qt : value ? a.vt : a.kt;
            const int hh = g < 0 ? h : value ? g - a.hkv : g;
            const int64_t in = (int64_t)t * (g < 0 ? a.ldq : value ? a.ldv : a.ldk) + (int64_t)hh * a.D + d;
            void* dst = g < 0 ? a.qo : value ? a.vc : a.kc;
            const int dt = g < 0 ? a.qot : a.ctype;
            const int64_t out = g < 0 ? (int64_t)t * a.ldqo + (int64_t)hh * a.D + d
                                      : (((int64_t)page * a.hkv + hh) * a.page_size + index % a.page_size) * a.D + d;
            if (!paired) {
                float x[VEC];
                load_vec<VEC>(src, st, in, x);
                store_vec<VEC>(dst, dt, out, x);
            } else if constexpr (ADJ) {
                float x[PW], y[PW];
                load_vec<PW>(src, st, in, x);
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    const float c = value ? 1.0f : cs[i].x, s = value ? 0.0f : cs[i].y;
                    y[2 * i] = value ? x[2 * i] : x[2 * i] * c - x[2 * i + 1] * s;
                    y[2 * i + 1] = value ? x[2 * i + 1] : x[2 * i] * s + x[2 * i + 1] * c;
                }
                store_vec<PW>(dst, dt, out, y);
            } else {
                const int half = a.rot / 2;
                float x[VEC], y[VEC], xr[VEC], yr[VEC];
                load_vec<VEC>(src, st, in, x);
                load_vec<VEC>(src, st, in + half, y);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    xr[i] = value ? x[i] : x[i] * cs[i].x - y[i] * cs[i].y;
                    yr[i] = value ? y[i] : x[i] * cs[i].y + y[i] * cs[i].x;
                }
                store_vec<VEC>(dst, dt, out, xr);
                store_vec<VEC>(dst, dt, out + half, yr);
            }
        }
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
    // 16-byte accesses need every row, and the two halves of a pair unit, on 16-byte boundaries
    auto ok = [](const void* p, int type, int64_t ld) {
        return !p || (((uintptr_t)p & 15) == 0 && (ld * (type == MGPU_F32 ? 4 : 2)) % 16 == 0);
    };
    const bool vec = ok(a.q, a.qt, a.ldq) && ok(a.k, a.kt, a.ldk) && ok(a.v, a.vt, a.ldv) && ok(a.qo, a.qot, a.ldqo) &&
                     a.rot % (a.interleaved ? 8 : 16) == 0;
    const int w = vec ? 8 : 1;
    const int units = (a.interleaved ? a.rot / (vec ? 8 : 2) : a.rot / (2 * w)) + (a.D - a.rot) / w;
    const int abreast = units < kAppendThreads ? kAppendThreads / units : 1;
    const int passes = (a.hq + 2 * a.hkv + abreast - 1) / abreast;
    // Few tokens: one pass of heads per CTA, so that a decode step's launch is one round of loads.
    // Many: a CTA keeps its token's heads, so that the sequence search and the angles are paid once.
    int gy = 1;
    while (gy < passes && (int64_t)a.batch.n_tokens * gy < 4 * c.sm_count) ++gy;
    const dim3 grid((unsigned)a.batch.n_tokens, (unsigned)gy);
    if (a.interleaved) {
        if (vec) kv_append_kernel<8, true><<<grid, kAppendThreads, 0, c.stream>>>(a);
        else kv_append_kernel<1, true><<<grid, kAppendThreads, 0, c.stream>>>(a);
    } else {
        if (vec) kv_append_kernel<8, false><<<grid, kAppendThreads, 0, c.stream>>>(a);
        else kv_append_kernel<1, false><<<grid, kAppendThreads, 0, c.stream>>>(a);
    }
    return cudaGetLastError();
}

}  // namespace mgpu_k
