// attention.cu - attention of a step's new tokens over the paged cache.
//
// out[i] = sum_j w_ij V[j],  w_ij = softmax_j(scale q_i . K[j]) over the keys j that row i sees, in
// one pass over the keys with a running maximum m and sum l: a block of scores s gives
// m' = max(m, max s), l' = l 2^(m - m') + sum 2^(s - m'), O' = O 2^(m - m') + 2^(s - m') V, with
// scores in units of log2 (scale log2 e folded in), and out = O / l.  States (m, l, O) of disjoint
// sets of keys join by the same rule, so the keys can be split over warps and CTAs.
//
// The rows of one key head - its G query heads times the sequence's new tokens - share every key
// they load.  Rows are ordered token-major: row r is token r / G, head r % G of the group.
#include <atomic>

#include "common.cuh"
#include "kernels.h"
#include "paged.cuh"

using namespace mgpu_dev;

namespace {

constexpr int kBlock = 64;  // keys of a block: one row of the TMA boxes' 64-row destination

// ------------------------------------------------------------------ masks -----------
// First and one-past-last key that the row of token i (of n, at the end of kv) sees.
struct Seen {
    int lo, hi;
};
__device__ __forceinline__ Seen seen_by(const mgpu_k::AttendArgs& a, const SeqView& s, int i) {
    const long long p = (long long)s.kv - s.n + i;
    Seen r;
    r.hi = (int)max(0ll, a.causal ? min(p + 1, (long long)s.kv) : (long long)s.kv);
    r.lo = a.window > 0 ? (int)min((long long)r.hi, max(0ll, p - a.window + 1)) : 0;
    return r;
}
__device__ __forceinline__ bool odd16(uint32_t h, bool bf16) {
    const uint32_t e = bf16 ? 0x7F80u : 0x7C00u;
    return (h & e) == e;
}
__device__ __forceinline__ float ex2(float x) { return exp2f(x); }

// ------------------------------------------------------------------ tensor cores ----
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T> __device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ------------------------------------------------------------------ few rows --------
// At most 16 rows to a key head (a decode step): bound by reading K and V once from HBM, 4 G
// operations to a byte pair.  The blocks of all (sequence, key head) items are laid end to end and
// cut into equal shares, one per CTA, whatever the sequences' lengths; an item cut by a share's end
// is joined by the last of its CTAs to finish.  One warp feeds a ring of blocks by TMA; eight warps
// in two groups take every other block, a warp 16 of its keys, each with its own running state.
constexpr int kRowsWarps = 8, kRowsThreads = 32 * (kRowsWarps + 2);
constexpr int kRowsMax = 16;
constexpr int kSeqCap = 1024;  // sequences whose block counts are kept in shared memory

template <int DP> constexpr int rows_stage_bytes() { return 2 * kBlock * DP * 2; }
// 128 KB in flight, some three times what HBM's latency at full rate asks of an SM.  An even number,
// so that a stage always belongs to one group of warps: a wait on the parity of a barrier's phase
// must not be able to meet the phase before the last one, which a group two blocks ahead of the
// other could when they shared a stage.
template <int DP> constexpr int rows_stages() { return 128 * 1024 / rows_stage_bytes<DP>(); }
template <int DP> constexpr int rows_pitch() { return DP + 4; }
template <int DP> constexpr int rows_smem() {
    return 1024 + rows_stages<DP>() * rows_stage_bytes<DP>() + 4 * kRowsMax * rows_pitch<DP>() * 4;
}

__device__ __forceinline__ int first_block(const mgpu_k::AttendArgs& a, const SeqView& s) {
    return seen_by(a, s, 0).lo / kBlock;
}
// Blocks of one item of sequence b; a sequence that sees no key has one, in which nothing is seen,
// so that its rows are written.
__device__ __forceinline__ int item_blocks(const mgpu_k::AttendArgs& a, const SeqView& s, int max_rows) {
    if (s.n <= 0 || (long long)s.n * (a.hq / a.hkv) > max_rows) return 0;
    return max(1, (s.kv + kBlock - 1) / kBlock - first_block(a, s));
}

// The blocks [k0, k1) of key head h of sequence b.
struct Walk {
    int b, h, k;
    SeqView s;
    int blocks;
};

template <typename T, int DP>
__global__ void __launch_bounds__(kRowsThreads, 1)
    attend_rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                       const mgpu_k::AttendArgs a) {
    constexpr int S = rows_stages<DP>(), SB = rows_stage_bytes<DP>(), PITCH = rows_pitch<DP>();
    constexpr int SLABS = DP / 64, SLAB = kBlock * 128;  // 64 dims x 64 keys, 128-byte rows, swizzled
    constexpr bool kBf16 = !std::is_same<T, __half>::value;
    static_assert(S % 2 == 0, "a stage belongs to one group of warps");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    float* scratch = reinterpret_cast<float*>(ring + S * SB);
    __shared__ __align__(8) uint64_t full_bar[S], empty_bar[S];
    __shared__ int counts[kSeqCap];
    __shared__ long long warp_sum[kRowsWarps + 2];
    __shared__ bool last;
    __shared__ int start_before;
    __shared__ int start_seq;
    __shared__ float sm_m[kRowsWarps][kRowsMax], sm_l[kRowsWarps][kRowsMax];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = a.hq / a.hkv;

    if (tid == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&full_bar[s], 2);
            mbar_init(&empty_bar[s], kRowsWarps / 2);
        }
        fence_mbar_init();
        prefetch_tensormap(&tmK);
        prefetch_tensormap(&tmV);
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    }
    // the step's contents and the cache may be the preceding kernel's
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // ---- this CTA's share of all blocks
    auto count = [&](int b) {
        bool bad = false;
        const SeqView s = seq_view(a.batch, b, a.page_size, &bad);
        if (bad) atomicExch(a.status, (int)MGPU_ERR_INVALID_ARG);
        return item_blocks(a, s, a.max_rows);
    };
    long long sum = 0;
    for (int b = tid; b < a.batch.n_seqs; b += kRowsThreads) {
        const int n = count(b);
        if (b < kSeqCap) counts[b] = n;
        sum += n;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (lane == 0) warp_sum[warp] = sum;
    __syncthreads();
    long long sum_all = 0;
    for (int x = 0; x < kRowsWarps + 2; ++x) sum_all += warp_sum[x];
    const int total = (int)(sum_all * a.hkv);  // the host has bounded it
    const int shares = min((int)gridDim.x, total);  // none is empty
    if ((int)blockIdx.x >= shares) return;
    const int quota = total / shares, more = total % shares;  // the first `more` shares have one block more
    auto share = [&](int c) { return c * quota + min(c, more); };
    const int begin = share(blockIdx.x), end = share(blockIdx.x + 1);
    if (warp == 0) {
        // the sequence that holds block `begin`, and the blocks of the sequences before it
        int before = 0;
        for (int b0 = 0; b0 < a.batch.n_seqs; b0 += 32) {
            const int b = b0 + lane;
            const int n = b < a.batch.n_seqs ? (b < kSeqCap ? counts[b] : count(b)) * a.hkv : 0;
            int incl = n;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, off);
                if (lane >= off) incl += v;
            }
            const unsigned past = __ballot_sync(0xffffffffu, before + incl > begin);
            if (past) {
                if (lane == __ffs(past) - 1) {
                    start_seq = b;
                    start_before = before + incl - n;
                }
                break;
            }
            before += __shfl_sync(0xffffffffu, incl, 31);
        }
    }
    __syncthreads();
    auto enter = [&](Walk& w, int b) {  // the next sequence from b on that has blocks
        for (;; ++b) {
            const int n = b < kSeqCap ? counts[b] : -1;
            if (n == 0) continue;
            bool bad = false;
            w.s = seq_view(a.batch, b, a.page_size, &bad);
            w.blocks = n > 0 ? n : item_blocks(a, w.s, a.max_rows);
            if (w.blocks > 0) break;
        }
        w.b = b;
        w.h = 0;
        w.k = 0;
    };
    Walk w;
    enter(w, start_seq);
    w.h = (begin - start_before) / w.blocks;
    w.k = (begin - start_before) % w.blocks;

    if (warp >= kRowsWarps) {
        // ---------------------------------------------------------------- loads
        // one warp for the keys, one for the values; a lane loads one chunk (rows of one page) of a slab
        const int rows = a.box_rows, chunks = kBlock / rows, side = warp - kRowsWarps;
        const bool loads = lane < chunks * SLABS;
        const int first = (lane % chunks) * rows, slab = lane / chunks;
        const CUtensorMap* map = side ? &tmV : &tmK;
        int base = first_block(a, w.s);
        // the page of this lane's chunk of block k, asked for one block ahead; chunks past the end are
        // read from outside the map, which gives zeros
        auto key = [&] { return (base + w.k) * kBlock + first; };
        auto page_of = [&](int j) {
            if (!loads || j >= w.s.kv) return -2;
            return __ldg(a.batch.page_table + (int64_t)w.b * a.batch.max_pages + (a.page_shift >= 0 ? j >> a.page_shift : j / a.page_size));
        };
        int j = key(), page = page_of(j);
        for (int pos = begin, it = 0; pos < end; ++pos, ++it) {
            const uint32_t st = it % S;
            if (!__all_sync(0xffffffffu, mbar_wait(&empty_bar[st], ((it / S) & 1u) ^ 1u, a.status))) return;
            if (lane == 0) mbar_arrive_expect_tx(&full_bar[st], SB / 2);
            __syncwarp();
            if (loads) {
                const bool in = page >= 0 && page < a.num_pages;
                if (!in && page != -2) atomicExch(a.status, (int)MGPU_ERR_INVALID_ARG);
                const int z = in ? page * a.hkv + w.h : a.num_pages * a.hkv;
                const int y = in ? (a.page_shift >= 0 ? j & ((1 << a.page_shift) - 1) : j % a.page_size) : 0;
                tma_load_3d(ring + st * SB + side * (SB / 2) + slab * SLAB + first * 128, map, slab * 64, y, z, &full_bar[st]);
            }
            if (++w.k == w.blocks && pos + 1 < end) {
                w.k = 0;
                if (++w.h == a.hkv) {
                    enter(w, w.b + 1);
                    base = first_block(a, w.s);
                }
            }
            j = key();
            if (pos + 1 < end) page = page_of(j);
        }
        return;
    }

    // -------------------------------------------------------------------- scores and sums
    const int group = warp >> 2, part = warp & 3;  // blocks of one parity; 16 keys of each
    const int g = lane >> 2, c2 = 2 * (lane & 3);  // this thread's rows g and g + 8, and first column
    bool dead = false;  // a wait ran out: walk on without data, so that every barrier is still met
    uint32_t it = 0;
    for (int pos = begin; pos < end;) {
        const int k0 = w.k, k1 = min(w.blocks, k0 + (end - pos));
        const int base = first_block(a, w.s), R = w.s.n * G;
        // queries: A fragments of every 16 dims
        uint32_t qf[DP / 16][4];
        Seen sr[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = g + 8 * i;
            const int64_t at = r < R ? (int64_t)(w.s.q0 + r / G) * a.ldq + (int64_t)(w.h * G + r % G) * a.D : 0;
            const uint16_t* q = reinterpret_cast<const uint16_t*>(a.q) + at;
            sr[i] = r < R ? seen_by(a, w.s, r / G) : Seen{0, 0};
#pragma unroll
            for (int k = 0; k < DP / 16; ++k)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int d = 16 * k + 8 * half + c2;
                    uint32_t v = 0;
                    if (r < R && d < a.D)
                        v = a.q_pairs ? *reinterpret_cast<const uint32_t*>(q + d) : (uint32_t)q[d] | ((uint32_t)q[d + 1] << 16);
                    qf[k][2 * half + i] = v;
                }
        }
        // keys [s1.lo, s0.hi) are seen by every row
        const Seen s0 = seen_by(a, w.s, 0), s1 = seen_by(a, w.s, w.s.n - 1);
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, o[DP / 8][4];
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;

        for (int k = k0; k < k1; ++k, ++it) {
            if ((int)(it & 1u) != group || dead) continue;
            const uint32_t st = it % S;
            if (!__all_sync(0xffffffffu, mbar_wait(&full_bar[st], (it / S) & 1u, a.status))) {
                dead = true;
                continue;
            }
            const uint32_t kb = smem_u32(ring + st * SB), vb = kb + SB / 2;
            const int j0 = (base + k) * kBlock + 16 * part;  // this warp's first key
            // S = Q K^T: 16 rows x 16 keys
            float sc[2][4] = {};
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                // matrices: keys 0-7 / 8-15 x dims 0-7 / 8-15 of this step
                const int row = 16 * part + (lane & 7) + ((lane >> 4) << 3), ch = (2 * d + ((lane >> 3) & 1)) & 7;
                uint32_t b[4];
                ldsm4(b, kb + (d / 4) * SLAB + row * 128 + ((ch ^ (row & 7)) << 4));
                mma16816<T>(sc[0], qf[d], b[0], b[1]);
                mma16816<T>(sc[1], qf[d], b[2], b[3]);
            }
            const bool whole = j0 >= s1.lo && j0 + 16 <= s0.hi;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sc[n][e] *= a.scale_log2;
                    const int j = j0 + 8 * n + c2 + (e & 1);
                    if (!whole && (j < sr[e >> 1].lo || j >= sr[e >> 1].hi)) sc[n][e] = -INFINITY;
                }
            // running maximum and sum
            uint32_t pf[4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float top = fmaxf(fmaxf(sc[0][2 * i], sc[0][2 * i + 1]), fmaxf(sc[1][2 * i], sc[1][2 * i + 1]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float mn = fmaxf(m[i], top), mu = mn == -INFINITY ? 0.0f : mn;
                const float r = ex2(m[i] - mu);
                m[i] = mn;
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) p[e] = ex2(sc[e >> 1][2 * i + (e & 1)] - mu);
                l[i] = l[i] * r + ((p[0] + p[1]) + (p[2] + p[3]));
                pf[i] = pack2<T>(p[0], p[1]);
                pf[2 + i] = pack2<T>(p[2], p[3]);
                if (__any_sync(0xffffffffu, r != 1.0f)) {
#pragma unroll
                    for (int n = 0; n < DP / 8; ++n) {
                        o[n][2 * i] *= r;
                        o[n][2 * i + 1] *= r;
                    }
                }
            }
            if (!whole) {
                // Values that some row does not see: a weight of 0 times NaN or Inf is not 0, so those
                // are taken out of the block and added to the rows that see them.
                const int row = 16 * part + (lane >> 1);
                bool found = false;
#pragma unroll
                for (int i = 0; i < DP / 16; ++i) {
                    const int ch = (lane & 1) * (DP / 16) + i;
                    const uint4 v = *reinterpret_cast<const uint4*>(ring + st * SB + SB / 2 + (ch >> 3) * SLAB + row * 128 +
                                                                    (((ch & 7) ^ (row & 7)) << 4));
                    const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) found |= odd16(x[e], kBf16) || odd16(x[e] >> 16, kBf16);
                }
                if (__any_sync(0xffffffffu, found)) {
                    for (int j = 0; j < 16; ++j) {
                        const int r = 16 * part + j;
                        const bool s_lo = j0 + j >= sr[0].lo && j0 + j < sr[0].hi, s_hi = j0 + j >= sr[1].lo && j0 + j < sr[1].hi;
#pragma unroll
                        for (int n = 0; n < DP / 8; ++n) {
                            const uint32_t v = *reinterpret_cast<const uint32_t*>(ring + st * SB + SB / 2 + (n >> 3) * SLAB +
                                                                                 r * 128 + (((n & 7) ^ (r & 7)) << 4) + 2 * c2);
                            const float2 f = unpack2<T>(v);
                            const float x = odd16(v, kBf16) ? f.x : 0.0f, y = odd16(v >> 16, kBf16) ? f.y : 0.0f;
                            if (s_lo) { o[n][0] += x; o[n][1] += y; }
                            if (s_hi) { o[n][2] += x; o[n][3] += y; }
                        }
                    }
                    __syncwarp();
                    for (int i = 0; i < DP / 16; ++i) {
                        const int ch = (lane & 1) * (DP / 16) + i;
                        uint16_t* v = reinterpret_cast<uint16_t*>(ring + st * SB + SB / 2 + (ch >> 3) * SLAB + row * 128 +
                                                                  (((ch & 7) ^ (row & 7)) << 4));
                        for (int e = 0; e < 8; ++e)
                            if (odd16(v[e], kBf16)) v[e] = 0;
                    }
                    fence_proxy_async_smem();  // before the ring's next load of this stage
                    __syncwarp();
                }
            }
            // O += P V
#pragma unroll
            for (int n = 0; n < DP / 16; ++n) {
                // matrices: keys 0-7 / 8-15 x dims 0-7 / 8-15 of this step, transposed
                const int row = 16 * part + (lane & 7) + (((lane >> 3) & 1) << 3), ch = (2 * n + (lane >> 4)) & 7;
                uint32_t b[4];
                ldsm4_t(b, vb + (n / 4) * SLAB + row * 128 + ((ch ^ (row & 7)) << 4));
                mma16816<T>(o[2 * n], pf, b[0], b[1]);
                mma16816<T>(o[2 * n + 1], pf, b[2], b[3]);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty_bar[st]);
        }

        // ---- the eight warps' states join
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
            if ((lane & 3) == 0) {
                sm_m[warp][g + 8 * i] = m[i];
                sm_l[warp][g + 8 * i] = l[i];
            }
        }
        named_barrier_sync(1, 32 * kRowsWarps);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float top = -INFINITY;
#pragma unroll
            for (int x = 0; x < kRowsWarps; ++x) top = fmaxf(top, sm_m[x][g + 8 * i]);
            const float f = m[i] == -INFINITY ? 0.0f : ex2(m[i] - top);
#pragma unroll
            for (int n = 0; n < DP / 8; ++n) {
                o[n][2 * i] *= f;
                o[n][2 * i + 1] *= f;
            }
        }
        float* mine = scratch + part * kRowsMax * PITCH;
        auto put = [&] {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (g + 8 * i < R)
#pragma unroll
                    for (int n = 0; n < DP / 8; ++n)
                        *reinterpret_cast<float2*>(mine + (g + 8 * i) * PITCH + 8 * n + c2) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
        };
        if (group == 1) put();
        named_barrier_sync(1, 32 * kRowsWarps);
        if (group == 0) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (g + 8 * i < R)
#pragma unroll
                    for (int n = 0; n < DP / 8; ++n) {
                        const float2 v = *reinterpret_cast<const float2*>(mine + (g + 8 * i) * PITCH + 8 * n + c2);
                        o[n][2 * i] += v.x;
                        o[n][2 * i + 1] += v.y;
                    }
            put();  // each thread reads and then writes its own places
        }
        named_barrier_sync(1, 32 * kRowsWarps);
        // ---- rows out, or this share's state of an item that other CTAs have parts of
        const bool complete = k0 == 0 && k1 == w.blocks;
        auto state = [&](int r, float* top, float* den) {
            float t = -INFINITY, d = 0.0f;
#pragma unroll
            for (int x = 0; x < kRowsWarps; ++x) t = fmaxf(t, sm_m[x][r]);
            if (t > -INFINITY)
#pragma unroll
                for (int x = 0; x < kRowsWarps; ++x) d += sm_l[x][r] * ex2(sm_m[x][r] - t);
            *top = t;
            *den = d;
        };
        auto write = [&](int r, int d, float x, float y) {
            T* out = reinterpret_cast<T*>(a.out) + (int64_t)(w.s.q0 + r / G) * a.ldo + (int64_t)(w.h * G + r % G) * a.D + d;
            if (a.out_pairs) {
                *reinterpret_cast<uint32_t*>(out) = pack2<T>(x, y);
            } else {
                out[0] = from_f32<T>(x);
                out[1] = from_f32<T>(y);
            }
        };
        // pieces of CTA c: slot 2c for the item its share begins in, 2c + 1 for a later one
        constexpr int PIECE = kRowsMax * (DP + 2);
        const int item_begin = pos - k0;
        float* piece = a.partials + (2 * (int64_t)blockIdx.x + (item_begin > begin ? 1 : 0)) * PIECE;
        for (int e = tid; e < R * (DP / 2); e += 32 * kRowsWarps) {
            const int r = e / (DP / 2), d = 2 * (e % (DP / 2));
            if (d >= a.D) continue;
            float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float2 t = *reinterpret_cast<const float2*>(scratch + (x * kRowsMax + r) * PITCH + d);
                v.x += t.x;
                v.y += t.y;
            }
            float top, den;
            state(r, &top, &den);
            if (complete) {
                // a row that saw nothing has den = 0: its zeros stay zeros
                const float inv = den > 0.0f ? 1.0f / den : 0.0f;
                write(r, d, v.x * inv, v.y * inv);
            } else {
                __stcg(reinterpret_cast<float2*>(piece + r * DP + d), v);
                if (d == 0) {
                    __stcg(piece + kRowsMax * DP + 2 * r, top);
                    __stcg(piece + kRowsMax * DP + 2 * r + 1, den);
                }
            }
        }
        if (!complete) {
            // CTAs c0 .. c1 have the item's blocks; the last of them to arrive joins their pieces in order
            const int cut = more * (quota + 1);
            auto owner = [&](int x) { return x < cut ? x / (quota + 1) : more + (x - cut) / quota; };
            const int c0 = owner(item_begin), c1 = owner(item_begin + w.blocks - 1), pieces = c1 - c0 + 1;
            __threadfence();
            named_barrier_sync(1, 32 * kRowsWarps);
            if (tid == 0) {
                last = atomicAdd(&a.tickets[c0], 1u) == (unsigned)(pieces - 1);
                if (last) a.tickets[c0] = 0;
            }
            named_barrier_sync(1, 32 * kRowsWarps);
            if (last) {
                __threadfence();
                auto piece_of = [&](int i) {
                    return a.partials + (2 * (int64_t)(c0 + i) + (i == 0 && item_begin > share(c0) ? 1 : 0)) * PIECE;
                };
                // Every thread sums a pair of a row's values over some of the pieces; with few values the
                // threads take turns at the pieces, and their sums are added in order.
                const int values = R * (DP / 2);
                int turns = 1;
                while (2 * turns * values <= 32 * kRowsWarps) turns *= 2;
                for (int e0 = 0; e0 < values; e0 += 32 * kRowsWarps / turns) {
                    const int e = e0 + tid % (32 * kRowsWarps / turns), turn = tid / (32 * kRowsWarps / turns);
                    const int r = e / (DP / 2), d = 2 * (e % (DP / 2));
                    const bool mine_too = e < values && d < a.D;
                    float top = -INFINITY, den = 0.0f;
                    float2 v = make_float2(0.0f, 0.0f);
                    if (mine_too) {
                        for (int i = 0; i < pieces; i += 8) {
                            float t[8];
#pragma unroll
                            for (int x = 0; x < 8; ++x)
                                t[x] = i + x < pieces ? __ldcg(piece_of(i + x) + kRowsMax * DP + 2 * r) : -INFINITY;
#pragma unroll
                            for (int x = 0; x < 8; ++x) top = fmaxf(top, t[x]);
                        }
                        const float mu = top == -INFINITY ? 0.0f : top;
                        for (int i = turn; i < pieces; i += 8 * turns) {
                            float2 ml[8], o2[8];
#pragma unroll
                            for (int x = 0; x < 8; ++x) {
                                const bool has = i + x * turns < pieces;
                                const float* p = piece_of(has ? i + x * turns : 0);
                                ml[x] = has ? __ldcg(reinterpret_cast<const float2*>(p + kRowsMax * DP + 2 * r)) : make_float2(-INFINITY, 0.0f);
                                o2[x] = has ? __ldcg(reinterpret_cast<const float2*>(p + r * DP + d)) : make_float2(0.0f, 0.0f);
                            }
#pragma unroll
                            for (int x = 0; x < 8; ++x) {
                                const float f = ex2(ml[x].x - mu);
                                v.x += o2[x].x * f;
                                v.y += o2[x].y * f;
                                den += ml[x].y * f;
                            }
                        }
                    }
                    if (turns > 1) {
                        scratch[3 * tid] = v.x;
                        scratch[3 * tid + 1] = v.y;
                        scratch[3 * tid + 2] = den;
                        named_barrier_sync(1, 32 * kRowsWarps);
                        if (turn == 0)
                            for (int x = 1; x < turns; ++x) {
                                const float* o = scratch + 3 * (tid + x * (32 * kRowsWarps / turns));
                                v.x += o[0];
                                v.y += o[1];
                                den += o[2];
                            }
                    }
                    if (mine_too && turn == 0) {
                        const float inv = den > 0.0f ? 1.0f / den : 0.0f;
                        write(r, d, v.x * inv, v.y * inv);
                    }
                }
            }
        }
        named_barrier_sync(1, 32 * kRowsWarps);  // scratch and the joined states are free again
        pos += k1 - k0;
        w.k = 0;
        if (++w.h == a.hkv && pos < end) enter(w, w.b + 1);
    }
}

template <typename K>
cudaError_t allow_smem(K kern, int smem, std::atomic<uint64_t>& configured) {
    int ordinal = 0;
    cudaError_t e = cudaGetDevice(&ordinal);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (ordinal & 63);
    if (ordinal >= 64 || !(configured.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        configured.fetch_or(bit, std::memory_order_acq_rel);
    }
    return cudaSuccess;
}

template <typename T, int DP>
cudaError_t launch_rows(const mgpu_k::LaunchCtx& c, const CUtensorMap& mk, const CUtensorMap& mv, const mgpu_k::AttendArgs& a) {
    auto kern = attend_rows_kernel<T, DP>;
    static std::atomic<uint64_t> configured{0};
    const cudaError_t e = allow_smem(kern, rows_smem<DP>(), configured);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)c.sm_count);
    cfg.blockDim = dim3(kRowsThreads);
    cfg.dynamicSmemBytes = rows_smem<DP>();
    cfg.stream = c.stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, mk, mv, a);
}

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
    if ((long long)s.n * (a.hq / a.hkv) <= kRowsMax) return;
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
        x *= a.scale_log2;
        const float mn = fmaxf(m, x), r = exp2f(m - mn), w = exp2f(x - mn);
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

template <typename T>
cudaError_t launch_attend(const mgpu_k::LaunchCtx& c, const CUtensorMap& mk, const CUtensorMap& mv, const mgpu_k::AttendArgs& a) {
    cudaError_t e = a.D <= 64 ? launch_rows<T, 64>(c, mk, mv, a) : launch_rows<T, 128>(c, mk, mv, a);
    if (e != cudaSuccess || a.batch.max_q_len * (int64_t)(a.hq / a.hkv) <= kRowsMax) return e;
    const dim3 grid((unsigned)a.batch.n_tokens, (unsigned)((a.hq + 3) / 4));
    attend_kernel<T><<<grid, 128, 0, c.stream>>>(a);
    return cudaGetLastError();
}

}  // namespace

namespace mgpu_k {

size_t attend_scratch_bytes(int sm_count) { return (size_t)sm_count * 2 * kRowsMax * (128 + 2) * sizeof(float); }

bool make_cache_map(CUtensorMap* m, const void* side, int type, int num_pages, int page_size, int kv_heads, int head_dim) {
    int rows = kBlock;
    while (page_size % rows) rows /= 2;
    const int64_t dims[3] = {head_dim, page_size, (int64_t)num_pages * kv_heads};
    const int64_t strides[2] = {(int64_t)head_dim * 2, (int64_t)page_size * head_dim * 2};
    const int box[3] = {64, rows, 1};
    return make_tensor_map_u16_3d(m, side, dims, strides, box, true);
}

cudaError_t paged_attention(const LaunchCtx& c, const CUtensorMap& mk, const CUtensorMap& mv, const AttendArgs& in) {
    AttendArgs a = in;
    a.box_rows = kBlock;
    while (a.page_size % a.box_rows) a.box_rows /= 2;
    a.max_rows = kRowsMax;
    a.page_shift = -1;
    for (int i = 3; i < 31; ++i)
        if (a.page_size == 1 << i) a.page_shift = i;
    a.q_pairs = ((uintptr_t)a.q & 3) == 0 && a.ldq % 2 == 0;
    a.out_pairs = ((uintptr_t)a.out & 3) == 0 && a.ldo % 2 == 0;
    return a.type == MGPU_F16 ? launch_attend<__half>(c, mk, mv, a) : launch_attend<__nv_bfloat16>(c, mk, mv, a);
}

}  // namespace mgpu_k
