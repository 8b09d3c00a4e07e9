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
#include <climits>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "paged.cuh"

using namespace mgpu_dev;

namespace {

constexpr float kGrowth = 8.0f;  // log2 of how far a weight may exceed 1 before its row's reference moves
// log2 of what a weight of 1 is in fp16, whose values are 2^-24 apart at least: with kGrowth weights stay below
// 2^16, and those down to 2^-32 count, not only in the sums l.  (What the tensor cores' fp32 sums drop, in either
// type, are products below some 2^-24 of the sum that they are added to.)
template <typename T> __host__ __device__ constexpr float weight_log2() { return std::is_same<T, __half>::value ? 7.0f : 0.0f; }
constexpr int kBoxRows = 64;  // most rows of a box of the cache's TMA maps

// ------------------------------------------------------------------ masks -----------
// First and one-past-last key that the row of token i (of n, at the end of kv) sees.
struct Seen {
    int lo, hi;
};
// `p`: the row's token's index in a sequence of kv (lengths, windows and counts stay below 2^30).
__device__ __forceinline__ Seen seen_at(const mgpu_k::AttendArgs& a, int kv, int p) {
    Seen r;
    r.hi = max(0, a.causal ? min(p + 1, kv) : kv);
    r.lo = a.window > 0 ? min(r.hi, max(0, p - a.window + 1)) : 0;
    return r;
}
__device__ __forceinline__ Seen seen_by(const mgpu_k::AttendArgs& a, const SeqView& s, int i) {
    return seen_at(a, s.kv, s.kv - s.n + i);
}
__device__ __forceinline__ bool odd16(uint32_t h, bool bf16) {
    const uint32_t e = bf16 ? 0x7F80u : 0x7C00u;
    return (h & e) == e;
}
// 2^x: the hardware's approximation, some 2^-22 off, zero for results below 2^-126.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two weights in the products' 16 bits, and what that leaves of them: together 16 bits of bf16, 22 of fp16.
// With few rows to a key head both are multiplied, so that the result is rounded once: without the rests errors
// against 64 bits are up to 1.26 times those of one rounding (in mean squares; 1.4 at their greatest).  Up to 8
// rows leave 8 of the products' 16 free, and these take the rests (64 sequences of 4 rows: 102.5 us without, 102.0
// with).  9 to 16 rows take a second product (64 sequences of 16 rows: 125 us without, 128 with).  Many rows are
// bound by their products, and their weights are rounded.
template <typename T> __device__ __forceinline__ void split2(float x, float y, uint32_t& w, uint32_t& rest) {
    w = pack2<T>(x, y);
    const float2 f = unpack2<T>(w);
    rest = pack2<T>(x - f.x, y - f.y);
}

// The maximum of three; a NaN loses, as in fmaxf.
__device__ __forceinline__ float max3(float x, float y, float z) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}

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

// A barrier of `threads` threads that says whether any of them brought `p`.
__device__ __forceinline__ bool named_barrier_or(int id, int threads, bool p) {
    uint32_t r;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.pred q, %2, %3, p;\n selp.u32 %0, 1, 0, q;\n}\n"
        : "=r"(r)
        : "r"((uint32_t)p), "r"(id), "r"(threads)
        : "memory");
    return r != 0;
}

// ------------------------------------------------------------------ few rows --------
// At most 16 rows to a key head (a decode step): bound by reading K and V once from HBM, some G
// operations to a byte.  The blocks of all (sequence, key head) items are laid end to end and cut into
// equal shares, one per CTA, whatever the sequences' lengths; an item cut by a share's end is joined
// by the last of its CTAs to finish, in the pieces' order.  A warp hands the items out ahead, with
// their queries; one each feeds keys and values to a ring of 32 KB blocks by TMA; eight warps in two
// groups take every other block, each a quarter of its keys, with a running state of its own, and
// leave it in shared memory at an item's end.  Code that runs once an item is kept short: at some
// 15 clocks an instruction (it has left the instruction caches by then) 600 of them cost as much as
// five blocks.
// Measured (bf16, 8 key heads of 128, 4 rows): 64 sequences of 2150 tokens on average, 559 MB, in
// 102 us, 5.48 TB/s, 84 % of a copy's; one of 131,002 tokens, 537 MB, in 91 us, 90 %.  256 sequences of
// 540 reach 67 %: what an item costs is then seen.  16 rows: 128 us for the 64 sequences.
constexpr int kRowsWarps = 8, kRowsThreads = 32 * (kRowsWarps + 3);  // then: keys, values, items
constexpr int kRowsMax = 16;
constexpr int kSeqCap = 1024;  // sequences whose block counts are kept in shared memory

// Keys of a block: 32 KB whatever the head's dims, so that what a block costs beside its products
// (waits, maxima) falls on as many bytes (64 sequences of 64 dims: 77 us with 64 keys, 60 with 128).
// Heads of 72 to 96 dims take the stages of 128, filled to 56 to 75 %: 97 us for 64 sequences of 80 dims,
// 349 MB, 55 % of a copy's.
template <int DP> constexpr int rows_keys() { return DP == 64 ? 128 : 64; }
template <int DP> constexpr int rows_stage_bytes() { return 2 * rows_keys<DP>() * DP * 2; }
// 128 KB in flight, some three times what HBM's latency at full rate asks of an SM.  An even number,
// so that a stage always belongs to one group of warps: a wait on the parity of a barrier's phase
// must not be able to meet the phase before the last one, which a group two blocks ahead of the
// other could when they shared a stage.
template <int DP> constexpr int rows_stages() { return 128 * 1024 / rows_stage_bytes<DP>(); }
template <int DP> constexpr int rows_pitch() { return DP + 4; }
template <int DP> constexpr int rows_q_pitch() { return DP * 2 + 16; }  // bytes; rows start in different banks
constexpr int kItems = 4;  // handed out ahead
template <int DP> constexpr int rows_smem() {
    return 1024 + rows_stages<DP>() * rows_stage_bytes<DP>() + kRowsWarps * kRowsMax * rows_pitch<DP>() * 4 +
           kItems * kRowsMax * rows_q_pitch<DP>();
}

// What a CTA does of one item, handed out by a warp of its own.
struct Item {
    SeqView s;
    int seq, h, base, k0, k1, blocks, begin, more;  // base: the item's first block; begin: its place among all blocks
};

template <int KEYS> __device__ __forceinline__ int first_block(const mgpu_k::AttendArgs& a, const SeqView& s) {
    return seen_by(a, s, 0).lo / KEYS;
}
// Blocks of one item of sequence b; a sequence that sees no key has one, in which nothing is seen,
// so that its rows are written.
template <int KEYS> __device__ __forceinline__ int item_blocks(const mgpu_k::AttendArgs& a, const SeqView& s, int max_rows) {
    if (s.n <= 0 || (long long)s.n * (a.hq / a.hkv) > max_rows) return 0;
    return max(1, (s.kv + KEYS - 1) / KEYS - first_block<KEYS>(a, s));
}

// The blocks [k0, k1) of key head h of sequence b.
struct Walk {
    int b, h, k;
    SeqView s;
    int blocks;
};

// The sums of the NaN and Inf that row r sees in dims d and d + 1 of V.  (The products of a weight and its rest
// with Inf can be Inf and -Inf; such a value is rare, and looked up in the cache again: eight keys of a page at a
// time, so that a million of them take a thread some 0.1 s and not a second, within which loads wait for a stage.)
template <typename T>
__device__ __noinline__ float2 odd_values(const mgpu_k::AttendArgs& a, SeqView s, int seq, int h, int r, int d) {
    constexpr bool kBf16 = !std::is_same<T, __half>::value;
    const Seen seen = seen_by(a, s, r / (a.hq / a.hkv));
    float2 odd = make_float2(0.0f, 0.0f);
    constexpr int ABREAST = 8;  // a page's places are a multiple of it
#pragma unroll 1
    for (int j0 = seen.lo / ABREAST * ABREAST, at = j0 / a.page_size, place = j0 % a.page_size, page = -1; j0 < seen.hi; j0 += ABREAST) {
        if (place == a.page_size) {
            place = 0;
            ++at;
            page = -1;
        }
        if (page < 0) page = __ldg(a.batch.page_table + (int64_t)seq * a.batch.max_pages + at);
        if (page >= 0 && page < a.num_pages) {
            const T* v = reinterpret_cast<const T*>(a.vc) + (((int64_t)page * a.hkv + h) * a.page_size + place) * a.D + d;
            uint32_t y[ABREAST];
#pragma unroll
            for (int x = 0; x < ABREAST; ++x) y[x] = *reinterpret_cast<const uint32_t*>(v + (int64_t)x * a.D);
#pragma unroll
            for (int x = 0; x < ABREAST; ++x) {
                if (j0 + x < seen.lo || j0 + x >= seen.hi) continue;
                const float2 f = unpack2<T>(y[x]);
                if (odd16(y[x], kBf16)) odd.x += f.x;
                if (odd16(y[x] >> 16, kBf16)) odd.y += f.y;
            }
        }
        place += ABREAST;
    }
    return odd;
}

// NARROW: at most 8 rows, and the products' other 8 take the rests of their weights.
template <typename T, int DP, bool NARROW>
__global__ void __launch_bounds__(kRowsThreads, 1)
    attend_rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                       const __grid_constant__ mgpu_k::AttendArgs a) {
    constexpr int S = rows_stages<DP>(), SB = rows_stage_bytes<DP>(), PITCH = rows_pitch<DP>();
    constexpr int KEYS = rows_keys<DP>(), KW = KEYS / 4;   // of a block, of a warp
    constexpr int SLABS = DP / 64, SLAB = KEYS * 128;      // 64 dims of a block's keys, 128-byte rows, swizzled
    constexpr bool kBf16 = !std::is_same<T, __half>::value;
    constexpr float LOG2_1 = weight_log2<T>();
    static_assert(S % 2 == 0, "a stage belongs to one group of warps");
    constexpr int QP = rows_q_pitch<DP>();
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    float* scratch = reinterpret_cast<float*>(ring + S * SB);
    uint8_t* q_smem = reinterpret_cast<uint8_t*>(scratch + kRowsWarps * kRowsMax * PITCH);
    __shared__ __align__(8) uint64_t full_bar[S], empty_bar[S], item_full[kItems], item_empty[kItems];
    __shared__ Item slots[kItems];
    __shared__ int counts[kSeqCap];
    __shared__ long long warp_sum[kRowsThreads / 32];
    __shared__ bool last;
    __shared__ int start_before;
    __shared__ int start_seq;
    __shared__ float sm_m[2][kRowsWarps][kRowsMax], sm_l[2][kRowsWarps][kRowsMax];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = a.hq / a.hkv;

    if (tid == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&full_bar[s], 2);
            mbar_init(&empty_bar[s], kRowsWarps / 2);
        }
        for (int i = 0; i < kItems; ++i) {
            mbar_init(&item_full[i], 1);
            mbar_init(&item_empty[i], kRowsWarps + 2);  // the warps that score and those that load
        }
        fence_mbar_init();
        prefetch_tensormap(&tmK);
        prefetch_tensormap(&tmV);
    }
    // the step's contents and the cache may be the preceding kernel's
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // not before: what came before us is then over
    // dims beyond the head's stay zero, whatever the rows become
    for (int x = tid; x < kItems * kRowsMax * QP / 16; x += kRowsThreads) reinterpret_cast<uint4*>(q_smem)[x] = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
    // ---- this CTA's share of all blocks
    auto count = [&](int b) {
        bool bad = false;
        const SeqView s = seq_view(a.batch, b, a.page_size, &bad);
        if (bad) report_contents(a.status);
        return item_blocks<KEYS>(a, s, a.max_rows);
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
    for (int x = 0; x < kRowsThreads / 32; ++x) sum_all += warp_sum[x];
    const int total = (int)(sum_all * a.hkv);  // the host has bounded it
    const int shares = min((int)gridDim.x, total);  // none is empty
    if ((int)blockIdx.x >= shares) return;
    const int quota = total / shares, extra = total % shares;  // the first `extra` shares have one block more
    auto share = [&](int c) { return c * quota + min(c, extra); };
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
            w.blocks = n > 0 ? n : item_blocks<KEYS>(a, w.s, a.max_rows);
            if (w.blocks > 0) break;
        }
        w.b = b;
        w.h = 0;
        w.k = 0;
    };
    auto wait = [&](uint64_t* bar, uint32_t phase) { return __all_sync(0xffffffffu, mbar_wait(bar, phase & 1u, a.status)); };

    if (warp == kRowsWarps + 2) {
        // ---------------------------------------------------------------- items, and their queries
        Walk w;
        enter(w, start_seq);
        w.h = (begin - start_before) / w.blocks;
        w.k = (begin - start_before) % w.blocks;
        int i = 0;
        for (int pos = begin; pos < end; ++i) {
            const int x = i % kItems, k1 = min(w.blocks, w.k + (end - pos)), R = w.s.n * G;
            if (!wait(&item_empty[x], (i / kItems) ^ 1)) break;
            if (lane == 0) {
                Item& it = slots[x];
                it.s = w.s;
                it.seq = w.b;
                it.h = w.h;
                it.base = first_block<KEYS>(a, w.s);
                it.k0 = w.k;
                it.k1 = k1;
                it.blocks = w.blocks;
                it.begin = pos - w.k;
                it.more = pos + k1 - w.k < end;
                if (a.q_vec) mbar_arrive_expect_tx(&item_full[x], (uint32_t)(R * a.D * 2));
            }
            __syncwarp();
            const uint16_t* q = reinterpret_cast<const uint16_t*>(a.q) + (int64_t)w.s.q0 * a.ldq + (int64_t)w.h * G * a.D;
            uint8_t* to = q_smem + x * kRowsMax * QP;
            if (a.q_vec) {  // a row to a lane
                if (lane < R) bulk_g2s(to + lane * QP, q + (int64_t)(lane / G) * a.ldq + (lane % G) * a.D, (uint32_t)a.D * 2, &item_full[x]);
            } else {  // no 16-byte boundaries
                for (int e = lane; e < R * a.D; e += 32) {
                    const int r = e / a.D, d = e % a.D;
                    reinterpret_cast<uint16_t*>(to + r * QP)[d] = q[(int64_t)(r / G) * a.ldq + (r % G) * a.D + d];
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&item_full[x]);
            }
            __syncwarp();
            pos += k1 - w.k;
            w.k = 0;
            if (++w.h == a.hkv && pos < end) enter(w, w.b + 1);
        }
        // the copies under way land before the CTA may end, also where other warps gave up
        for (int x = max(0, i - kItems); x < i; ++x) wait(&item_full[x % kItems], x / kItems);
        return;
    }
    if (warp >= kRowsWarps) {
        // ---------------------------------------------------------------- loads
        // one warp for the keys, one for the values; a lane loads one chunk (rows of one page) of a slab
        const int rows = a.box_rows, chunks = KEYS / rows, side = warp - kRowsWarps;
        const bool loads = lane < chunks * SLABS;
        const int first = (lane % chunks) * rows, slab = lane / chunks;
        const CUtensorMap* map = side ? &tmV : &tmK;
        bool ok = true, more = true;
        uint32_t n = 0;  // blocks so far
        for (int i = 0; ok && more; ++i) {
            ok = wait(&item_full[i % kItems], i / kItems);
            if (!ok) break;
            const Item it = slots[i % kItems];
            __syncwarp();
            if (lane == 0) mbar_arrive(&item_empty[i % kItems]);
            more = it.more;
            // the page of this lane's chunk of a block, asked for one block ahead; chunks past the end are
            // read from outside the map, which gives zeros
            const int* pages = a.batch.page_table + (int64_t)it.seq * a.batch.max_pages;
            auto page_of = [&](int j) {
                return loads && j < it.s.kv ? __ldg(pages + (a.page_shift >= 0 ? j >> a.page_shift : j / a.page_size)) : -1;
            };
            int j = (it.base + it.k0) * KEYS + first, page = page_of(j);
            for (int k = it.k0; k < it.k1; ++k, ++n) {
                const uint32_t st = n % S;
                ok = wait(&empty_bar[st], (n / S) ^ 1);
                if (!ok) break;
                if (lane == 0) mbar_arrive_expect_tx(&full_bar[st], SB / 2);
                __syncwarp();
                if (loads) {
                    const bool in = page >= 0 && page < a.num_pages;
                    if (!in && j < it.s.kv) report_contents(a.status);
                    const int z = in ? page * a.hkv + it.h : a.num_pages * a.hkv;
                    const int y = in ? (a.page_shift >= 0 ? j & ((1 << a.page_shift) - 1) : j % a.page_size) : 0;
                    tma_load_3d(ring + st * SB + side * (SB / 2) + slab * SLAB + first * 128, map, slab * 64, y, z, &full_bar[st]);
                }
                j += KEYS;
                if (k + 1 < it.k1) page = page_of(j);
                __syncwarp();
            }
        }
        // a wait ran out: the copies under way still have to land before the CTA may end
        if (!ok)
            for (uint32_t x = n > S ? n - S : 0; x < n; ++x) wait(&full_bar[x % S], x / S);
        return;
    }

    // -------------------------------------------------------------------- scores and sums
    const int group = warp >> 2, part = warp & 3;  // blocks of one parity; KW keys of each
    const int g = lane >> 2, c2 = 2 * (lane & 3);  // this thread's rows g and g + 8, and first column
    // Two items' states of up to 8 rows fit the scratch, and the barrier of the item between says that the
    // last ones have been read.  Where an item may have more rows, each takes both places, and a barrier more.
    constexpr int HALVES = NARROW ? 1 : 2, room = 8 * HALVES;  // of 8 rows: this thread's are g + 8 x, x < HALVES
    uint32_t it = 0;
    struct {
        SeqView s;
        int seq, h, blocks;
    } w;
    for (int i = 0, more = 1; more; ++i) {
        const int slot = i % kItems, turn = i & 1;
        int k0 = 0, k1 = 0, base = 0, item_begin = 0, R = 0;
        Seen sr[HALVES];
        float m[HALVES], l[HALVES], o[DP / 8][4];
#pragma unroll
        for (int x = 0; x < HALVES; ++x) {
            m[x] = -INFINITY;
            l[x] = 0.0f;
        }
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;
        bool dead = !wait(&item_full[slot], i / kItems);  // a wait ran out: all warps leave at the item's barrier
        if (!dead) {
            k0 = slots[slot].k0;
            k1 = slots[slot].k1;
            base = slots[slot].base;
            item_begin = slots[slot].begin;
            w.s = slots[slot].s;
            w.seq = slots[slot].seq;
            w.h = slots[slot].h;
            w.blocks = slots[slot].blocks;
            more = slots[slot].more;
            R = w.s.n * G;
            // Queries: A fragments of every 16 dims.  Rows beyond the item's hold older ones; nothing of
            // theirs is written.
            uint32_t qf[DP / 16][4];
            const uint32_t qa = smem_u32(q_smem) + (slot * kRowsMax + (lane & 15)) * QP + (lane >> 4) * 16;
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) ldsm4(qf[k], qa + 32 * k);
#pragma unroll
            for (int x = 0; x < HALVES; ++x) sr[x] = g + 8 * x < R ? seen_by(a, w.s, (g + 8 * x) / G) : Seen{0, 0};
            __syncwarp();
            if (lane == 0) mbar_arrive(&item_empty[slot]);
            // keys [s1.lo, s0.hi) are seen by every row
            const Seen s0 = seen_by(a, w.s, 0), s1 = seen_by(a, w.s, w.s.n - 1);
            for (int k = k0; k < k1; ++k, ++it) {
                if ((int)(it & 1u) != group || dead) continue;
                const uint32_t st = it % S;
                if (!__all_sync(0xffffffffu, mbar_wait(&full_bar[st], (it / S) & 1u, a.status))) {
                    dead = true;
                    continue;
                }
                const uint32_t kb = smem_u32(ring + st * SB), vb = kb + SB / 2;
                const int j0 = (base + k) * KEYS + KW * part;  // this warp's first key
                // S = Q K^T: 16 rows x KW keys
                float sc[KW / 8][4];
#pragma unroll
                for (int n = 0; n < KW / 8; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[n][e] = 0.0f;
#pragma unroll
                for (int d = 0; d < DP / 16; ++d)
#pragma unroll
                    for (int u = 0; u < KW / 16; ++u) {
                        // matrices: keys 0-7 / 8-15 x dims 0-7 / 8-15 of this step
                        const int row = KW * part + 16 * u + (lane & 7) + ((lane >> 4) << 3), ch = (2 * d + ((lane >> 3) & 1)) & 7;
                        uint32_t b[4];
                        ldsm4(b, kb + (d / 4) * SLAB + row * 128 + ((ch ^ (row & 7)) << 4));
                        mma16816<T>(sc[2 * u], qf[d], b[0], b[1]);
                        mma16816<T>(sc[2 * u + 1], qf[d], b[2], b[3]);
                    }
                const bool whole = j0 >= s1.lo && j0 + KW <= s0.hi;
                if (__builtin_expect(!whole, 0)) {
#pragma unroll
                    for (int n = 0; n < KW / 8; ++n)
#pragma unroll
                        for (int e = 0; e < 2 * HALVES; ++e) {
                            const int j = j0 + 8 * n + c2 + (e & 1);
                            if (j < sr[e >> 1].lo || j >= sr[e >> 1].hi) sc[n][e] = -INFINITY;
                        }
                }
                // The reference m, which the maximum may exceed by kGrowth (and LOG2_1, as a weight of 1 counts)
                // before it moves, so that O mostly stays as it is, and the sum.
                uint32_t pf[KW / 16][4], rest[KW / 16][4];
                float top[HALVES];
                bool grown = false;
#pragma unroll
                for (int i = 0; i < HALVES; ++i) {
                    top[i] = fmaxf(sc[0][2 * i], sc[0][2 * i + 1]);
#pragma unroll
                    for (int n = 1; n < KW / 8; ++n) top[i] = fmaxf(top[i], fmaxf(sc[n][2 * i], sc[n][2 * i + 1]));
                    top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
                    top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2)) * a.scale_log2;
                    grown |= top[i] > m[i] + (LOG2_1 + kGrowth);
                }
                if (__any_sync(0xffffffffu, grown)) {
                    float r[HALVES];
#pragma unroll
                    for (int i = 0; i < HALVES; ++i) {
                        const float mn = fmaxf(m[i], top[i] - LOG2_1);
                        r[i] = mn == -INFINITY ? 1.0f : ex2(m[i] - mn);
                        m[i] = mn;
                        l[i] *= r[i];
                    }
#pragma unroll
                    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[n][e] *= r[NARROW ? 0 : e >> 1];
                }
#pragma unroll
                for (int i = 0; i < HALVES; ++i) {
                    const float neg = m[i] == -INFINITY ? 0.0f : -m[i];
#pragma unroll
                    for (int u = 0; u < KW / 16; ++u) {
                        float p[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) p[e] = ex2(fmaf(sc[2 * u + (e >> 1)][2 * i + (e & 1)], a.scale_log2, neg));
                        l[i] += (p[0] + p[1]) + (p[2] + p[3]);
                        split2<T>(p[0], p[1], pf[u][i], NARROW ? pf[u][1] : rest[u][i]);
                        split2<T>(p[2], p[3], pf[u][2 + i], NARROW ? pf[u][3] : rest[u][2 + i]);
                    }
                }
                if (__builtin_expect(!whole, 0)) {
                    // Values that some row does not see: a weight of 0 times NaN or Inf is not 0, so those
                    // are taken out of the block and added to the rows that see them.
                    uint8_t* vs = ring + st * SB + SB / 2;
                    bool found = false;
#pragma unroll 4
                    for (int x = lane; x < KW * DP / 8; x += 32) {
                        const int row = KW * part + x / (DP / 8), ch = x % (DP / 8);
                        const uint4 v = *reinterpret_cast<const uint4*>(vs + (ch >> 3) * SLAB + row * 128 + (((ch & 7) ^ (row & 7)) << 4));
                        const uint32_t y[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) found |= odd16(y[e], kBf16) || odd16(y[e] >> 16, kBf16);
                    }
                    if (__builtin_expect(__any_sync(0xffffffffu, found), 0)) {
#pragma unroll 1
                        for (int j = 0; j < KW; ++j) {
                            const int r = KW * part + j;
                            const bool s_lo = j0 + j >= sr[0].lo && j0 + j < sr[0].hi;
                            const bool s_hi = !NARROW && j0 + j >= sr[HALVES - 1].lo && j0 + j < sr[HALVES - 1].hi;
#pragma unroll
                            for (int n = 0; n < DP / 8; ++n) {
                                const uint32_t v = *reinterpret_cast<const uint32_t*>(vs + (n >> 3) * SLAB + r * 128 +
                                                                                     (((n & 7) ^ (r & 7)) << 4) + 2 * c2);
                                const float2 f = unpack2<T>(v);
                                const float x = odd16(v, kBf16) ? f.x : 0.0f, y = odd16(v >> 16, kBf16) ? f.y : 0.0f;
                                if (s_lo) { o[n][0] += x; o[n][1] += y; }
                                if (s_hi) { o[n][2] += x; o[n][3] += y; }
                            }
                        }
                        __syncwarp();
#pragma unroll 1
                        for (int x = lane; x < KW * DP; x += 32) {
                            const int row = KW * part + x / DP, d = x % DP;
                            uint16_t* v = reinterpret_cast<uint16_t*>(vs + (d >> 6) * SLAB + row * 128 + ((((d >> 3) & 7) ^ (row & 7)) << 4)) + (d & 7);
                            if (odd16(*v, kBf16)) *v = 0;
                        }
                        fence_proxy_async_smem();  // before the ring's next load of this stage
                        __syncwarp();
                    }
                }
                // O += P V
#pragma unroll
                for (int u = 0; u < KW / 16; ++u)
#pragma unroll
                    for (int n = 0; n < DP / 16; ++n) {
                        // matrices: keys 0-7 / 8-15 x dims 0-7 / 8-15 of this step, transposed
                        const int row = KW * part + 16 * u + (lane & 7) + (((lane >> 3) & 1) << 3), ch = (2 * n + (lane >> 4)) & 7;
                        uint32_t b[4];
                        ldsm4_t(b, vb + (n / 4) * SLAB + row * 128 + ((ch ^ (row & 7)) << 4));
                        mma16816<T>(o[2 * n], pf[u], b[0], b[1]);
                        mma16816<T>(o[2 * n + 1], pf[u], b[2], b[3]);
                        if constexpr (!NARROW) {
                            mma16816<T>(o[2 * n], rest[u], b[0], b[1]);
                            mma16816<T>(o[2 * n + 1], rest[u], b[2], b[3]);
                        }
                    }
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty_bar[st]);
            }
        }
        // ---- the eight warps' states join: each leaves its own, and whoever writes a value weighs them
#pragma unroll
        for (int x = 0; x < HALVES; ++x) {
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
            if ((lane & 3) == 0) {
                sm_m[turn][warp][g + 8 * x] = m[x];
                sm_l[turn][warp][g + 8 * x] = l[x];
            }
        }
        float* states = scratch + (NARROW ? turn * kRowsWarps * 8 * PITCH : 0);
#pragma unroll
        for (int x = 0; x < HALVES; ++x)
            if (g + 8 * x < R)
#pragma unroll
                for (int n = 0; n < DP / 8; ++n)
                    *reinterpret_cast<float2*>(states + (warp * room + g + 8 * x) * PITCH + 8 * n + c2) =
                        NARROW ? make_float2(o[n][0] + o[n][2], o[n][1] + o[n][3]) : make_float2(o[n][2 * x], o[n][2 * x + 1]);
        if (named_barrier_or(1, 32 * kRowsWarps, dead)) break;
        // ---- rows out, or this share's state of an item that other CTAs have parts of
        const bool complete = k0 == 0 && k1 == w.blocks;
        auto write = [&](int r, int d, float2 v, float den) {
            // a row that saw nothing has den = 0: its zeros stay zeros
            const float inv = den > 0.0f ? 1.0f / den : 0.0f;
            float x = v.x * inv, y = v.y * inv;
            if (__builtin_expect(!(fabsf(x) + fabsf(y) < INFINITY), 0) && den > 0.0f) {
                const float2 odd = odd_values<T>(a, w.s, w.seq, w.h, r, d);
                if (!(fabsf(odd.x) < INFINITY)) x = odd.x;
                if (!(fabsf(odd.y) < INFINITY)) y = odd.y;
            }
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
        float* piece = a.partials + (2 * (int64_t)blockIdx.x + (item_begin > begin ? 1 : 0)) * PIECE;
        for (int e = tid; e < R * (DP / 2); e += 32 * kRowsWarps) {
            const int r = e / (DP / 2), d = 2 * (e % (DP / 2));
            if (d >= a.D) continue;
            float top = -INFINITY, den = 0.0f;
#pragma unroll
            for (int x = 0; x < kRowsWarps; ++x) top = fmaxf(top, sm_m[turn][x][r]);
            const float mu = top == -INFINITY ? 0.0f : top;
            float2 v = make_float2(0.0f, 0.0f);
#pragma unroll 2
            for (int x = 0; x < kRowsWarps; ++x) {
                const float f = ex2(sm_m[turn][x][r] - mu);
                const float2 t = *reinterpret_cast<const float2*>(states + (x * room + r) * PITCH + d);
                v.x += t.x * f;
                v.y += t.y * f;
                den += sm_l[turn][x][r] * f;
            }
            if (complete) {
                write(r, d, v, den);
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
            const int cut = extra * (quota + 1);
            auto owner = [&](int x) { return x < cut ? x / (quota + 1) : extra + (x - cut) / quota; };
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
                    if (mine_too && turn == 0) write(r, d, v, den);
                }
            }
        }
        if (!NARROW || !complete) named_barrier_sync(1, 32 * kRowsWarps);  // the places are free again
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

template <typename T, int DP, bool NARROW>
cudaError_t launch_rows(const mgpu_k::LaunchCtx& c, const CUtensorMap& mk, const CUtensorMap& mv, const mgpu_k::AttendArgs& a) {
    auto kern = attend_rows_kernel<T, DP, NARROW>;
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

// ------------------------------------------------------------------ many rows -------
// More than 16 rows to a key head (a chunk of a prompt): bound by the two products, 4 D operations to a
// row and key, and beside them one exponential.  A CTA takes two tiles of up to 128 rows (whole
// tokens: 128 / G of them) over the same blocks of 128 keys.  A warp to each tile issues
// S_t = Q_t K^T and O_t += P_t V; scores, weights and O stay in TMEM (its 512 columns are full at 128
// dims), weights in the place of their scores.  Each tile has four softmax warps, a thread to a row,
// which needs no exchange for its maximum and sum.  O is rescaled only when a row's maximum has grown
// by more than 2^kGrowth since its reference was taken, and most blocks leave it alone.  All blocks
// of all items (sequence, key head, pair of tiles) are cut into equal shares as above.
// Measured (bf16, 32 query and 8 key heads of 128): 4096 new tokens over 4096 in 392 us at 1965 MHz, 1052
// TFLOP/s, 63 % of a library product's rate; calls in a row reach the power limit after 50 ms and settle
// at 437 us (1.75 GHz), 68 % of what the library then holds.  A block of 128 keys takes 4150 clocks for
// both tiles, of which the tensor cores' arithmetic is 2048, their reads of shared memory 2560 (all of Q
// for every 64 keys), the exponentials 2048.  A softmax warp's half block: 1050 clocks of exponentials,
// which the two warps of a scheduler mostly do at the same time, 380 of masks and maxima, 300 of waiting
// for scores, 350 of the rest.  Scores come in halves of 64 keys: next to whole blocks 24.0 -> 20.7 us for
// 761 tokens and 137 -> 129 for a mixed batch, at 452 -> 461 for 4096 tokens over 4096.  Tried and slower:
// a quarter of the exponentials as polynomials (+4 %), turns at the exponentials (a lock to each scheduler:
// +14 %), two threads to a row (453 us), the next scores in registers a half ahead (517 us).
//
// Which kernel: at most 16 rows go to the one above (64 sequences of 2150 tokens, 4 rows: 102 us there,
// 146 here; 16 rows: 128 and 147; 256 sequences of 250 tokens and 16 rows are the exception, 166 and 142), or
// at most 8 of them (see paged_attention).  A call with one sequence that may have more rows launches this
// kernel alone (761 tokens: 20.5 us, and 23.5 with the other beside it).
constexpr int kTileKeys = 128, kTileRows = 128;
constexpr int kTileThreads = 384;  // 8 softmax warps, then: products, loads, products, scheduling
constexpr int kTileSeqs = 1024;    // sequences of one launch
constexpr int kTileEntries = 2048; // entries of the table of items
constexpr int kJoinBlocks = 6;     // what a join costs, in blocks (some 10 us for 64 dims, more for 128)

template <int DP> constexpr int tile_stage_bytes() { return kTileKeys * DP * 2; }
// K on even and V on odd stages: two blocks of 128 dims, four of 64
template <int DP> constexpr int tile_stages() { return 128 * 1024 / tile_stage_bytes<DP>(); }
template <int DP> constexpr int tile_smem() {
    return 1024 + 2 * kTileRows * DP * 2 + tile_stages<DP>() * tile_stage_bytes<DP>() + 4 * (kTileSeqs + 1 + kTileEntries + 1);
}

__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// 32 columns of this thread's TMEM lane; valid after tmem_ld_wait and tmem_use.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
          "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
          "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Keeps uses of the loaded registers behind the wait.
template <int N = 32> __device__ __forceinline__ void tmem_use(uint32_t* r) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two tiles of one sequence's tokens.  Blocks are counted from the sequence's start.
struct Pair {
    int lo, blocks;                // the blocks that either tile needs: [lo, lo + blocks)
    int first[2], rows[2];         // a tile's first token and its rows (0: no tile)
    int t_lo[2], t_hi[2];          // its blocks
    int whole_lo[2], whole_hi[2];  // the keys that all its rows see
};
__device__ __forceinline__ Pair pair_of(const mgpu_k::AttendArgs& a, const SeqView& s, int j, int per_tile) {
    Pair p;
    const int G = a.hq / a.hkv;
    int lo = INT_MAX, hi = 0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int first = (2 * j + t) * per_tile, n = min(max(s.n - first, 0), per_tile);
        p.first[t] = first;
        p.rows[t] = n * G;
        p.t_lo[t] = p.t_hi[t] = p.whole_lo[t] = p.whole_hi[t] = 0;
        if (n == 0) continue;
        const Seen a0 = seen_by(a, s, first), a1 = seen_by(a, s, first + n - 1);
        p.whole_lo[t] = a1.lo;
        p.whole_hi[t] = a0.hi;
        if (a1.hi <= a0.lo) continue;
        p.t_lo[t] = a0.lo / kTileKeys;
        p.t_hi[t] = (a1.hi + kTileKeys - 1) / kTileKeys;
        lo = min(lo, p.t_lo[t]);
        hi = max(hi, p.t_hi[t]);
    }
    // a pair that sees nothing has one block, which no tile takes, so that its rows are written
    p.lo = hi > 0 ? lo : 0;
    p.blocks = max(1, hi - p.lo);
    return p;
}

// What a CTA does of one item, as its scheduling warp hands it to the others.
struct Segment {
    int kb0, kb1;                  // blocks
    int lo[2], hi[2];              // those that each tile takes (none: lo >= hi)
    int whole_lo[2], whole_hi[2];  // keys that all rows of a tile see
    int rows[2], row0[2], index[2];  // rows of a tile; activation row and index in the sequence of its first token
    int kv, seq, h;
    int complete;                  // all of the item's blocks; else the piece's slot and who has the others
    int slot, c0, pieces, first_slot;
    int more;                      // another segment follows
    int odd;                       // NaN or Inf was taken out of a block of V
    __device__ __forceinline__ bool in(int t, int kb) const { return kb >= lo[t] && kb < hi[t]; }
    __device__ __forceinline__ bool whole(int t, int kb) const {
        return kb * kTileKeys >= whole_lo[t] && (kb + 1) * kTileKeys <= whole_hi[t];
    }
    // some row of a tile that takes the block does not see all of it
    __device__ __forceinline__ bool masked(int kb) const { return (in(0, kb) && !whole(0, kb)) || (in(1, kb) && !whole(1, kb)); }
};
constexpr int kSegments = 4;  // handed out ahead

__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p != 0;
}

template <typename T, int DP>
__global__ void __launch_bounds__(kTileThreads, 1)
    attend_tile_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                       const __grid_constant__ CUtensorMap tmQ, const mgpu_k::AttendArgs a, int seq0) {
    constexpr int SLABS = DP / 64, QB = kTileRows * DP * 2, SB = tile_stage_bytes<DP>(), SLAB = kTileKeys * 128;
    constexpr int S = tile_stages<DP>();
    constexpr int PIECE = kTileRows * (DP + 2);
    constexpr bool kBf16 = !std::is_same<T, __half>::value;
    constexpr float LOG2_1 = weight_log2<T>();
    extern __shared__ uint8_t smem_raw[];
    uint8_t* qs = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* ring = qs + 2 * QB;
    int* seq_first = reinterpret_cast<int*>(ring + S * SB);  // [n + 1] pairs before a sequence
    int* cum = seq_first + kTileSeqs + 1;                    // [entries + 1] blocks before an entry
    __shared__ __align__(8) uint64_t full_bar[S], empty_bar[S], clean_bar[S], q_bar[2], s_bar[2][2], p_bar[2][2], o_bar[2][2], q_free[2], drain_bar,
        seg_full[kSegments], seg_empty[kSegments];
    __shared__ Segment segs[kSegments];
    __shared__ uint32_t tmem_slot;
    __shared__ int warp_part[kTileThreads / 32];
    __shared__ bool beyond;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = a.hq / a.hkv, per_tile = kTileRows / G;

    if (tid == 0) {
        for (int i = 0; i < S; ++i) {
            mbar_init(&full_bar[i], 1);
            mbar_init(&empty_bar[i], 2);  // both tiles' products
            mbar_init(&clean_bar[i], 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&q_bar[t], a.q_tma ? 1 : 4);
            mbar_init(&q_free[t], 1);
            for (int half = 0; half < 2; ++half) {
                mbar_init(&s_bar[t][half], 1);
                mbar_init(&p_bar[t][half], 4);
                mbar_init(&o_bar[t][half], 1);
            }
        }
        mbar_init(&drain_bar, 2);
        for (int i = 0; i < kSegments; ++i) {
            mbar_init(&seg_full[i], 1);
            mbar_init(&seg_empty[i], 11);  // all warps but the scheduling one
        }
        beyond = false;
        fence_mbar_init();
        prefetch_tensormap(&tmK);
        prefetch_tensormap(&tmV);
        if (a.q_tma) prefetch_tensormap(&tmQ);
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // not before: what came before us is then over
    // ---- the table of items: pairs before each sequence, blocks before each run of pairs
    const int seqs = min(a.batch.n_seqs - seq0, kTileSeqs);
    auto view = [&](int b) {
        bool bad = false;
        SeqView s = seq_view(a.batch, seq0 + b, a.page_size, &bad);
        if (bad) report_contents(a.status);
        if ((long long)s.n * G <= a.max_rows) s.n = 0;  // the rows kernel's
        return s;
    };
    // exclusive prefix sums of v[0 .. n) in place, the total at v[n]; `beyond` is set if one is more than `most`
    auto scan = [&](int* v, int n, int most) {
        const int each = (n + kTileThreads - 1) / kTileThreads, i0 = min(n, tid * each), i1 = min(n, i0 + each);
        int sum = 0;
        for (int i = i0; i < i1; ++i) sum += v[i];
        int incl = sum;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, incl, off);
            if (lane >= off) incl += x;
        }
        if (lane == 31) warp_part[warp] = incl;
        __syncthreads();
        int before = incl - sum;
        for (int w = 0; w < warp; ++w) before += warp_part[w];
        for (int i = i0; i < i1; ++i) {
            const int x = v[i];
            v[i] = before;
            before += x;
            if ((unsigned)before > (unsigned)most) beyond = true;
        }
        if (tid == kTileThreads - 1) v[n] = before;
        __syncthreads();
    };
    for (int b = tid; b < seqs; b += kTileThreads) seq_first[b] = (view(b).n + 2 * per_tile - 1) / (2 * per_tile);
    __syncthreads();
    // Sequences that share rows, between which cu_q descends, could have more pairs than the host's bound on the
    // 32-bit counts below allows for.  (One has at most 2^23, so that the sums cannot pass over the bound.)
    scan(seq_first, seqs, a.batch.n_tokens / (2 * per_tile) + a.batch.n_seqs);
    const int pairs = seq_first[seqs];
    if (pairs == 0 || beyond) return;
    auto seq_of_pair = [&](int p) {  // the last b with seq_first[b] <= p
        int lo2 = 0, hi2 = seqs;
        while (hi2 - lo2 > 1) {
            const int mid = (lo2 + hi2) / 2;
            if (seq_first[mid] <= p) lo2 = mid;
            else hi2 = mid;
        }
        return lo2;
    };
    const int run = (pairs + kTileEntries - 1) / kTileEntries, entries = (pairs + run - 1) / run;
    int most = 0;
    for (int e = tid; e < entries; e += kTileThreads) {
        int sum = 0, b = seq_of_pair(e * run);
        SeqView s = view(b);
        for (int p = e * run; p < min(pairs, (e + 1) * run); ++p) {
            while (seq_first[b + 1] <= p) s = view(++b);
            const int n = pair_of(a, s, p - seq_first[b], per_tile).blocks;
            sum += n;
            most = max(most, n);
        }
        cum[e] = sum;
    }
    most = __reduce_max_sync(0xffffffffu, most);
    __syncthreads();
    scan(cum, entries, INT_MAX);
    if (lane == 0) warp_part[warp] = most;
    __syncthreads();
    for (int w = 0; w < kTileThreads / 32; ++w) most = max(most, warp_part[w]);
    const int head_blocks = cum[entries], total = head_blocks * a.hkv, items = pairs * a.hkv;
    // Whole items, one to a CTA, unless cutting them saves more than a join costs.  32 heads of 64 dims: 257 new
    // tokens 13.2 us whole and 21.0 cut, 761 tokens 20.5 and 22.7, 1024 tokens 24.8 and 27.8; of 128 dims: 16.3 and
    // 30.2, 24.9 and 30.0, 29.4 and 36.5; 2000 tokens have too many items.
    const bool by_item = items <= (int)gridDim.x && most <= (total + (int)gridDim.x - 1) / (int)gridDim.x + kJoinBlocks;
    const int shares = by_item ? items : min((int)gridDim.x, total);
    if ((int)blockIdx.x >= shares) return;
    if (warp == 8) {
        tmem_alloc(&tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    auto wait = [&](uint64_t* bar, uint32_t phase) { return __all_sync(0xffffffffu, mbar_wait(bar, phase & 1u, a.status)); };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        // Every warp below walks as one; only single instructions are one thread's.
        bool ok = true, more = true;
        uint32_t n = 0;  // blocks so far
        if (warp == 11) {
            // ------------------------------------------------------------ scheduling, and NaN and Inf in V
            const int quota = total / shares, extra = total % shares;
            auto share = [&](int c) { return c * quota + min(c, extra); };
            const int cut = extra * (quota + 1);
            auto owner = [&](int x) { return x < cut ? x / (quota + 1) : extra + (x - cut) / quota; };
            const int begin = by_item ? 0 : share(blockIdx.x);
            int h, p, k = 0, b;
            if (by_item) {
                h = blockIdx.x / pairs;
                p = blockIdx.x % pairs;
                b = seq_of_pair(p);
            } else {
                h = begin / head_blocks;
                int y = begin % head_blocks, lo2 = 0, hi2 = entries;
                while (hi2 - lo2 > 1) {
                    const int mid = (lo2 + hi2) / 2;
                    if (cum[mid] <= y) lo2 = mid;
                    else hi2 = mid;
                }
                y -= cum[lo2];
                for (p = lo2 * run, b = seq_of_pair(p); run > 1; ++p) {
                    while (seq_first[b + 1] <= p) ++b;
                    const int blocks = pair_of(a, view(b), p - seq_first[b], per_tile).blocks;
                    if (y < blocks) break;
                    y -= blocks;
                }
                k = y;
            }
            int end = by_item ? INT_MAX : share(blockIdx.x + 1), pos = begin, handed = 0;
            auto hand_out = [&] {  // the next segment, if there is one
                if (pos >= end) return;
                const SeqView s = view(b);
                const Pair pr = pair_of(a, s, p - seq_first[b], per_tile);
                if (by_item) end = pr.blocks;
                const int k1 = min(pr.blocks, k + (end - pos)), item = pos - k;
                ok = wait(&seg_empty[handed % kSegments], (handed / kSegments) ^ 1);
                if (!ok) return;
                if (lane == 0) {
                    Segment& g = segs[handed % kSegments];
                    g.kb0 = pr.lo + k;
                    g.kb1 = pr.lo + k1;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        g.lo[t] = max(pr.t_lo[t], pr.lo + k);
                        g.hi[t] = min(pr.t_hi[t], pr.lo + k1);
                        g.whole_lo[t] = pr.whole_lo[t];
                        g.whole_hi[t] = pr.whole_hi[t];
                        g.rows[t] = pr.rows[t];
                        g.row0[t] = s.q0 + pr.first[t];
                        g.index[t] = s.kv - s.n + pr.first[t];
                    }
                    g.kv = s.kv;
                    g.seq = seq0 + b;
                    g.h = h;
                    g.complete = k == 0 && k1 == pr.blocks;
                    if (!g.complete) {
                        // a share's pieces: slot 2c for the item it begins in, 2c + 1 for a later one
                        g.slot = 2 * blockIdx.x + (item > begin);
                        g.c0 = owner(item);
                        g.pieces = owner(item + pr.blocks - 1) - g.c0 + 1;
                        g.first_slot = 2 * g.c0 + (item > share(g.c0));
                    }
                    g.more = pos + k1 - k < end;
                    g.odd = 0;
                    mbar_arrive(&seg_full[handed % kSegments]);
                }
                __syncwarp();
                ++handed;
                pos += k1 - k;
                k = 0;
                if (++p == pairs) {
                    p = 0;
                    ++h;
                    b = 0;
                }
                if (pos < end)
                    while (seq_first[b + 1] <= p) ++b;
            };
            for (int i = -1; ok && more; ++i) {
                hand_out();  // one ahead of the values looked over below
                if (!ok) break;
                if (i < 0) continue;
                Segment& g = segs[i % kSegments];
                more = g.more;
                // A weight of 0 times NaN or Inf is not 0: where some row does not see all keys of a block,
                // such values leave the block, and the rows that see them add them at the end.
                const int kb1 = g.kb1;
                for (int kb = g.kb0; ok && kb < kb1; ++kb, ++n) {
                    const uint32_t st = (2 * n + 1) % S;
                    ok = wait(&full_bar[st], (2 * n + 1) / S);
                    if (!ok) break;
                    if (g.masked(kb)) {
                        uint4* v = reinterpret_cast<uint4*>(ring + st * SB);
                        bool found = false;
#pragma unroll 8
                        for (int x = lane; x < SB / 16; x += 32) {
                            const uint4 q = v[x];
                            found |= odd16(q.x, kBf16) || odd16(q.x >> 16, kBf16) || odd16(q.y, kBf16) || odd16(q.y >> 16, kBf16) ||
                                     odd16(q.z, kBf16) || odd16(q.z >> 16, kBf16) || odd16(q.w, kBf16) || odd16(q.w >> 16, kBf16);
                        }
                        if (__any_sync(0xffffffffu, found)) {
                            for (int x = lane; x < SB / 2; x += 32) {
                                uint16_t* u = reinterpret_cast<uint16_t*>(v) + x;
                                if (odd16(*u, kBf16)) *u = 0;
                            }
                            if (lane == 0) g.odd = 1;
                            fence_proxy_async_smem();
                            __syncwarp();
                        }
                    }
                    if (lane == 0) mbar_arrive(&clean_bar[st]);
                    __syncwarp();
                }
            }
        } else if (warp == 9) {
            // ------------------------------------------------------------ loads: a lane has a chunk of one page
            const int rows = a.box_rows, chunks = kTileKeys / rows;
            for (int i = 0; ok && more; ++i) {
                ok = wait(&seg_full[i % kSegments], i / kSegments);
                if (!ok) break;
                const Segment& g = segs[i % kSegments];
                more = g.more;
                const int kb1 = g.kb1;
                for (int kb = g.kb0; ok && kb < kb1; ++kb, ++n) {
                    const int j = kb * kTileKeys + lane * rows;
                    // chunks past the end are read from outside the map, which gives zeros
                    int z = a.num_pages * a.hkv, y = 0;
                    if (lane < chunks && j < g.kv) {
                        const int at = a.page_shift >= 0 ? j >> a.page_shift : j / a.page_size;
                        const int page = a.batch.page_table[(int64_t)g.seq * a.batch.max_pages + at];
                        if (page >= 0 && page < a.num_pages) {
                            z = page * a.hkv + g.h;
                            y = j - at * a.page_size;
                        } else {
                            report_contents(a.status);
                        }
                    }
#pragma unroll
                    for (int side = 0; side < 2; ++side) {
                        const uint32_t it = 2 * n + side, st = it % S;
                        if (!ok) break;
                        ok = wait(&empty_bar[st], (it / S) ^ 1);
                        if (!ok) break;
                        if (lane == 0) mbar_arrive_expect_tx(&full_bar[st], SB);
                        __syncwarp();
                        if (lane < chunks) {
#pragma unroll
                            for (int slab = 0; slab < SLABS; ++slab)
                                tma_load_3d(ring + st * SB + slab * SLAB + lane * rows * 128, side ? &tmV : &tmK, slab * 64, y, z,
                                            &full_bar[st]);
                        }
                        __syncwarp();
                    }
                }
                if (lane == 0) mbar_arrive(&seg_empty[i % kSegments]);
                __syncwarp();
            }
            // a wait ran out: the copies under way still have to land before the CTA may end
            if (!ok)
                for (uint32_t it = 2 * n > S ? 2 * n - S : 0; it < 2 * n; ++it) wait(&full_bar[it % S], it / S);
        } else {
            // ------------------------------------------------------------ products: a warp to a tile
            // A block's keys are taken in halves, each with its own 64 columns of scores: the scores of a
            // half of block kb + 1 are asked for as soon as the weights of that half of kb have been used,
            // while the softmax is at the other half, so that it finds its next scores there.
            // Descriptors of the tile's Q, of stage 0 as keys and as values; steps and stages are added to
            // their address fields, in units of 16 bytes.
            const int t = warp == 8 ? 0 : 1;
            uint32_t q_phase = 0, p_phase = 0;
            const uint64_t q_desc = smem_desc(smem_u32(qs + t * QB), 16, 1024, kSwizzle128B);
            const uint64_t k_desc = smem_desc(smem_u32(ring), 16, 1024, kSwizzle128B);
            const uint64_t v_desc = smem_desc(smem_u32(ring), SLAB, 1024, kSwizzle128B);
            const uint32_t id_s = idesc_f16(kBf16, false, false, kTileRows, kTileKeys / 2);
            const uint32_t id_o = idesc_f16(kBf16, false, true, kTileRows, (a.D + 15) / 16 * 16);
            const uint32_t d_s = tmem + t * kTileKeys, d_o = tmem + 256 + t * 128;
            const int dims = (a.D + 15) / 16;
            uint32_t free_phase = 0, q_loads = 0;
            // A tile's queries: whole tokens of the key head's query heads, which lie in its rows' order.
            // Rows beyond the tile's hold other tokens' or old values; nothing of theirs is written.
            auto load_q = [&](const Segment& g) {
                if (!a.q_tma || g.lo[t] >= g.hi[t]) return;
                ++q_loads;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&q_bar[t], (uint32_t)(SLABS * 128 * G * per_tile));
                    for (int slab = 0; slab < SLABS; ++slab)
                        tma_load_3d(qs + t * QB + slab * SLAB, &tmQ, slab * 64, g.h * G, g.row0[t], &q_bar[t]);
                }
                __syncwarp();
            };
            for (int i = 0; ok && more; ++i) {
                ok = wait(&seg_full[i % kSegments], i / kSegments);
                if (!ok) break;
                const Segment& g = segs[i % kSegments];
                more = g.more;
                const int kb0 = g.kb0, kb1 = g.kb1, lo = g.lo[t], hi = g.hi[t];
                if (i == 0) load_q(g);
                // kb0 - 1 stands for the scores of the first block alone
                for (int kb = kb0 - 1; kb < kb1; ++kb) {
                    const uint32_t ks = (2 * n) % S, vs = (2 * n + S - 1) % S;  // keys of kb + 1, values of kb
                    const bool scores = kb + 1 < kb1, score = scores && kb + 1 >= lo && kb + 1 < hi, weigh = kb >= lo && kb < hi;
                    // Keys, values (looked over, and so there), weights of half 0 and queries: a lane waits for
                    // each.  Beside the products' reads of shared memory a wait takes some 250 clocks even when
                    // its phase is over (a mixed batch: 119.9 us one after another, 118.1 so).
                    const bool first = score && kb + 1 == lo;
                    const bool mine = lane == 0 ? scores : lane == 1 ? kb >= kb0 : lane == 2 ? weigh : lane == 3 && first;
                    uint64_t* const bar = lane == 0 ? &full_bar[ks] : lane == 1 ? &clean_bar[vs] : lane == 2 ? &p_bar[t][0] : &q_bar[t];
                    const uint32_t phase = lane == 0 ? 2 * n / S : lane == 1 ? (2 * n - 1) / S : lane == 2 ? p_phase : q_phase;
                    ok = __all_sync(0xffffffffu, !mine || mbar_wait(bar, phase & 1u, a.status));
                    q_phase += first;
                    const uint64_t vd = v_desc + vs * (SB >> 4), kd = k_desc + ks * (SB >> 4);
#pragma unroll 1
                    for (int half = 0; half < 2; ++half) {
                        if (half && weigh) ok = wait(&p_bar[t][1], p_phase);
                        if (!ok) break;
                        tc_fence_after();
                        if (elect_one()) {
                            if (weigh) {
                                const uint64_t vh = vd + half * (kTileKeys / 2 * 128 >> 4);
#pragma unroll
                                for (int d = 0; d < kTileKeys / 32; ++d)
                                    umma_f16_ts(d_o, d_s + half * 64 + d * 8, vh + d * (2048 >> 4), id_o, kb > lo || half != 0 || d != 0);
                                umma_commit(&o_bar[t][half]);
                            }
                            if (score) {
                                const uint64_t kh = kd + half * (kTileKeys / 2 * 128 >> 4);
#pragma unroll
                                for (int d = 0; d < DP / 16; ++d) {
                                    const int step = (d >> 2) * (SLAB >> 4) + (d & 3) * 2;  // Q and K have the same slabs
                                    if (d < dims) umma_f16(d_s + half * 64, q_desc + step, kh + step, id_s, d != 0);
                                }
                                umma_commit(&s_bar[t][half]);
                                if (half == 1 && kb + 2 >= hi) umma_commit(&q_free[t]);
                            }
                        }
                        __syncwarp();
                    }
                    if (!ok) break;
                    p_phase ^= weigh;
                    if (elect_one()) {
                        if (kb >= kb0) umma_commit(&empty_bar[vs]);
                        if (scores) umma_commit(&empty_bar[ks]);
                    }
                    __syncwarp();
                    if (scores) ++n;
                    if (!scores && more) {
                        // the next segment's queries, while this one's rows are written
                        ok = (lo >= hi || wait(&q_free[t], free_phase++)) && wait(&seg_full[(i + 1) % kSegments], (i + 1) / kSegments);
                        if (ok) load_q(segs[(i + 1) % kSegments]);
                    }
                }
                if (lane == 0) mbar_arrive(&seg_empty[i % kSegments]);
                __syncwarp();
            }
            // a wait ran out: queries under way still have to land before the CTA may end
            if (q_loads > q_phase) wait(&q_bar[t], q_phase);
            if (elect_one()) umma_commit(&drain_bar);  // all products have ended before TMEM is given back
            __syncwarp();
            wait(&drain_bar, 0);
        }
    } else {
        // ---------------------------------------------------------------- softmax: a thread to a row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int t = warp >> 2, row = tid & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's 32 lanes of TMEM
        const uint32_t s_tm = tmem + t * kTileKeys + lanes, o_tm = tmem + 256 + t * 128 + lanes;
        // Where TMA cannot read the queries: this warp's 32 rows of Q into the swizzled slabs, zeros beyond
        // the tile's rows and the head's dims.
        auto stage_q = [&](const Segment& g) {
            if (a.q_tma || g.lo[t] >= g.hi[t]) return;
            constexpr int PER = DP / 8, ROWS = 32 / PER;  // 16-byte chunks of a row; rows of one access
            const int c = lane % PER, rows = g.rows[t];
            const uint32_t dst = smem_u32(qs + t * QB + (c >> 3) * SLAB);
            const uint16_t* q = reinterpret_cast<const uint16_t*>(a.q) + (int64_t)g.row0[t] * a.ldq + (int64_t)g.h * G * a.D + c * 8;
            int r = (warp & 3) * 32 + lane / PER, token = r / G, head = r % G;
#pragma unroll 1
            for (int x = 0; x < 32; x += ROWS) {
                const bool in = r < rows && c * 8 < a.D;
                const uint16_t* at = in ? q + (int64_t)token * a.ldq + head * a.D : reinterpret_cast<const uint16_t*>(a.q);
                const uint32_t to = dst + r * 128 + (((c & 7) ^ (r & 7)) << 4);
                uint32_t w[4] = {0, 0, 0, 0};
                if (in)
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = (uint32_t)at[2 * e] | ((uint32_t)at[2 * e + 1] << 16);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                r += ROWS;
                head += ROWS;
                while (head >= G) {
                    head -= G;
                    ++token;
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_bar[t]);
            __syncwarp();
        };
        uint32_t s_phase = 0, o_phase = 0;
        bool ok = wait(&seg_full[0], 0), more = ok;
        if (ok) stage_q(segs[0]);
        for (int i = 0; ok && more; ++i) {
            const Segment& g = segs[i % kSegments];
            const int kb0 = g.lo[t], kb1 = g.hi[t];
            const bool valid = row < g.rows[t];
            const Seen sr = valid ? seen_at(a, g.kv, g.index[t] + row / G) : Seen{0, 0};
            float m = -INFINITY, l = 0.0f;  // the reference (log2 units, less LOG2_1) and the sum of 2^(s - m)
            // The scores of half `half` at keys j0 .. are asked for; they are there after tmem_ld_wait.
            auto fetch = [&](uint32_t (&sa)[32], uint32_t (&sb)[32], const int half) {
                ok = wait(&s_bar[t][half], s_phase);
                if (!ok) return;
                s_phase ^= half;
                tc_fence_after();
                tmem_ld32(s_tm + half * (kTileKeys / 2), sa);
                tmem_ld32(s_tm + half * (kTileKeys / 2) + 32, sb);
            };
            // Masks, the maximum, and with it the reference; O is rescaled where that moves.
            auto refer = [&](uint32_t (&sa)[32], uint32_t (&sb)[32], const int half, int j0) {
                tmem_ld_wait();
                tmem_use(sa);
                tmem_use(sb);
                if (j0 < g.whole_lo[t] || j0 + kTileKeys / 2 > g.whole_hi[t]) {
                    const int c0 = sr.lo - j0, c1 = sr.hi - j0;
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        if (e < c0 || e >= c1) sa[e] = 0xFF800000u;
                        if (e + 32 < c0 || e + 32 >= c1) sb[e] = 0xFF800000u;
                    }
                }
                float x0 = -INFINITY, x1 = -INFINITY, x2 = -INFINITY, x3 = -INFINITY;
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    x0 = max3(x0, __uint_as_float(sa[e]), __uint_as_float(sa[e + 1]));
                    x1 = max3(x1, __uint_as_float(sa[e + 2]), __uint_as_float(sa[e + 3]));
                    x2 = max3(x2, __uint_as_float(sb[e]), __uint_as_float(sb[e + 1]));
                    x3 = max3(x3, __uint_as_float(sb[e + 2]), __uint_as_float(sb[e + 3]));
                }
                const float top = fmaxf(fmaxf(x0, x1), fmaxf(x2, x3)) * a.scale_log2;
                const bool grown = top > m + (LOG2_1 + kGrowth);
                if (__any_sync(0xffffffffu, grown)) {
                    const float f = grown ? ex2(m - (top - LOG2_1)) : 1.0f;
                    if (grown) m = top - LOG2_1;
                    l *= f;
                    if (j0 > kb0 * kTileKeys) {
                        // O as the half before left it.  A barrier to each half: the phases before that one's
                        // are then over for certain, and a parity tells only one phase from the next.
                        ok = wait(&o_bar[t][half ^ 1], half ? o_phase : o_phase - 1);
                        if (!ok) return;
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < DP; c += 16) {
                            uint32_t o[16];
                            tmem_ld16(o_tm + c, o);
                            tmem_ld_wait();
                            tmem_use<16>(o);
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tmem_st16(o_tm + c, o);
                        }
                    }
                }
            };
            // The weights, in place of the scores.
            auto weigh = [&](const uint32_t (&sa)[32], const uint32_t (&sb)[32], const int half) {
                const float neg = m == -INFINITY ? 0.0f : -m;
                float2 sum = make_float2(0.0f, 0.0f);
                const float2 sc2 = make_float2(a.scale_log2, a.scale_log2), neg2 = make_float2(neg, neg);
                auto part = [&](const uint32_t (&s)[32], int at) {
                    uint32_t w[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float2 z = __ffma2_rn(make_float2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), sc2, neg2);
                        const float2 w2 = make_float2(ex2(z.x), ex2(z.y));
                        // The sum takes the weights before they are rounded to the products' type.  Taken after
                        // (errors against 64 bits 1.16 to 1.25 times those of one rounding, not 1.27 to 1.41), prompt
                        // 761 takes 21.2 us for 20.4, 4096 over 4096 448 for 441.
                        sum = __fadd2_rn(sum, w2);
                        w[e] = pack2<T>(w2.x, w2.y);
                    }
                    tmem_st16(s_tm + half * (kTileKeys / 2) + at / 2, w);
                };
                part(sa, 0);
                part(sb, 32);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_bar[t][half]);
                __syncwarp();
                o_phase += half;  // blocks so far
                l += sum.x + sum.y;
            };
            for (int j0 = kb0 * kTileKeys; j0 < kb1 * kTileKeys; j0 += kTileKeys / 2) {
                const int half = (j0 / (kTileKeys / 2)) & 1;
                uint32_t sa[32], sb[32];
                fetch(sa, sb, half);
                if (!ok) break;
                refer(sa, sb, half, j0);
                if (!ok) break;
                weigh(sa, sb, half);
            }
            if (!ok) break;
            const bool took = kb0 < kb1;
            if (took) {
                ok = wait(&o_bar[t][1], o_phase - 1);
                if (!ok) break;
                tc_fence_after();
            }
            // the next segment's queries before this one's rows are written: their first scores run beside that
            more = g.more;
            if (more) {
                ok = wait(&seg_full[(i + 1) % kSegments], (i + 1) / kSegments);
                if (ok) stage_q(segs[(i + 1) % kSegments]);
            }
            const bool odd = took && valid && *reinterpret_cast<const volatile int*>(&g.odd) != 0;
            // 32 values of O; every lane of the warp comes here
            auto load_o = [&](float (&o)[32], int d0) {
                __syncwarp();
                uint32_t r[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) r[e] = 0;
                if (took) {
                    tmem_ld32(o_tm + d0, r);
                    tmem_ld_wait();
                    tmem_use(r);
                }
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __uint_as_float(r[e]);
                if (odd) {  // NaN and Inf that this row sees
#pragma unroll 1
                    for (int j = max(sr.lo, kb0 * kTileKeys); j < min(sr.hi, kb1 * kTileKeys); ++j) {
                        if (!g.masked(j / kTileKeys)) continue;
                        const int page = a.batch.page_table[(int64_t)g.seq * a.batch.max_pages + j / a.page_size];
                        if (page < 0 || page >= a.num_pages) continue;
                        const uint16_t* v = reinterpret_cast<const uint16_t*>(a.vc) +
                                            (((int64_t)page * a.hkv + g.h) * a.page_size + j % a.page_size) * a.D + d0;
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (d0 + e < a.D && odd16(v[e], kBf16)) o[e] += unpack2<T>(v[e]).x;
                    }
                }
            };
            T* const out_row = reinterpret_cast<T*>(a.out) + (int64_t)(g.row0[t] + row / G) * a.ldo + (int64_t)(g.h * G + row % G) * a.D;
            auto write = [&](const float (&o)[32], int d0, float inv) {
#pragma unroll
                for (int e = 0; e < 32; e += 16) {
                    uint32_t w[8];
#pragma unroll
                    for (int x = 0; x < 8; ++x) w[x] = pack2<T>(o[e + 2 * x] * inv, o[e + 2 * x + 1] * inv);
                    if (a.out_wide && d0 + e + 16 <= a.D) {
                        // a whole 32-byte sector to a thread
                        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(out_row + d0 + e), "r"(w[0]), "r"(w[1]),
                                     "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                                     : "memory");
                        continue;
                    }
#pragma unroll
                    for (int x = 0; x < 16; x += 8) {
                        if (d0 + e + x >= a.D) break;
                        T* out = out_row + d0 + e + x;
                        if (a.out_vec) {
                            *reinterpret_cast<uint4*>(out) = make_uint4(w[x / 2], w[x / 2 + 1], w[x / 2 + 2], w[x / 2 + 3]);
                        } else {
#pragma unroll
                            for (int y = 0; y < 8; ++y) out[y] = from_f32<T>(o[e + x + y] * inv);
                        }
                    }
                }
            };
            const bool any = (warp & 3) * 32 < g.rows[t];  // this warp has rows
            if (any && g.complete) {
                const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll 1
                for (int d0 = 0; d0 < a.D; d0 += 32) {
                    float o[32];
                    load_o(o, d0);
                    if (valid) write(o, d0, inv);
                }
            } else if (any) {
                // a piece: dims outside, rows inside, so that a warp writes whole lines
                auto piece_of = [&](int slot) { return a.partials + (int64_t)(2 * slot + t) * PIECE + row; };
                float* piece = piece_of(g.slot);
#pragma unroll 1
                for (int d0 = 0; d0 < a.D; d0 += 32) {
                    float o[32];
                    load_o(o, d0);
#pragma unroll
                    for (int e = 0; e < 32; ++e) __stcg(piece + (d0 + e) * kTileRows, o[e]);
                }
                __stcg(piece + DP * kTileRows, m);
                __stcg(piece + (DP + 1) * kTileRows, l);
                // the last warp to come to these rows joins their pieces, in order
                __threadfence();
                __syncwarp();
                unsigned last = 0;
                if (lane == 0) {
                    unsigned int* ticket = a.tickets + 8 * g.c0 + warp;
                    last = atomicAdd(ticket, 1u) == (unsigned)(g.pieces - 1);
                    if (last) *ticket = 0;
                }
                if (__shfl_sync(0xffffffffu, last, 0)) {
                    __threadfence();
                    const int pieces = g.pieces;
                    auto slot_of = [&](int x) { return x == 0 ? g.first_slot : 2 * (g.c0 + x); };
                    float top = -INFINITY, den = 0.0f;
                    for (int x = 0; x < pieces; ++x) top = fmaxf(top, __ldcg(piece_of(slot_of(x)) + DP * kTileRows));
                    const float mu = top == -INFINITY ? 0.0f : top;
                    for (int x = 0; x < pieces; ++x) {
                        const float* pc = piece_of(slot_of(x));
                        den += __ldcg(pc + (DP + 1) * kTileRows) * ex2(__ldcg(pc + DP * kTileRows) - mu);
                    }
                    const float inv = den > 0.0f ? 1.0f / den : 0.0f;
#pragma unroll 1
                    for (int d0 = 0; d0 < a.D; d0 += 32) {
                        float o[32];
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = 0.0f;
#pragma unroll 1
                        for (int x = 0; x < pieces; ++x) {
                            const float* pc = piece_of(slot_of(x));
                            const float f = ex2(__ldcg(pc + DP * kTileRows) - mu);
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] += __ldcg(pc + (d0 + e) * kTileRows) * f;
                        }
                        if (valid) write(o, d0, inv);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&seg_empty[i % kSegments]);
            __syncwarp();
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 8) tmem_dealloc(tmem, 512);
}

template <typename T, int DP>
cudaError_t launch_tiles(const mgpu_k::LaunchCtx& c, const CUtensorMap& mk, const CUtensorMap& mv, const mgpu_k::AttendArgs& a) {
    auto kern = attend_tile_kernel<T, DP>;
    static std::atomic<uint64_t> configured{0};
    cudaError_t e = allow_smem(kern, tile_smem<DP>(), configured);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)c.sm_count);
    cfg.blockDim = dim3(kTileThreads);
    cfg.dynamicSmemBytes = tile_smem<DP>();
    cfg.stream = c.stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    // [tokens][heads][dims] of q; a box is a tile's tokens, a key head's query heads and 64 dims
    const int group = a.hq / a.hkv;
    const int64_t dims[3] = {a.D, a.hq, a.batch.n_tokens}, strides[2] = {(int64_t)a.D * 2, a.ldq * 2};
    const int box[3] = {64, group, kTileRows / group};
    CUtensorMap mq = {};
    mgpu_k::AttendArgs b = a;
    b.q_tma = a.q_vec && mgpu_k::make_tensor_map_u16_3d(&mq, a.q, dims, strides, box, true);
    for (int seq0 = 0; seq0 < a.batch.n_seqs && e == cudaSuccess; seq0 += kTileSeqs)
        e = cudaLaunchKernelEx(&cfg, kern, mk, mv, mq, b, seq0);
    return e;
}

template <typename T>
cudaError_t launch_attend(const mgpu_k::LaunchCtx& c, const CUtensorMap& mk, const CUtensorMap& mv, const mgpu_k::AttendArgs& a) {
    cudaError_t e = cudaSuccess;
    const bool narrow = a.max_rows <= 8;
    if (a.max_rows > 0 && narrow) e = a.D <= 64 ? launch_rows<T, 64, true>(c, mk, mv, a) : launch_rows<T, 128, true>(c, mk, mv, a);
    else if (a.max_rows > 0) e = a.D <= 64 ? launch_rows<T, 64, false>(c, mk, mv, a) : launch_rows<T, 128, false>(c, mk, mv, a);
    if (e != cudaSuccess || !mgpu_k::attend_many_rows(a)) return e;
    return a.D <= 64 ? launch_tiles<T, 64>(c, mk, mv, a) : launch_tiles<T, 128>(c, mk, mv, a);
}

}  // namespace

namespace mgpu_k {

size_t attend_scratch_bytes(int sm_count, bool many_rows) {
    return (size_t)sm_count * 2 * (many_rows ? 2 * kTileRows : kRowsMax) * (128 + 2) * sizeof(float);
}
bool attend_many_rows(const AttendArgs& a) { return a.batch.max_q_len * (int64_t)(a.hq / a.hkv) > kRowsMax; }

bool make_cache_map(CUtensorMap* m, const void* side, int type, int num_pages, int page_size, int kv_heads, int head_dim) {
    int rows = kBoxRows;
    while (page_size % rows) rows /= 2;
    const int64_t dims[3] = {head_dim, page_size, (int64_t)num_pages * kv_heads};
    const int64_t strides[2] = {(int64_t)head_dim * 2, (int64_t)page_size * head_dim * 2};
    const int box[3] = {64, rows, 1};
    return make_tensor_map_u16_3d(m, side, dims, strides, box, true);
}

cudaError_t paged_attention(const LaunchCtx& c, const CUtensorMap& mk, const CUtensorMap& mv, const AttendArgs& in) {
    AttendArgs a = in;
    a.box_rows = kBoxRows;
    while (a.page_size % a.box_rows) a.box_rows /= 2;
    // The most rows that go to the kernel for few.  One sequence of a chunk: none, however few it turns out to
    // have.  Where no sequence has more than 8: those, whose weights' rests are then free.  Beside chunks the same,
    // if single tokens have no more than 8 (4 chunks of 300 and 20 single tokens of 4 rows: 117.7 us, 119.3 with
    // 16; 20 times 3 tokens, which are then tiles: 110 and 128; 60 times 4 tokens: 204 and 202).
    const int64_t group = a.hq / a.hkv;
    const bool many = attend_many_rows(a);
    a.max_rows = many && a.batch.n_seqs == 1 ? 0 : a.batch.max_q_len * group <= 8 || (many && group <= 8) ? 8 : kRowsMax;
    a.page_shift = -1;
    for (int i = 3; i < 31; ++i)
        if (a.page_size == 1 << i) a.page_shift = i;
    a.q_vec = ((uintptr_t)a.q & 15) == 0 && a.ldq % 8 == 0;
    a.out_vec = ((uintptr_t)a.out & 15) == 0 && a.ldo % 8 == 0;
    a.out_wide = ((uintptr_t)a.out & 31) == 0 && a.ldo % 16 == 0 && a.D % 16 == 0;
    a.out_pairs = ((uintptr_t)a.out & 3) == 0 && a.ldo % 2 == 0;
    return a.type == MGPU_F16 ? launch_attend<__half>(c, mk, mv, a) : launch_attend<__nv_bfloat16>(c, mk, mv, a);
}

}  // namespace mgpu_k
