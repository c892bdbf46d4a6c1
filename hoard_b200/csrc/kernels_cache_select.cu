// kernels_cache_select.cu -- choosing rows and blocks of a KV cache: eviction by accumulated weight, the
// blocks' bounds and scores, the selection of blocks, and the moves of rows.
//
// Both selections are "the k largest of n keys, the lower index where equal", n from a few to 10^5. The keys of a
// problem sit in the shared memory of one CTA, or where there are many in that of a cluster of eight, each CTA a
// contiguous range so that order is kept. The threshold is narrowed by radix, eleven bits at a time from the
// top (the exponent of a weight and two bits of its mantissa, the exponent of a score), histograms added up over the
// cluster through distributed shared memory, until the bin that holds the k-th key holds no more than are
// wanted: two or three passes. Counting ranks by pairs is n^2, and a sort moves what is not asked for.
#include "common.cuh"
#include "kernels_cache.h"
#include "async_copy.cuh"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace hoard {

namespace {

constexpr int CL = 8;                    // CTAs of a cluster (the portable maximum)
// 512 threads: two CTAs of a cluster fit on an SM (with 1024 they do not, and of 16 clusters some wait for a second wave:
// 65521 rows x 16 heads took 62 us), and barriers are cheaper
constexpr int SEL_THREADS = 512, SEL_WARPS = SEL_THREADS / 32;
constexpr int DIGIT = 11, BINS = 1 << DIGIT;

// Shared state of a selection
struct Select {
    unsigned hist[2][BINS];
    unsigned warp[2][SEL_WARPS];         // one value per warp, alternately (a scan's values may still be read)
    unsigned seg[CL], found[3];          // cluster: segment totals; bin, count in it, count above it
    uint2 bits[2][SEL_WARPS];            // OR and AND of the keys of the last bin, alternately
    unsigned ex[2];                      // this CTA's totals, for prefixes over the cluster
};

// exclusive prefix sum over the CTA of one value per thread; total receives the sum. `use`: 0, 1, 0, ..
__device__ __forceinline__ unsigned block_scan(Select& s, int use, unsigned v, unsigned& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto scan32 = [&](unsigned x) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        return x;
    };
    const unsigned x = scan32(v);
    if (lane == 31) s.warp[use][warp] = x;
    __syncthreads();
    const unsigned w = scan32(lane < SEL_WARPS ? s.warp[use][lane] : 0);
    total = __shfl_sync(0xffffffffu, w, SEL_WARPS - 1);
    const unsigned before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
    return (warp ? before : 0) + x - v;
}

// sums over the cluster's CTAs before this one and over all of `total` (a slot is used once, so nothing overwrites it)
template <int CLN>
__device__ __forceinline__ void cluster_sums(Select& s, int slot, unsigned total, unsigned& before, unsigned& all) {
    before = 0;
    all = total;
    if constexpr (CLN > 1) {
        cg::cluster_group cl = cg::this_cluster();
        if (threadIdx.x == 0) s.ex[slot] = total;
        cl.sync();
        unsigned v[CLN];
#pragma unroll
        for (int r = 0; r < CLN; ++r) v[r] = *cl.map_shared_rank(&s.ex[slot], r);
        all = 0;
#pragma unroll
        for (int r = 0; r < CLN; ++r) {
            all += v[r];
            if (r < (int)cl.block_rank()) before += v[r];
        }
    }
}

// Up to 32 strips of SEL_THREADS flags, bit k of a thread's mask its flag in strip k: leaves in hist[0] for each (strip,
// warp) the number of flags before it in index order, which is also returned for (strip, warp) = thread in `at`, with
// its own number of flags; total receives the sum. The caller synchronises before others' entries are read.
constexpr int SPAN = 32 * SEL_THREADS;
static_assert(32 * SEL_WARPS == SEL_THREADS, "one (strip, warp) per thread");
__device__ __forceinline__ unsigned strip_scan(Select& s, unsigned mask, unsigned& at, unsigned& total) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned any = __reduce_or_sync(0xffffffffu, mask);
    // lane k keeps strip k's count of this warp
    unsigned mine = 0;
    for (unsigned left = any; left; left &= left - 1) {
        const int k = __ffs(left) - 1;
        const unsigned b = __ballot_sync(0xffffffffu, mask >> k & 1);
        if (lane == k) mine = __popc(b);
    }
    s.hist[0][lane * SEL_WARPS + warp] = mine;
    __syncthreads();
    const unsigned v = s.hist[0][tid];
    at = block_scan(s, 1, v, total);
    s.hist[0][tid] = at;
    return v;
}

// The bin, counted from the top of the histogram, that holds the need-th key: its number, its count, the count above.
// Every CTA of a cluster adds up and searches its share of the bins.
template <int CLN>
__device__ __forceinline__ void find_bin(Select& s, const unsigned* hist, unsigned need, unsigned& bin, unsigned& in_bin,
                                         unsigned& above) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int SHARE = BINS / CLN, PER = CLN == 1 ? BINS / SEL_THREADS : 1, LAST = SHARE / PER;      // threads with bins
    unsigned mine[PER] = {}, sum = 0, before = 0;
    int top = 0;                                       // this thread's highest bin
    if constexpr (CLN == 1) {
        __syncthreads();
        top = BINS - 1 - PER * threadIdx.x;
#pragma unroll
        for (int i = 0; i < PER; ++i) mine[i] = hist[top - i];
    } else {
        cg::cluster_group cl = cg::this_cluster();
        cl.sync();
        top = BINS - 1 - SHARE * (int)cl.block_rank() - threadIdx.x;
        if (threadIdx.x < LAST) {
            unsigned v[CLN];
#pragma unroll
            for (int r = 0; r < CLN; ++r) v[r] = cl.map_shared_rank(hist, r)[top];
#pragma unroll
            for (int r = 0; r < CLN; ++r) mine[0] += v[r];
        }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += mine[i];
    const unsigned in_warp = __reduce_add_sync(0xffffffffu, sum);
    if (lane == 0) s.warp[0][warp] = in_warp;
    __syncthreads();
    // every warp: the warps' totals, and which of them holds the key
    const unsigned w = lane < LAST / 32 ? s.warp[0][lane] : 0;
    unsigned incl = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if constexpr (CLN > 1) {
        cg::cluster_group cl = cg::this_cluster();
        const unsigned total = __shfl_sync(0xffffffffu, incl, 31);
        if (threadIdx.x < CLN) cl.map_shared_rank(s.seg, threadIdx.x)[cl.block_rank()] = total;
        cl.sync();
#pragma unroll
        for (int r = 0; r < CLN; ++r)
            if (r < (int)cl.block_rank()) before += s.seg[r];
    }
    const unsigned below = before + incl - w;
    const unsigned hit = __ballot_sync(0xffffffffu, below < need && below + w >= need);
    if (hit && warp == __ffs(hit) - 1) {
        unsigned x = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        unsigned up = __shfl_sync(0xffffffffu, below, warp) + x - sum;           // keys above this thread's bins
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (up < need && up + mine[i] >= need) {
                const unsigned f[3] = {(unsigned)(top - i), mine[i], up};
#pragma unroll
                for (int k = 0; k < 3; ++k) {
                    if constexpr (CLN == 1) s.found[k] = f[k];
                    else
                        for (int r = 0; r < CLN; ++r) cg::this_cluster().map_shared_rank(s.found, r)[k] = f[k];
                }
            }
            up += mine[i];
        }
    }
    if constexpr (CLN == 1) __syncthreads();
    else cg::this_cluster().sync();
    bin = s.found[0];
    in_bin = s.found[1];
    above = s.found[2];
}

// The `need` largest of the keys, the lower index where equal: afterwards this CTA's i-th key is in if
// (key >> shift) > prefix, or == prefix and i <= cut. key(i): this CTA's i-th key.
template <typename K> struct Threshold {
    K prefix;
    int shift, cut;
    __device__ __forceinline__ bool in(K key, int i) const {
        const K k = key >> shift;
        return k > prefix || (k == prefix && i <= cut);
    }
};
template <int CLN, int BITS, typename K, typename Key>
__device__ __forceinline__ Threshold<K> select_threshold(Select& s, Key key, int n_local, int need) {
    // weights are often equal (rows that nothing looked at): one CTA sees that in the second pass
    constexpr bool SAME = CLN == 1 && BITS <= 32;
    const int tid = threadIdx.x;
    for (int i = tid; i < 2 * BINS; i += SEL_THREADS) s.hist[0][i] = 0;
    __syncthreads();
    Threshold<K> th{0, BITS, 0x7fffffff};
    for (int pass = 0;; ++pass) {
        const int width = min(DIGIT, th.shift);
        th.shift -= width;
        unsigned* hist = s.hist[pass & 1];
        unsigned any = 0, every = ~0u;                 // bits of the bin's keys
        for (int i = tid; i < n_local; i += SEL_THREADS) {
            const K k = key(i);
            const unsigned d = (unsigned)(k >> th.shift) & ((1u << width) - 1);
            if (pass == 0 || (k >> (th.shift + width)) == th.prefix) {
                atomicAdd(&hist[d], 1u);
                any |= (unsigned)k;
                every &= (unsigned)k;
            }
        }
        if (SAME && pass) {
            any = __reduce_or_sync(0xffffffffu, any);
            every = __reduce_and_sync(0xffffffffu, every);
            if ((tid & 31) == 0) s.bits[pass & 1][tid >> 5] = make_uint2(any, every);
        }
        unsigned bin, in_bin, above;
        find_bin<CLN>(s, hist, (unsigned)need, bin, in_bin, above);
        th.prefix = th.prefix << width | bin;
        need -= (int)above;
        if (SAME && pass) {                            // the bin's keys are one key: no more digits to look at
            any = 0, every = ~0u;
#pragma unroll
            for (int w = 0; w < SEL_WARPS; ++w) {
                const uint2 b = s.bits[pass & 1][w];
                any |= b.x;
                every &= b.y;
            }
            if (any == every) {
                th.prefix = any;
                th.shift = 0;
            }
        }
        if (in_bin == (unsigned)need) return th;
        if (th.shift == 0) break;
        // the next pass's counts are zero already; these are made so for the pass after it
        for (int i = tid; i < BINS; i += SEL_THREADS) hist[i] = 0;
    }
    // more equal keys than are wanted: the index of the need-th of them
    unsigned total, before = 0;
    if constexpr (CLN > 1) {
        unsigned mine = 0, all;
        for (int i = tid; i < n_local; i += SEL_THREADS) mine += key(i) == th.prefix;
        block_scan(s, 0, mine, total);
        cluster_sums<CLN>(s, 0, total, before, all);
        if (before + total <= (unsigned)need) return th;             // uniform over the CTA
        th.cut = -1;
        if (before >= (unsigned)need) return th;
    } else {
        th.cut = -1;
    }
    for (int i0 = 0; i0 < n_local; i0 += SPAN) {
        unsigned mask = 0, at;
        const int strips = min(32, (n_local - i0 + SEL_THREADS - 1) / SEL_THREADS);
#pragma unroll 4
        for (int k = 0; k < strips; ++k) {
            const int i = i0 + k * SEL_THREADS + tid;
            mask |= (unsigned)(i < n_local && key(i) == th.prefix) << k;
        }
        const unsigned v = strip_scan(s, mask, at, total), x = (unsigned)need - 1 - before;
        if (at <= x && x < at + v) {                   // one thread, at most: its (strip, warp) holds the key
            s.found[0] = tid;
            s.found[1] = x - at;
        }
        __syncthreads();
        if (x < total) {                               // uniform
            const int k = s.found[0] / SEL_WARPS, w = s.found[0] % SEL_WARPS;
            const unsigned b = __ballot_sync(0xffffffffu, mask >> k & 1), j = s.found[1];
            if (tid >> 5 == w && (mask >> k & 1) && __popc(b & ((1u << (tid & 31)) - 1)) == (int)j)
                s.found[2] = i0 + k * SEL_THREADS + tid;
            __syncthreads();
            th.cut = (int)s.found[2];
            break;
        }
        before += total;
    }
    __syncthreads();
    return th;
}

// Calls emit(i, rank) for every flagged index of this CTA, rank counted over the cluster in index order, after
// begin(number of flagged ones over the cluster).
template <int CLN, typename Flag, typename Begin, typename Emit>
__device__ __forceinline__ void ranked(Select& s, Flag flag, int n_local, Begin begin, Emit emit) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto flags = [&](int i0) {
        unsigned mask = 0;
        const int strips = min(32, (n_local - i0 + SEL_THREADS - 1) / SEL_THREADS);
#pragma unroll 4
        for (int k = 0; k < strips; ++k) {
            const int i = i0 + k * SEL_THREADS + tid;
            mask |= (unsigned)(i < n_local && flag(i)) << k;
        }
        return mask;
    };
    auto report = [&](int i0, unsigned mask, unsigned before) {
        const int strips = min(32, (n_local - i0 + SEL_THREADS - 1) / SEL_THREADS);
#pragma unroll 4
        for (int k = 0; k < strips; ++k) {
            const unsigned b = __ballot_sync(0xffffffffu, mask >> k & 1);
            if (mask >> k & 1)
                emit(i0 + k * SEL_THREADS + tid, before + s.hist[0][k * SEL_WARPS + warp] + __popc(b & ((1u << lane) - 1)));
        }
    };
    unsigned total, before, all, at;
    if (CLN == 1 || n_local <= SPAN) {
        const unsigned mask = flags(0);
        strip_scan(s, mask, at, total);
        cluster_sums<CLN>(s, 1, total, before, all);
        begin(all);
        __syncthreads();                               // the scan's ranks are in place
        report(0, mask, before);
        return;
    }
    unsigned mine = 0;
    for (int i0 = 0; i0 < n_local; i0 += SPAN) mine += __popc(flags(i0));
    __syncthreads();
    block_scan(s, 0, mine, total);
    cluster_sums<CLN>(s, 1, total, before, all);
    begin(all);
    for (int i0 = 0; i0 < n_local; i0 += SPAN) {
        const unsigned mask = flags(i0);
        __syncthreads();
        strip_scan(s, mask, at, total);
        __syncthreads();
        report(i0, mask, before);
        before += total;
    }
}

// ---- eviction -------------------------------------------------------------------------------------------------
// Key of a row: protected rows above everything; weights in order; NaN below everything. -0 equals +0.
constexpr int EV_KEYS = 40960;           // keys that a CTA of a cluster holds in shared memory (160 KiB)
// Rows up to which one CTA chooses alone. One against a cluster, 4 / 16 heads: 13.7 / 15.2 us against 15.2 / 19.5 for 8000
// rows, 17.8 / 19.2 against 15.5 / 19.7 for 12000, 47 / 66 against 23 / 43 for 30000.
constexpr int EV_SINGLE = 10240;
// Moves up to which that CTA makes them itself, one a warp: an SM moves some 35 bytes a clock, a second kernel starts in
// 1.5 us. By the CTA against the kernel, heads of 128 / 256 dims: at most 32 moves 6.3 / 7.7 us against 6.3 / 6.6, 64 moves 7.5 / 9.1
// against 7.2 / 7.5, 256 moves 10.4 / 13.3 against 8.2 / 8.6.
constexpr int EV_FUSED = 16, EV_MOVES = 2;
__device__ __forceinline__ unsigned evict_key(float acc, int pos, int n_sink, int recent_from) {
    if (pos < n_sink || pos >= recent_from) return 0xFFFFFFFFu;
    if (acc != acc) return 0u;
    const unsigned b = __float_as_uint(acc + 0.f);
    return b >> 31 ? ~b : b | 0x80000000u;
}
// Moves i0 .. i1 - 1, at most N: K and V rows by 16-byte pieces, all loads before the first store. Rows read are at or
// above n_keep, rows written below it.
template <int N>
__device__ __forceinline__ void move_rows(const CacheEvict& e, int kv, const int32_t* to, const int32_t* from, int i0,
                                          int i1) {
    static_assert(N <= 32, "a lane for each row's weight and position");
    const int lane = threadIdx.x & 31, c16 = e.hd / 8;
    const int64_t hb = (int64_t)kv * e.max_rows;
    const bool mine = lane < i1 - i0;                  // lane k: row k's weight and position
    int t1 = -1, f1 = 0, p1 = 0;
    float a1 = 0.f;
    if (mine) {
        t1 = to[i0 + lane];
        f1 = from[i0 + lane];
        a1 = e.acc[hb + f1];
        p1 = e.pos[hb + f1];
    }
    for (int p = lane; p < (2 * c16 + 31) / 32 * 32; p += 32) {
        char* c = static_cast<char*>(p < c16 ? e.kc : e.vc) + (int64_t)kv * e.hs * 2 + (p < c16 ? p : p - c16) * 16;
        uint4 v[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int f = __shfl_sync(0xffffffffu, f1, k);
            if (i0 + k < i1 && p < 2 * c16) v[k] = *reinterpret_cast<const uint4*>(c + (int64_t)f * e.rs * 2);
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int t = __shfl_sync(0xffffffffu, t1, k);
            if (i0 + k < i1 && p < 2 * c16) *reinterpret_cast<uint4*>(c + (int64_t)t * e.rs * 2) = v[k];
        }
    }
    if (mine) {
        e.acc_out[hb + t1] = a1;
        e.pos_out[hb + t1] = p1;
    }
}
// Bound by barriers and dependent shared loads: 2304 rows 4.3 us to the threshold (two passes, equal weights) and 1.8 for the
// ranks; 65521 rows by a cluster 3.6 for the keys, 7.8 to the threshold, 5.6 for the ranks.
// Grid (CLN, n_kv). Lists the rows to fill and the rows to move (ascending both), copies acc and pos of the rows below
// n_keep to their outputs, and makes the moves itself where there are few (to, from then sit in shared memory). HELD: a CTA's keys fit in shared memory;
// otherwise they are formed again each time.
template <int CLN, bool HELD>
__global__ void __launch_bounds__(SEL_THREADS) k_evict_choose(const CacheEvict e, const bool fused) {
    pdl_enter();
    extern __shared__ unsigned s_key[];
    __shared__ Select sel;
    __shared__ int32_t s_to[CLN == 1 ? EV_FUSED : 1], s_from[CLN == 1 ? EV_FUSED : 1];
    const int kv = blockIdx.y, rank = CLN == 1 ? 0 : blockIdx.x, tid = threadIdx.x;
    const float* acc = e.acc + (int64_t)kv * e.max_rows;
    const int32_t* pos = e.pos + (int64_t)kv * e.max_rows;
    const int first = (int)((int64_t)e.n_rows * rank / CLN), last = (int)((int64_t)e.n_rows * (rank + 1) / CLN);
    const int n = last - first;
    // rows that stay are copied where the outputs are other buffers; rows that are filled are written again, later
    float* acc_out = e.acc_out + (int64_t)kv * e.max_rows;
    int32_t* pos_out = e.pos_out + (int64_t)kv * e.max_rows;
    const bool copy = e.acc_out != e.acc || e.pos_out != e.pos;
    auto fresh = [&](int i) { return evict_key(acc[first + i], pos[first + i], e.n_sink, e.recent_from); };
    if constexpr (HELD) {
        for (int i0 = tid; i0 < n; i0 += 8 * SEL_THREADS) {
            float a[8];
            int p[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (i0 + k * SEL_THREADS < n) {
                    a[k] = acc[first + i0 + k * SEL_THREADS];
                    p[k] = pos[first + i0 + k * SEL_THREADS];
                }
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (i0 + k * SEL_THREADS < n) {
                    const int i = i0 + k * SEL_THREADS;
                    s_key[i] = evict_key(a[k], p[k], e.n_sink, e.recent_from);
                    if (copy && first + i < e.n_keep) {
                        acc_out[first + i] = a[k];
                        pos_out[first + i] = p[k];
                    }
                }
        }
    } else if (copy) {
        for (int i = tid; i < n && first + i < e.n_keep; i += SEL_THREADS) {
            acc_out[first + i] = acc[first + i];
            pos_out[first + i] = pos[first + i];
        }
    }
    __syncthreads();
    auto key = [&](int i) { return HELD ? s_key[i] : fresh(i); };
    const Threshold<unsigned> th = select_threshold<CLN, 32, unsigned>(sel, key, n, e.n_keep);
    // rows to fill (below n_keep, not kept) come before rows to move (at or above n_keep, kept), as many of each
    int32_t* to = CLN == 1 && fused ? s_to : e.to + (int64_t)kv * e.max_rows;
    int32_t* from = CLN == 1 && fused ? s_from : e.from + (int64_t)kv * e.max_rows;
    int moves = 0;
    ranked<CLN>(
        sel, [&](int i) { return (first + i < e.n_keep) != th.in(key(i), i); }, n,
        [&](unsigned all) {
            moves = (int)(all / 2);
            if (rank == 0 && tid == 0) e.n_moves[kv] = moves;
        },
        [&](int i, unsigned r) {
            if (first + i < e.n_keep) to[r] = first + i;
            else from[r - moves] = first + i;
        });
    if constexpr (CLN == 1) {
        if (fused) {
            __syncthreads();
            for (int i = tid >> 5; i < moves; i += SEL_WARPS) move_rows<1>(e, kv, s_to, s_from, i, i + 1);
        }
    } else {
        cg::this_cluster().sync();                     // no CTA leaves while its counts may be read
    }
}
// EV_MOVES rows a warp: 61440 rows of 256 bytes each in K and V (16 heads) 35.5 us for the whole eviction with 2, 39.2 with 1, 39.3
// with 4, 43.5 with 8; 240 rows 8.2, 8.0, 8.7, 9.7.
__global__ void __launch_bounds__(256) k_evict_move(const CacheEvict e) {
    pdl_enter();
    const int kv = blockIdx.y, i = (blockIdx.x * 8 + (threadIdx.x >> 5)) * EV_MOVES, n = e.n_moves[kv];
    if (i >= n) return;
    move_rows<EV_MOVES>(e, kv, e.to + (int64_t)kv * e.max_rows, e.from + (int64_t)kv * e.max_rows, i, min(i + EV_MOVES, n));
}

// ---- bounds of complete blocks: 16 bytes of a row per thread, as many (block, KV head) per CTA as its threads take ----
// Bound by DRAM and the CTAs' start: 120000 rows x 4 heads of 128, 123 MB in 23.2 us, 5.3 TB/s; 32767 rows 8.6 us, 3.9 TB/s.
// A CTA for each block of 16 rows took 18 us for the latter, now 8.8. Sixteen rows a thread leave too few loads under way for
// keys that are in L2 (2 us more); CTAs that take one block after another need the next one's loads in registers (spills).
__device__ __forceinline__ __half2 min2(__half2 a, __half2 b) { return __hmin2(a, b); }
__device__ __forceinline__ __half2 max2(__half2 a, __half2 b) { return __hmax2(a, b); }
__device__ __forceinline__ __nv_bfloat162 min2(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmin2(a, b); }
__device__ __forceinline__ __nv_bfloat162 max2(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmax2(a, b); }

constexpr int BN_THREADS = 128, BN_ROWS = 8;
template <typename T2>
__global__ void __launch_bounds__(BN_THREADS) k_cache_bounds(const uint16_t* __restrict__ kc, int64_t rs, int64_t hs,
                                                             int hd, int max_rows, int shift, int row0, int row1,
                                                             const int32_t* __restrict__ row1_dev,
                                                             uint16_t* __restrict__ bounds) {
    pdl_enter();
    __shared__ uint4 s_lo[BN_THREADS], s_hi[BN_THREADS];
    if (row1_dev) {
        row0 = max(0, *row1_dev);
        row1 = min(row0 + 1, max_rows);
    }
    const int kv = blockIdx.y, block = 1 << shift, b0 = (row0 >> shift) + blockIdx.x * blockDim.z;
    const int b = b0 + threadIdx.z, last = row1 >> shift;
    if (b0 >= last) return;
    const int cols = blockDim.x, groups = blockDim.y, c = threadIdx.x, gi = threadIdx.y;
    const int tid = (threadIdx.z * groups + gi) * cols + c;
    const bool live = b < last;
    union V {
        uint4 u;
        T2 h[4];
    };
    V lo, hi;
    if (live) {
        const uint16_t* base = kc + (int64_t)b * block * rs + (int64_t)kv * hs + 8 * c;
        lo.u = hi.u = *reinterpret_cast<const uint4*>(base + gi * rs);
        for (int r = gi + groups; r < block; r += 8 * groups) {      // eight rows' loads in flight
            V x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                x[k].u = r + k * groups < block ? *reinterpret_cast<const uint4*>(base + (r + k * groups) * rs) : lo.u;
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    lo.h[i] = min2(lo.h[i], x[k].h[i]);
                    hi.h[i] = max2(hi.h[i], x[k].h[i]);
                }
        }
        s_lo[tid] = lo.u;
        s_hi[tid] = hi.u;
    }
    __syncthreads();
    if (live && gi == 0) {
        for (int g = 1; g < groups; ++g) {
            V x, y;
            x.u = s_lo[tid + g * cols];
            y.u = s_hi[tid + g * cols];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                lo.h[i] = min2(lo.h[i], x.h[i]);
                hi.h[i] = max2(hi.h[i], y.h[i]);
            }
        }
        uint16_t* out = bounds + ((int64_t)kv * (max_rows >> shift) + b) * 2 * hd + 8 * c;
        *reinterpret_cast<uint4*>(out) = lo.u;
        *reinterpret_cast<uint4*>(out + hd) = hi.u;
    }
}

// ---- scores: u[kv][row][b - first] = sum_d max(q_d kmin_d, q_d kmax_d) = sum_d q+_d kmax_d + q-_d kmin_d ----
// In 64 bits, because the scores decide which rows are read: products of 24 and 11 (or 8) bits are exact, and
// sums differ from the true ones in the 16th digit. The positive and the negative part of q are two products by f64
// matrix instructions (m8n8k4: eight query rows, four dims, eight blocks); a multiply-add with a select of the bound does
// half the arithmetic, but spends the issue slots on selects and on reading q again for every product. A warp takes eight
// query rows and eight blocks of a CTA's 32, 128 dims; more dims take four more warps, whose sums are added. The bounds come
// from memory as a lane needs them, and which dim a step's k-th place holds is free as long as both operands
// agree. u_top receives the rows' maxima over the 32 blocks.
// Bound by the f64 pipe (64 multiply-adds a clock and SM, 5.7 us for 1557 blocks of 64 query rows and 4 KV heads of 128) and
// by the bounds' way from L2, once for every eight query rows: 12.7 us there; with multiply-adds and selects 20.4. CTAs
// that keep q for further blocks hold it as f64 in 64 registers, and their loads wait for one another: 16.5.
// A bound's f64 is made from its bits by shifting them under the exponent field (two or three integer instructions), which
// is its value times 2^-1008 (f16) or 2^-896 (bf16), subnormals included; q is scaled up to make up for all but
// 2^-128 of it, which cancels in nothing but the comparison of scores. Infinite bounds thereby count as one step above the
// largest finite value.
struct Candidates {
    int n_past, nb, first, last;
};
__device__ __forceinline__ Candidates candidates(const CacheSelect& c) {
    const int past = c.n_past_dev ? max(0, min(*c.n_past_dev, c.max_rows - c.m)) : c.n_past;
    const int nb = (past + c.block - 1) >> c.block_shift, first = min(c.n_sink, nb);
    return {past, nb, first, max(first, nb - min(nb, c.n_local))};
}
template <typename KT> struct Shift;     // of a packed value's bits under f64's exponent field; the scale of q
template <> struct Shift<__half> {
    static constexpr int N = 6;
    static constexpr int MASK = (int)0x81FFFC00u, Q_EXP = 1008 - 128;
};
template <> struct Shift<__nv_bfloat16> {
    static constexpr int N = 3;
    static constexpr int MASK = (int)0x8FFFE000u, Q_EXP = 896 - 128;
};
// high words of the f64s of a packed pair
template <typename KT> __device__ __forceinline__ int2 high_words(uint32_t w) {
    return make_int2(((int)(w << 16) >> Shift<KT>::N) & Shift<KT>::MASK, ((int)w >> Shift<KT>::N) & Shift<KT>::MASK);
}

constexpr int SC_ROWS = 8, SC_TOP = 32;  // query rows and blocks of a CTA; an entry of u_top has as many blocks
constexpr int SC_WARPS = SC_TOP / 8;     // warps of 128 dims
__device__ __forceinline__ void mma884(double* c, double a, double b) {
    asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0,%1}, {%2}, {%3}, {%0,%1};"
                 : "+d"(c[0]), "+d"(c[1]) : "d"(a), "d"(b));
}
template <typename KT, int PARTS>
__global__ void __launch_bounds__(32 * SC_WARPS * PARTS, PARTS == 1 ? 5 : 2) k_block_score(const CacheSelect c, int nb_cap) {
    pdl_enter();
    __shared__ double s_top[SC_WARPS][SC_ROWS];
    __shared__ double2 s_sum[PARTS == 1 ? 1 : SC_WARPS * 32];
    const Candidates cd = candidates(c);
    const int n_cand = cd.last - cd.first, b0 = blockIdx.x * SC_TOP, kv = blockIdx.y, row0 = blockIdx.z * SC_ROWS;
    if (n_cand <= c.n_sel || b0 >= n_cand) return;     // every candidate is taken: no scores needed
    const int R = c.m * c.g, tid = threadIdx.x, lane = tid & 31, warp = (tid >> 5) % SC_WARPS, part = tid / (32 * SC_WARPS);
    // lane = (row of q, place k) and (block, place k) of the operands, (row, two blocks) of the sums
    const int j = lane & 3, i8 = lane >> 2, row = row0 + i8, c8 = c.hd / 8, t = row / c.g;
    const float* q = c.q + (row < R ? t * c.q_ts + (kv * c.g + row - t * c.g) * c.q_hs : 0);
    const bool wide = (reinterpret_cast<uintptr_t>(q) & 15) == 0;
    const uint4* src = reinterpret_cast<const uint4*>(c.bounds) +
                       ((int64_t)kv * nb_cap + cd.first + min(b0 + 8 * warp + i8, n_cand - 1)) * 2 * c8;
    uint4 lo[4], hi[4];
    float x[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {                      // this lane's pieces of eight dims: j, j + 4, .. of the warp's 128
        const int p = part * 16 + 4 * i + j;
        lo[i] = hi[i] = make_uint4(0, 0, 0, 0);
        if (p < c8) {
            lo[i] = src[p];
            hi[i] = src[c8 + p];
        }
        const bool there = row < R && p < c8;
        if (wide) {
            const float4 a = there ? *reinterpret_cast<const float4*>(q + 8 * p) : make_float4(0.f, 0.f, 0.f, 0.f);
            const float4 b = there ? *reinterpret_cast<const float4*>(q + 8 * p + 4) : make_float4(0.f, 0.f, 0.f, 0.f);
            x[i][0] = a.x, x[i][1] = a.y, x[i][2] = a.z, x[i][3] = a.w;
            x[i][4] = b.x, x[i][5] = b.y, x[i][6] = b.z, x[i][7] = b.w;
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) x[i][k] = there ? q[8 * p + k] : 0.f;
        }
    }
    const double up = __hiloint2double((1023 + Shift<KT>::Q_EXP) << 20, 0);
    double pos[2] = {0.0, 0.0}, neg[2] = {0.0, 0.0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t lw[4] = {lo[i].x, lo[i].y, lo[i].z, lo[i].w}, hw[4] = {hi[i].x, hi[i].y, hi[i].z, hi[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int2 l = high_words<KT>(lw[k]), h = high_words<KT>(hw[k]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                // the part of q of one sign: the high word of the other's becomes 0, and what the low word leaves is below
                // 2^-1022, so that its products are 0
                const double d = (double)x[i][2 * k + e] * up;
                const int dh = __double2hiint(d), dl = __double2loint(d);
                mma884(pos, __hiloint2double(max(dh, 0), dl), __hiloint2double(e ? h.y : h.x, 0));
                mma884(neg, __hiloint2double(min(dh, 0), dl), __hiloint2double(e ? l.y : l.x, 0));
            }
        }
    }
    double sum[2] = {pos[0] + neg[0], pos[1] + neg[1]}, top = -INFINITY;
    if constexpr (PARTS > 1) {
        if (part) s_sum[warp * 32 + lane] = make_double2(sum[0], sum[1]);
        __syncthreads();
        if (!part) {
            sum[0] += s_sum[warp * 32 + lane].x;
            sum[1] += s_sum[warp * 32 + lane].y;
        }
    }
    if (!part) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int b = b0 + 8 * warp + 2 * j + e;
            if (row < R && b < n_cand) {
                c.u[((int64_t)kv * R + row) * nb_cap + b] = sum[e];
                top = fmax(top, sum[e]);
            }
        }
        top = fmax(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmax(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (j == 0) s_top[warp][i8] = top;
    }
    __syncthreads();
    if (tid < SC_ROWS && row0 + tid < R) {
        top = s_top[0][tid];
#pragma unroll
        for (int w = 1; w < SC_WARPS; ++w) top = fmax(top, s_top[w][tid]);
        c.u_top[((int64_t)kv * R + row0 + tid) * ((nb_cap + SC_TOP - 1) / SC_TOP) + blockIdx.x] = top;
    }
}

// ---- selection: one CTA or cluster per (KV head, token) -------------------------------------------------------
// Key of a score max_h (u_h - top_h) <= 0: the bits of its magnitude, turned over; NaN lowest. Bound by latency: 506 candidates
// of 8 heads 5.7 us (loads 1, maxima 0.7, keys 1.1, threshold 1.9, ranks 1).
constexpr int BS_MAX_G = 64;
// Candidates up to which one CTA chooses, and above which a cluster's eight form the keys for it, if the clusters of all
// problems fit on the GPU at once: BS_ALONE and BS_MORE for each problem, because many clusters start later. Alone against a
// cluster (all of a call, 128 dims): 8 problems 18.9 / 20.7 us for 1089 candidates, 21.3 / 21.5 for 1557, 25.1 / 23.5 for 3120;
// 16 problems 22.5 / 25.3 for 1557, 30.4 / 30.6 for 3120, 46.7 / 42.1 for 6245.
constexpr int BS_ONE = 8192, BS_ALONE = 1024, BS_MORE = 128;
__device__ __forceinline__ unsigned long long score_key(double v) {
    return v != v ? 0ull : 0x7FFFFFFFFFFFFFFFull - (unsigned long long)__double_as_longlong(fabs(v));
}
// CLN > 1 and GATHER: the cluster's CTAs form the keys, the first of them chooses; without GATHER all choose together.
template <int CLN, bool GATHER>
__global__ void __launch_bounds__(SEL_THREADS) k_block_choose(const CacheSelect c, int nb_cap) {
    pdl_enter();
    extern __shared__ unsigned long long s_keys[];
    __shared__ Select ss;
    __shared__ double s_top[BS_MAX_G];
    const int kv = blockIdx.y, t = blockIdx.z, rank = CLN == 1 ? 0 : blockIdx.x, tid = threadIdx.x;
    const int lane = tid & 31, warp = tid >> 5;
    const Candidates cd = candidates(c);
    const int n_cand = cd.last - cd.first, n_take = min(n_cand, c.n_sel);
    const int prob = kv * c.m + t;
    int32_t* list = c.list + (int64_t)prob * c.list_cap;
    int32_t* sel = c.sel_out ? c.sel_out + ((int64_t)t * c.n_kv + kv) * c.n_sel : nullptr;
    // the blocks that are always attended, and the tail of sel
    const int gtid = rank * SEL_THREADS + tid, gn = CLN * SEL_THREADS;
    for (int i = gtid; i < cd.first; i += gn) list[i] = i;
    for (int i = gtid; i < cd.nb - cd.last; i += gn) list[cd.first + n_take + i] = cd.last + i;
    if (sel)
        for (int i = n_take + gtid; i < c.n_sel; i += gn) sel[i] = -1;
    if (gtid == 0) c.list_n[prob] = cd.first + n_take + cd.nb - cd.last;
    if (n_take == n_cand) {                            // uniform over the cluster: nothing to choose
        for (int i = gtid; i < n_cand; i += gn) {
            list[cd.first + i] = cd.first + i;
            if (sel) sel[i] = cd.first + i;
        }
        return;
    }
    if (n_take == 0) return;
    int i0 = (int)((int64_t)n_cand * rank / CLN), n = (int)((int64_t)n_cand * (rank + 1) / CLN) - i0;
    const int64_t row0 = ((int64_t)kv * c.m + t) * c.g;
    // four blocks by eight heads of loads in flight per thread, the first of them while the maxima are formed
    const double* u = c.u + row0 * nb_cap + i0;
    double v[4][8];
    auto load = [&](int i, int h0) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int h = 0; h < 8; ++h)
                v[k][h] = i + k * SEL_THREADS < n && h0 + h < c.g ? u[(h0 + h) * (int64_t)nb_cap + i + k * SEL_THREADS] : 0.0;
    };
    load(tid, 0);
    const int tops = (n_cand + SC_TOP - 1) / SC_TOP, top_cap = (nb_cap + SC_TOP - 1) / SC_TOP;
    for (int h = warp; h < c.g; h += SEL_WARPS) {
        const double* p = c.u_top + (row0 + h) * top_cap;
        double mx = -INFINITY;
        for (int i = lane; i < tops; i += 8 * 32) {
            double w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) w[k] = i + 32 * k < tops ? p[i + 32 * k] : -INFINITY;
#pragma unroll
            for (int k = 0; k < 8; ++k) mx = fmax(mx, w[k]);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmax(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        if (lane == 0) s_top[h] = mx;
    }
    unsigned long long* keys = s_keys;
    if constexpr (GATHER) {
        cg::this_cluster().sync();                     // the first CTA runs, its memory can be written
        keys = cg::this_cluster().map_shared_rank(s_keys, 0) + i0;
    } else {
        __syncthreads();
    }
    for (int i = tid; i < n; i += 4 * SEL_THREADS) {
        double best[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) best[k] = -INFINITY;
        for (int h0 = 0; h0 < c.g; h0 += 8) {
            if (i != tid || h0) load(i, h0);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int h = 0; h < 8; ++h)
                    if (h0 + h < c.g) best[k] = fmax(best[k], v[k][h] - s_top[h0 + h]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k * SEL_THREADS < n) keys[i + k * SEL_THREADS] = score_key(best[k]);
    }
    constexpr int SEL = GATHER ? 1 : CLN;              // CTAs that choose
    if constexpr (GATHER) {
        cg::this_cluster().sync();
        if (rank) return;
        i0 = 0;
        n = n_cand;
    } else {
        __syncthreads();
    }
    auto key = [&](int i) { return s_keys[i]; };
    const Threshold<unsigned long long> th = select_threshold<SEL, 63, unsigned long long>(ss, key, n, n_take);
    ranked<SEL>(
        ss, [&](int i) { return th.in(s_keys[i], i); }, n, [](unsigned) {},
        [&](int i, unsigned r) {
            const int b = cd.first + i0 + i;
            list[cd.first + r] = b;
            if (sel) sel[r] = b;
        });
    if constexpr (SEL > 1) cg::this_cluster().sync();  // no CTA leaves while its counts may be read
}

// ---- the accepted path of a tree: thread = a 16-byte column of the K or V rows of a KV head. Rows ascend and
// row0 + i <= row0 + path[i], so a batch that is read before it is written overwrites no later source ----
__global__ void __launch_bounds__(32) k_cache_take(char* kc, char* vc, int64_t rs, int64_t hs, int hd, int row0,
                                                   const TakePath path, int n) {
    pdl_enter();
    const int c = threadIdx.x;
    if (c >= hd / 8) return;
    char* base = (blockIdx.y ? vc : kc) + (int64_t)blockIdx.x * hs * 2 + c * 16;
    for (int i0 = 0; i0 < n; i0 += 8) {
        uint4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i0 + i < n) v[i] = *reinterpret_cast<const uint4*>(base + (int64_t)(row0 + path.row[i0 + i]) * rs * 2);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i0 + i < n) *reinterpret_cast<uint4*>(base + (int64_t)(row0 + i0 + i) * rs * 2) = v[i];
    }
}

}  // namespace

cudaError_t launch_cache_evict(const CacheEvict& e, cudaStream_t s) {
    const int most = e.n_keep < e.n_rows - e.n_keep ? e.n_keep : e.n_rows - e.n_keep;      // moves
    if (e.n_rows <= EV_SINGLE) {
        const bool fused = most <= EV_FUSED;
        static SmemLimit limit;
        cudaError_t rc = limit.raise((const void*)k_evict_choose<1, true>, EV_SINGLE * 4);
        if (rc != cudaSuccess) return rc;
        rc = launch_pdl(k_evict_choose<1, true>, dim3(1, e.n_kv), SEL_THREADS, (size_t)e.n_rows * 4, s, e, fused);
        if (rc != cudaSuccess || fused) return rc;
    } else {
        static SmemLimit limit;
        cudaError_t rc = limit.raise((const void*)k_evict_choose<CL, true>, EV_KEYS * 4);
        if (rc != cudaSuccess) return rc;
        const int n = (e.n_rows + CL - 1) / CL;
        rc = n <= EV_KEYS ? launch_pdl_cluster(k_evict_choose<CL, true>, CL, dim3(CL, e.n_kv), SEL_THREADS, (size_t)n * 4, s, e, false)
                          : launch_pdl_cluster(k_evict_choose<CL, false>, CL, dim3(CL, e.n_kv), SEL_THREADS, 0, s, e, false);
        if (rc != cudaSuccess) return rc;
    }
    if (most == 0) return cudaSuccess;
    return launch_pdl(k_evict_move, dim3((most + 8 * EV_MOVES - 1) / (8 * EV_MOVES), e.n_kv), 256, 0, s, e);
}

cudaError_t launch_cache_bounds(const void* kc, int64_t rs, int64_t hs, bool bf16, int n_kv, int hd, int max_rows,
                                int block, int row0, int row1, const int32_t* row1_dev, void* bounds, cudaStream_t s) {
    const int blocks = row1_dev ? 1 : row1 / block - row0 / block;
    if (blocks <= 0) return cudaSuccess;
    // threads: 16 bytes of a row, rows of a block (BN_ROWS each where there are threads enough), blocks
    const int cols = hd / 8, want = block / BN_ROWS, most = BN_THREADS / cols, groups = want < most ? want : most;
    const int at_once = BN_THREADS / (groups * cols), shift = __builtin_ctz(block);
    const dim3 grid((blocks + at_once - 1) / at_once, n_kv), threads(cols, groups, at_once);
    if (bf16)
        return launch_pdl(k_cache_bounds<__nv_bfloat162>, grid, threads, 0, s, (const uint16_t*)kc, rs, hs, hd,
                          max_rows, shift, row0, row1, row1_dev, (uint16_t*)bounds);
    return launch_pdl(k_cache_bounds<__half2>, grid, threads, 0, s, (const uint16_t*)kc, rs, hs, hd, max_rows, shift,
                      row0, row1, row1_dev, (uint16_t*)bounds);
}

ChooseForm choose_form(int n_cand, int problems) {
    if (n_cand > BS_ONE) return CHOOSE_CLUSTER;
    return n_cand <= BS_ALONE + BS_MORE * (int64_t)problems || problems * (int64_t)CL > KV_SMS ? CHOOSE_ONE : CHOOSE_GATHER;
}

cudaError_t launch_cache_select(const CacheSelect& asked, cudaStream_t s) {
    CacheSelect c = asked;
    c.block_shift = __builtin_ctz(c.block);
    const int nb_cap = c.max_rows / c.block;
    const int past_most = c.n_past_dev ? c.max_rows - c.m : c.n_past;
    int n_cand = (past_most + c.block - 1) / c.block - c.n_sink - c.n_local;
    if (n_cand < 0) n_cand = 0;
    cudaError_t e;
    if (n_cand > c.n_sel && c.n_sel > 0) {
        const int parts = c.hd <= 128 ? 1 : 2;
        const dim3 grid((n_cand + SC_TOP - 1) / SC_TOP, c.n_kv, (c.m * c.g + SC_ROWS - 1) / SC_ROWS);
        auto fn = c.bf16 ? (parts == 1 ? k_block_score<__nv_bfloat16, 1> : k_block_score<__nv_bfloat16, 2>)
                         : (parts == 1 ? k_block_score<__half, 1> : k_block_score<__half, 2>);
        e = launch_pdl(fn, grid, 32 * SC_WARPS * parts, 0, s, c, nb_cap);
        if (e != cudaSuccess) return e;
    }
    const ChooseForm form = choose_form(n_cand, c.n_kv * c.m);
    if (form == CHOOSE_ONE) {
        static SmemLimit limit;
        e = limit.raise((const void*)k_block_choose<1, false>, BS_ONE * 8);
        if (e != cudaSuccess) return e;
        return launch_pdl(k_block_choose<1, false>, dim3(1, c.n_kv, c.m), SEL_THREADS, (size_t)n_cand * 8, s, c, nb_cap);
    }
    const dim3 grid(CL, c.n_kv, c.m);
    if (form == CHOOSE_GATHER) {
        static SmemLimit limit;
        e = limit.raise((const void*)k_block_choose<CL, true>, BS_ONE * 8);
        if (e != cudaSuccess) return e;
        return launch_pdl_cluster(k_block_choose<CL, true>, CL, grid, SEL_THREADS, (size_t)n_cand * 8, s, c, nb_cap);
    }
    static SmemLimit limit;
    e = limit.raise((const void*)k_block_choose<CL, false>, 128 * 1024);
    if (e != cudaSuccess) return e;
    return launch_pdl_cluster(k_block_choose<CL, false>, CL, grid, SEL_THREADS, (size_t)((n_cand + CL - 1) / CL) * 8, s, c, nb_cap);
}

cudaError_t launch_cache_take(void* kc, void* vc, int64_t rs, int64_t hs, int n_kv, int hd, int row0,
                              const TakePath& path, int n, cudaStream_t s) {
    return launch_pdl(k_cache_take, dim3(n_kv, 2), 32, 0, s, (char*)kc, (char*)vc, rs, hs, hd, row0, path, n);
}

}  // namespace hoard
