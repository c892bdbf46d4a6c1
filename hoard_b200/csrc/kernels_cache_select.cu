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
constexpr int SEL_THREADS = 1024, SEL_WARPS = SEL_THREADS / 32;
constexpr int DIGIT = 11, BINS = 1 << DIGIT;
static_assert(BINS == 2 * SEL_THREADS, "two bins per thread");

// exclusive prefix sum over the CTA; total receives the sum
__device__ __forceinline__ unsigned long long block_scan(unsigned long long v, unsigned long long* s_warp,
                                                         unsigned long long& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto scan32 = [&](unsigned long long x) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        return x;
    };
    const unsigned long long x = scan32(v);
    __syncthreads();                     // s_warp may still be read from an earlier scan
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    const unsigned long long w = scan32(s_warp[lane]);
    total = __shfl_sync(0xffffffffu, w, SEL_WARPS - 1);
    const unsigned long long before = __shfl_sync(0xffffffffu, w, warp ? warp - 1 : 0);
    return (warp ? before : 0) + x - v;
}

// Shared state of a selection
struct Select {
    unsigned hist[2][BINS];
    unsigned long long warp[SEL_WARPS];
    unsigned long long ex[2];            // this CTA's totals, for prefixes over the cluster
    unsigned bin, in_bin, above;
};

// exclusive prefix over the cluster's CTAs of `total` (a slot is used once, so nothing overwrites it)
template <int CLN>
__device__ __forceinline__ unsigned long long cluster_before(Select& s, int slot, unsigned long long total) {
    if constexpr (CLN == 1) return 0;
    cg::cluster_group cl = cg::this_cluster();
    if (threadIdx.x == 0) s.ex[slot] = total;
    cl.sync();
    unsigned long long v[CLN], before = 0;
#pragma unroll
    for (int r = 0; r < CLN; ++r) v[r] = *cl.map_shared_rank(&s.ex[slot], r);
#pragma unroll
    for (int r = 0; r < CLN; ++r)
        if (r < (int)cl.block_rank()) before += v[r];
    return before;
}

// The `need` largest of the keys: afterwards a key is in if (key >> shift) > prefix, and of those with
// (key >> shift) == prefix the first `eq_need` in index order are. key(i): this CTA's i-th key.
struct Threshold {
    unsigned long long prefix;
    int shift, eq_need;
};
template <int CLN, int BITS, typename Key>
__device__ __forceinline__ Threshold select_threshold(Select& s, Key key, int n_local, int need) {
    unsigned long long prefix = 0;
    int shift = BITS, buf = 0;
    for (bool first = true;; first = false) {
        const int width = min(DIGIT, shift);
        shift -= width;
        unsigned* hist = s.hist[buf];
        hist[threadIdx.x] = 0;
        hist[threadIdx.x + SEL_THREADS] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n_local; i += SEL_THREADS) {
            const unsigned long long k = key(i);
            const unsigned d = (unsigned)(k >> shift) & ((1u << width) - 1);
            if (first) {                 // exponents: few bins, so a warp's equal ones are added at once
                const unsigned act = __activemask(), same = __match_any_sync(act, d);
                if ((int)(threadIdx.x & 31) == __ffs(same) - 1) atomicAdd(&hist[d], (unsigned)__popc(same));
            } else if ((k >> (shift + width)) == prefix) {
                atomicAdd(&hist[d], 1u);
            }
        }
        // thread i: bins BINS - 1 - 2i and BINS - 2 - 2i, so that the scan runs from the top
        unsigned hi = 0, lo = 0;
        if constexpr (CLN == 1) {
            __syncthreads();
            const uint2 h = *reinterpret_cast<const uint2*>(hist + BINS - 2 - 2 * threadIdx.x);
            lo = h.x;
            hi = h.y;
        } else {
            cg::cluster_group cl = cg::this_cluster();
            cl.sync();
            uint2 h[CLN];
#pragma unroll
            for (int r = 0; r < CLN; ++r)
                h[r] = *reinterpret_cast<const uint2*>(cl.map_shared_rank(hist, r) + BINS - 2 - 2 * threadIdx.x);
#pragma unroll
            for (int r = 0; r < CLN; ++r) {
                lo += h[r].x;
                hi += h[r].y;
            }
        }
        unsigned long long total;
        const unsigned above = (unsigned)block_scan(hi + lo, s.warp, total), n = (unsigned)need;
        if (above < n && above + hi >= n) {
            s.bin = BINS - 1 - 2 * threadIdx.x;
            s.in_bin = hi;
            s.above = above;
        } else if (above + hi < n && above + hi + lo >= n) {
            s.bin = BINS - 2 - 2 * threadIdx.x;
            s.in_bin = lo;
            s.above = above + hi;
        }
        __syncthreads();
        prefix = prefix << width | s.bin;
        need -= (int)s.above;
        const bool done = shift == 0 || s.in_bin == (unsigned)need;
        __syncthreads();                 // read before the next pass writes
        if (done) return {prefix, shift, need};
        buf ^= 1;                        // the cluster's other CTAs may still read this pass's counts
    }
}

// ---- eviction -------------------------------------------------------------------------------------------------
// Key of a row: protected rows above everything; weights in order; NaN below everything. -0 equals +0.
constexpr int EV_KEYS = 40960;           // keys that a CTA holds in shared memory (160 KiB)
constexpr int EV_SINGLE = 8192;          // rows up to which one CTA chooses alone
constexpr int EV_FUSED = 1024;           // moves up to which that CTA makes them itself
__device__ __forceinline__ unsigned evict_key(float acc, int pos, int n_sink, int recent_from) {
    if (pos < n_sink || pos >= recent_from) return 0xFFFFFFFFu;
    if (acc != acc) return 0u;
    const unsigned b = __float_as_uint(acc + 0.f);
    return b >> 31 ? ~b : b | 0x80000000u;
}
// Moves i0, i0 + 1, .. of N: K and V rows by 16-byte pieces, all N loads before the first store. Rows read are at or
// above n_keep, rows written below it.
template <int N>
__device__ __forceinline__ void move_rows(const CacheEvict& e, int kv, const int32_t* to, const int32_t* from, int i0,
                                          int n) {
    const int lane = threadIdx.x & 31, c16 = e.hd / 8;
    const int64_t hb = (int64_t)kv * e.max_rows;
    int t[N], f[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        t[k] = i0 + k < n ? to[i0 + k] : -1;
        f[k] = i0 + k < n ? from[i0 + k] : 0;
    }
    for (int p = lane; p < 2 * c16; p += 32) {
        char* c = static_cast<char*>(p < c16 ? e.kc : e.vc) + (int64_t)kv * e.hs * 2 + (p < c16 ? p : p - c16) * 16;
        uint4 v[N];
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (t[k] >= 0) v[k] = *reinterpret_cast<const uint4*>(c + (int64_t)f[k] * e.rs * 2);
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (t[k] >= 0) *reinterpret_cast<uint4*>(c + (int64_t)t[k] * e.rs * 2) = v[k];
    }
    if (lane < N && i0 + lane < n) {
        const int tt = to[i0 + lane], ff = from[i0 + lane];
        e.acc_out[hb + tt] = e.acc[hb + ff];
        e.pos_out[hb + tt] = e.pos[hb + ff];
    }
}
// Grid (CLN, n_kv). Lists the rows to fill and the rows to move (ascending both), writes acc_out / pos_out of the
// kept rows that stay where they are, and makes the moves itself where there are few (to, from then sit in
// shared memory).
template <int CLN>
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
    const bool held = CLN == 1 || n <= EV_KEYS;
    auto fresh = [&](int i) { return evict_key(acc[first + i], pos[first + i], e.n_sink, e.recent_from); };
    if (held) {
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
                if (i0 + k * SEL_THREADS < n) s_key[i0 + k * SEL_THREADS] = evict_key(a[k], p[k], e.n_sink, e.recent_from);
        }
    }
    __syncthreads();
    auto key = [&](int i) { return held ? s_key[i] : fresh(i); };
    const Threshold th = select_threshold<CLN, 32>(sel, key, n, e.n_keep);

    // a thread owns a run of rows (odd length: the runs' first words fall in different banks)
    const int len = (n + SEL_THREADS - 1) / SEL_THREADS | 1, i0 = min(n, tid * len), i1 = min(n, i0 + len);
    unsigned long long eq = 0, total;
    for (int i = i0; i < i1; ++i) eq += (unsigned long long)(key(i) >> th.shift) == th.prefix;
    unsigned long long eq_rank = block_scan(eq, sel.warp, total);
    eq_rank += cluster_before<CLN>(sel, 0, total);
    const unsigned long long eq_rank0 = eq_rank;
    auto kept = [&](int i) {
        const unsigned long long k = key(i) >> th.shift;
        return k > th.prefix || (k == th.prefix && eq_rank++ < (unsigned long long)th.eq_need);
    };
    unsigned long long counts = 0;                     // low half: rows to fill, high half: rows to move
    for (int i = i0; i < i1; ++i) {
        const bool k = kept(i);
        if (first + i < e.n_keep) counts += !k;
        else if (k) counts += 1ull << 32;
    }
    unsigned long long at = block_scan(counts, sel.warp, total);
    const unsigned long long before = cluster_before<CLN>(sel, 1, total);
    at += before;
    if (rank == CLN - 1 && tid == 0) e.n_moves[kv] = (int)((before + total) & 0xFFFFFFFFu);
    eq_rank = eq_rank0;
    int32_t* to = CLN == 1 && fused ? s_to : e.to + (int64_t)kv * e.max_rows;
    int32_t* from = CLN == 1 && fused ? s_from : e.from + (int64_t)kv * e.max_rows;
    int n_to = (int)(at & 0xFFFFFFFFu), n_from = (int)(at >> 32);
    const bool stay = e.acc_out != e.acc || e.pos_out != e.pos;
    for (int i = i0; i < i1; ++i) {
        const bool k = kept(i);
        const int row = first + i;
        if (row < e.n_keep) {
            if (!k) {
                to[n_to++] = row;
            } else if (stay) {
                e.acc_out[(int64_t)kv * e.max_rows + row] = acc[row];
                e.pos_out[(int64_t)kv * e.max_rows + row] = pos[row];
            }
        } else if (k) {
            from[n_from++] = row;
        }
    }
    if constexpr (CLN == 1) {
        if (fused) {
            const int moves = (int)(total & 0xFFFFFFFFu);
            __syncthreads();
            for (int i = (tid >> 5) * 4; i < moves; i += SEL_WARPS * 4) move_rows<4>(e, kv, s_to, s_from, i, moves);
        }
    } else {
        cg::this_cluster().sync();                     // no CTA leaves while its counts may be read
    }
}
__global__ void __launch_bounds__(256) k_evict_move(const CacheEvict e) {
    pdl_enter();
    const int kv = blockIdx.y, i = (blockIdx.x * 8 + (threadIdx.x >> 5)) * 4, n = e.n_moves[kv];
    if (i >= n) return;
    move_rows<4>(e, kv, e.to + (int64_t)kv * e.max_rows, e.from + (int64_t)kv * e.max_rows, i, n);
}

// ---- bounds of complete blocks: one CTA per (block, KV head) --------------------------------------------------
__device__ __forceinline__ __half2 min2(__half2 a, __half2 b) { return __hmin2(a, b); }
__device__ __forceinline__ __half2 max2(__half2 a, __half2 b) { return __hmax2(a, b); }
__device__ __forceinline__ __nv_bfloat162 min2(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmin2(a, b); }
__device__ __forceinline__ __nv_bfloat162 max2(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmax2(a, b); }

constexpr int BN_THREADS = 128;
template <typename T2>
__global__ void __launch_bounds__(BN_THREADS) k_cache_bounds(const uint16_t* __restrict__ kc, int64_t rs, int64_t hs,
                                                             int hd, int max_rows, int block, int row0, int row1,
                                                             const int32_t* __restrict__ row1_dev,
                                                             uint16_t* __restrict__ bounds) {
    pdl_enter();
    __shared__ uint4 s_lo[BN_THREADS], s_hi[BN_THREADS];
    if (row1_dev) {
        row0 = max(0, *row1_dev);
        row1 = min(row0 + 1, max_rows);
    }
    const int b = row0 / block + blockIdx.x, kv = blockIdx.y;
    if (b >= row1 / block) return;
    const int cols = hd / 8, groups = BN_THREADS / cols, gi = threadIdx.x / cols, c = threadIdx.x - gi * cols;
    union V {
        uint4 u;
        T2 h[4];
    };
    V lo, hi;
    if (gi < groups) {
        const uint16_t* base = kc + (int64_t)b * block * rs + (int64_t)kv * hs + 8 * c;
        const int r0 = min(gi, block - 1);
        lo.u = hi.u = *reinterpret_cast<const uint4*>(base + r0 * rs);
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
        s_lo[threadIdx.x] = lo.u;
        s_hi[threadIdx.x] = hi.u;
    }
    __syncthreads();
    if (gi == 0) {
        for (int g = 1; g < groups; ++g) {
            V x, y;
            x.u = s_lo[g * cols + c];
            y.u = s_hi[g * cols + c];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                lo.h[i] = min2(lo.h[i], x.h[i]);
                hi.h[i] = max2(hi.h[i], y.h[i]);
            }
        }
        uint16_t* out = bounds + ((int64_t)kv * (max_rows / block) + b) * 2 * hd + 8 * c;
        *reinterpret_cast<uint4*>(out) = lo.u;
        *reinterpret_cast<uint4*>(out + hd) = hi.u;
    }
}

// ---- scores: u[kv][row][b - first] = sum_d max(q_d kmin_d, q_d kmax_d) = sum_d q_d (q_d > 0 ? kmax_d : kmin_d) ----
// In 64 bits, because the scores decide which rows are read: products of 24 and 11 (or 8) bits are exact, and
// sums differ from the true ones in the 16th digit. A CTA takes 32 blocks (one per lane) and eight query rows;
// its warps share out the dims, eight at a time, and their sums are added in warp order. A value is converted once
// for the eight rows, since conversions to f64 run at a quarter of the rate of its multiply-adds. u_top receives
// the rows' maxima over the CTA's blocks.
struct Candidates {
    int n_past, nb, first, last;
};
__device__ __forceinline__ Candidates candidates(const CacheSelect& c) {
    const int past = c.n_past_dev ? max(0, min(*c.n_past_dev, c.max_rows - c.m)) : c.n_past;
    const int nb = (past + c.block - 1) / c.block, first = min(c.n_sink, nb);
    return {past, nb, first, max(first, nb - min(nb, c.n_local))};
}
template <typename KT> __device__ __forceinline__ double2 to_double2(uint32_t w);
template <> __device__ __forceinline__ double2 to_double2<__half>(uint32_t w) {
    return make_double2((double)h2f(w), (double)h2f(w >> 16));
}
template <> __device__ __forceinline__ double2 to_double2<__nv_bfloat16>(uint32_t w) {
    return make_double2((double)__uint_as_float(w << 16), (double)__uint_as_float(w & 0xFFFF0000u));
}

constexpr int SC_THREADS = 256, SC_ROWS = 8, SC_BLOCKS = 32;
constexpr int score_smem(int hd) { return SC_ROWS * hd * 8 + 8 * SC_ROWS * 32 * 8 + SC_BLOCKS * (hd + 4) * 4; }
template <typename KT>
__global__ void __launch_bounds__(SC_THREADS) k_block_score(const CacheSelect c, int nb_cap) {
    pdl_enter();
    extern __shared__ __align__(16) uint8_t s_raw[];
    const Candidates cd = candidates(c);
    const int n_cand = cd.last - cd.first, b0 = blockIdx.x * SC_BLOCKS, kv = blockIdx.y, row0 = blockIdx.z * SC_ROWS;
    if (n_cand <= c.n_sel || b0 >= n_cand) return;     // every candidate is taken: no scores needed
    const int R = c.m * c.g, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    double* sq = reinterpret_cast<double*>(s_raw);                              // [SC_ROWS][hd]
    double* red = sq + SC_ROWS * c.hd;                                          // [8 warps][SC_ROWS][32]
    // [32][hd + 4] words: 16-byte reads of eight lanes fall in eight bank groups
    uint32_t* sb = reinterpret_cast<uint32_t*>(red + 8 * SC_ROWS * 32);
    const int n = min(SC_BLOCKS, n_cand - b0), c4 = c.hd / 4, c8 = c.hd / 8;
    const uint32_t* src = reinterpret_cast<const uint32_t*>(c.bounds) +
                          ((int64_t)kv * (c.max_rows / c.block) + cd.first + b0) * c.hd;      // hd words a block
    for (int b = warp; b < n; b += 8)
        for (int p = lane; p < c4; p += 32) cp_async16(sb + b * (c.hd + 4) + 4 * p, src + b * c.hd + 4 * p);
    cp_async_commit();
    {
        const int row = row0 + warp;                   // a warp converts a query row
        const float* q = c.q + (row / c.g) * c.q_ts + (kv * c.g + row % c.g) * c.q_hs;
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = row < R && k * 32 + lane < c.hd ? q[k * 32 + lane] : 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k * 32 + lane < c.hd) sq[warp * c.hd + k * 32 + lane] = (double)x[k];
    }
    cp_async_wait_all();
    __syncthreads();
    double acc[SC_ROWS];
#pragma unroll
    for (int r = 0; r < SC_ROWS; ++r) acc[r] = 0.0;
    const uint32_t* mine = sb + min(lane, n - 1) * (c.hd + 4);
    for (int p = warp; p < c8; p += 8) {
        const uint4 l4 = *reinterpret_cast<const uint4*>(mine + 4 * p);
        const uint4 h4 = *reinterpret_cast<const uint4*>(mine + c.hd / 2 + 4 * p);
        const uint32_t lw[4] = {l4.x, l4.y, l4.z, l4.w}, hw[4] = {h4.x, h4.y, h4.z, h4.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const double2 lo = to_double2<KT>(lw[k]), hi = to_double2<KT>(hw[k]);
#pragma unroll
            for (int r = 0; r < SC_ROWS; ++r) {
                const double2 q = *reinterpret_cast<const double2*>(sq + r * c.hd + 8 * p + 2 * k);
                acc[r] = fma(q.x, q.x > 0.0 ? hi.x : lo.x, acc[r]);
                acc[r] = fma(q.y, q.y > 0.0 ? hi.y : lo.y, acc[r]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < SC_ROWS; ++r) red[(warp * SC_ROWS + r) * 32 + lane] = acc[r];
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += red[(w * SC_ROWS + warp) * 32 + lane];     // thread = (row, block)
    const int row = row0 + warp;
    if (row >= R) return;
    if (lane < n) c.u[((int64_t)kv * R + row) * nb_cap + b0 + lane] = s;
    double top = lane < n ? s : -INFINITY;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) c.u_top[((int64_t)kv * R + row) * ((nb_cap + SC_BLOCKS - 1) / SC_BLOCKS) + blockIdx.x] = top;
}

// ---- selection: one CTA or cluster per (KV head, token) -------------------------------------------------------
// Key of a score max_h (u_h - top_h) <= 0: the bits of its magnitude, turned over; NaN lowest.
constexpr int BS_MAX_G = 64;
constexpr int BS_SINGLE = 2048;          // candidates up to which one CTA chooses alone
__device__ __forceinline__ unsigned long long score_key(double v) {
    return v != v ? 0ull : 0x7FFFFFFFFFFFFFFFull - (unsigned long long)__double_as_longlong(fabs(v));
}
template <int CLN>
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
    const int i0 = (int)((int64_t)n_cand * rank / CLN), i1 = (int)((int64_t)n_cand * (rank + 1) / CLN), n = i1 - i0;
    const int64_t row0 = ((int64_t)kv * c.m + t) * c.g;
    const int tops = (n_cand + SC_BLOCKS - 1) / SC_BLOCKS, top_cap = (nb_cap + SC_BLOCKS - 1) / SC_BLOCKS;
    for (int h = warp; h < c.g; h += SEL_WARPS) {
        const double* p = c.u_top + (row0 + h) * top_cap;
        double mx = -INFINITY;
        for (int i = lane; i < tops; i += 8 * 32) {
            double v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = i + 32 * k < tops ? p[i + 32 * k] : -INFINITY;
#pragma unroll
            for (int k = 0; k < 8; ++k) mx = fmax(mx, v[k]);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmax(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        if (lane == 0) s_top[h] = mx;
    }
    // this thread's blocks' u are on their way while the maxima are waited for
    const double* u = c.u + row0 * nb_cap + i0;
    double v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = tid < n && k < c.g ? u[k * (int64_t)nb_cap + tid] : 0.0;
    __syncthreads();
    for (int i = tid; i < n; i += SEL_THREADS) {
        double best = -INFINITY;
        for (int h0 = 0; h0 < c.g; h0 += 8) {
            if (i != tid || h0) {
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = h0 + k < c.g ? u[(h0 + k) * (int64_t)nb_cap + i] : 0.0;
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (h0 + k < c.g) best = fmax(best, v[k] - s_top[h0 + k]);
        }
        s_keys[i] = score_key(best);
    }
    __syncthreads();
    auto key = [&](int i) { return s_keys[i]; };
    const Threshold th = select_threshold<CLN, 63>(ss, key, n, n_take);
    const int len = (n + SEL_THREADS - 1) / SEL_THREADS | 1, a0 = min(n, tid * len), a1 = min(n, a0 + len);
    unsigned long long eq = 0, count = 0, total;
    for (int i = a0; i < a1; ++i) eq += (s_keys[i] >> th.shift) == th.prefix;
    unsigned long long eq_rank = block_scan(eq, ss.warp, total);
    eq_rank += cluster_before<CLN>(ss, 0, total);
    const unsigned long long eq_rank0 = eq_rank;
    auto kept = [&](int i) {
        const unsigned long long k = s_keys[i] >> th.shift;
        return k > th.prefix || (k == th.prefix && eq_rank++ < (unsigned long long)th.eq_need);
    };
    for (int i = a0; i < a1; ++i) count += kept(i);
    unsigned long long at = block_scan(count, ss.warp, total);
    at += cluster_before<CLN>(ss, 1, total);
    eq_rank = eq_rank0;
    for (int i = a0; i < a1; ++i)
        if (kept(i)) {
            const int b = cd.first + i0 + i;
            list[cd.first + at] = b;
            if (sel) sel[at] = b;
            ++at;
        }
    if constexpr (CLN > 1) cg::this_cluster().sync();  // no CTA leaves while its counts may be read
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

// a programmatic dependent launch in clusters of `cl` CTAs along x
template <typename... KArgs, typename... Args>
static cudaError_t launch_cluster(void (*kernel)(KArgs...), int cl, dim3 grid, dim3 block, size_t smem, cudaStream_t s,
                                  Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cl;
    at[1].val.clusterDim.y = 1;
    at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

cudaError_t launch_cache_evict(const CacheEvict& e, cudaStream_t s) {
    const int most = e.n_keep < e.n_rows - e.n_keep ? e.n_keep : e.n_rows - e.n_keep;      // moves
    if (e.n_rows <= EV_SINGLE) {
        const bool fused = most <= EV_FUSED;
        const cudaError_t rc = launch_pdl(k_evict_choose<1>, dim3(1, e.n_kv), SEL_THREADS, (size_t)e.n_rows * 4, s, e, fused);
        if (rc != cudaSuccess || fused) return rc;
    } else {
        static SmemLimit limit;
        cudaError_t rc = limit.raise((const void*)k_evict_choose<CL>, EV_KEYS * 4);
        if (rc != cudaSuccess) return rc;
        const int n = (e.n_rows + CL - 1) / CL;
        rc = launch_cluster(k_evict_choose<CL>, CL, dim3(CL, e.n_kv), SEL_THREADS, n <= EV_KEYS ? (size_t)n * 4 : 0, s, e,
                            false);
        if (rc != cudaSuccess) return rc;
    }
    if (most == 0) return cudaSuccess;
    return launch_pdl(k_evict_move, dim3((most + 31) / 32, e.n_kv), 256, 0, s, e);
}

cudaError_t launch_cache_bounds(const void* kc, int64_t rs, int64_t hs, bool bf16, int n_kv, int hd, int max_rows,
                                int block, int row0, int row1, const int32_t* row1_dev, void* bounds, cudaStream_t s) {
    const int blocks = row1_dev ? 1 : row1 / block - row0 / block;
    if (blocks <= 0) return cudaSuccess;
    const dim3 grid(blocks, n_kv);
    if (bf16)
        return launch_pdl(k_cache_bounds<__nv_bfloat162>, grid, BN_THREADS, 0, s, (const uint16_t*)kc, rs, hs, hd,
                          max_rows, block, row0, row1, row1_dev, (uint16_t*)bounds);
    return launch_pdl(k_cache_bounds<__half2>, grid, BN_THREADS, 0, s, (const uint16_t*)kc, rs, hs, hd, max_rows, block,
                      row0, row1, row1_dev, (uint16_t*)bounds);
}

cudaError_t launch_cache_select(const CacheSelect& c, cudaStream_t s) {
    const int nb_cap = c.max_rows / c.block;
    const int past_most = c.n_past_dev ? c.max_rows - c.m : c.n_past;
    int n_cand = (past_most + c.block - 1) / c.block - c.n_sink - c.n_local;
    if (n_cand < 0) n_cand = 0;
    cudaError_t e;
    if (n_cand > c.n_sel && c.n_sel > 0) {
        const dim3 grid((n_cand + SC_BLOCKS - 1) / SC_BLOCKS, c.n_kv, (c.m * c.g + SC_ROWS - 1) / SC_ROWS);
        auto fn = c.bf16 ? k_block_score<__nv_bfloat16> : k_block_score<__half>;
        static SmemLimit limit[2];
        e = limit[c.bf16].raise((const void*)fn, score_smem(256));
        if (e != cudaSuccess) return e;
        e = launch_pdl(fn, grid, SC_THREADS, score_smem(c.hd), s, c, nb_cap);
        if (e != cudaSuccess) return e;
    }
    if (n_cand <= BS_SINGLE)
        return launch_pdl(k_block_choose<1>, dim3(1, c.n_kv, c.m), SEL_THREADS, (size_t)n_cand * 8, s, c, nb_cap);
    static SmemLimit limit;
    e = limit.raise((const void*)k_block_choose<CL>, 128 * 1024);
    if (e != cudaSuccess) return e;
    return launch_cluster(k_block_choose<CL>, CL, dim3(CL, c.n_kv, c.m), SEL_THREADS, (size_t)((n_cand + CL - 1) / CL) * 8, s,
                          c, nb_cap);
}

cudaError_t launch_cache_take(void* kc, void* vc, int64_t rs, int64_t hs, int n_kv, int hd, int row0,
                              const TakePath& path, int n, cudaStream_t s) {
    return launch_pdl(k_cache_take, dim3(n_kv, 2), 32, 0, s, (char*)kc, (char*)vc, rs, hs, hd, row0, path, n);
}

}  // namespace hoard
