// kernels_cache_select.cu -- choosing rows and blocks of a KV cache: eviction by accumulated weight, the
// blocks' bounds and scores, the selection of blocks, and the moves of rows.
//
// Both selections are "the k largest of n keys, the lower index where equal", n from a few to 10^5. A cluster
// of eight CTAs holds the keys of one problem in shared memory, each CTA a contiguous range so that order is
// kept, and narrows the threshold by radix: histograms of eight bits from the top, added up over the cluster
// through distributed shared memory, until the bin that holds the k-th key holds no more than are wanted.
// Counting ranks by pairs is n^2, a sort moves what is not asked for, and one CTA alone is bound by the
// bandwidth of one SM.
#include "common.cuh"
#include "kernels_cache.h"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace hoard {

namespace {

constexpr int CL = 8;                    // CTAs of a cluster (the portable maximum)

// exclusive prefix sum over the CTA; total receives the sum. One 64-bit value per thread.
template <int THREADS>
__device__ __forceinline__ unsigned long long block_scan(unsigned long long v, unsigned long long* s_warp,
                                                         unsigned long long& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();                     // s_warp may still be read from an earlier scan
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    unsigned long long before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        const unsigned long long y = s_warp[w];
        if (w < warp) before += y;
        all += y;
    }
    total = all;
    return before + x - v;
}

struct Exchange {                        // one CTA's contribution to cluster-wide prefixes
    unsigned long long v[2];
};

// exclusive prefix over the cluster's CTAs of `total` (slot: which of the two buffers; a buffer is not
// written again before every CTA has passed another cluster barrier)
__device__ __forceinline__ unsigned long long cluster_before(cg::cluster_group& cl, Exchange* ex, int slot,
                                                             unsigned long long total) {
    if (threadIdx.x == 0) ex->v[slot] = total;
    cl.sync();
    unsigned long long before = 0;
    for (unsigned r = 0; r < cl.block_rank(); ++r) before += cl.map_shared_rank(ex, r)->v[slot];
    return before;
}

// The `need` largest of the cluster's keys: afterwards a key is in if (key >> shift) > prefix, and of those
// with (key >> shift) == prefix the first `eq_need` in index order are. key(i): this CTA's i-th key.
// hist: two buffers of 256 counts.
struct Threshold {
    unsigned long long prefix;
    int shift, eq_need;
};
template <int THREADS, int BITS, typename Key>
__device__ __forceinline__ Threshold cluster_threshold(cg::cluster_group& cl, Key key, int n_local, int need,
                                                       unsigned (*hist)[256], unsigned long long* s_warp) {
    __shared__ unsigned s_bin, s_in_bin, s_above;
    unsigned long long prefix = 0;
    int shift = BITS, buf = 0;
    for (;;) {
        shift -= 8;
        for (int i = threadIdx.x; i < 256; i += THREADS) hist[buf][i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n_local; i += THREADS) {
            const unsigned long long k = key(i);
            if (shift == BITS - 8 || (k >> (shift + 8)) == prefix) atomicAdd(&hist[buf][(k >> shift) & 255], 1u);
        }
        cl.sync();
        unsigned mine = 0;               // thread i: bin 255 - i, so that the scan runs from the top
        if (threadIdx.x < 256)
            for (int r = 0; r < CL; ++r) mine += cl.map_shared_rank(&hist[buf][0], r)[255 - threadIdx.x];
        unsigned long long total;
        const unsigned above = (unsigned)block_scan<THREADS>(mine, s_warp, total);
        if (threadIdx.x < 256 && above < (unsigned)need && above + mine >= (unsigned)need) {
            s_bin = 255 - threadIdx.x;
            s_in_bin = mine;
            s_above = above;
        }
        __syncthreads();
        prefix = prefix << 8 | s_bin;
        need -= (int)s_above;
        const bool done = shift == 0 || s_in_bin == (unsigned)need;
        __syncthreads();                 // s_bin is read before the next pass writes it
        if (done) return {prefix, shift, need};
        buf ^= 1;
    }
}

// ---- eviction: the moves ------------------------------------------------------------------------------------
// Key of a row: protected rows above everything; weights in order; NaN below everything. -0 equals +0.
constexpr int EV_THREADS = 1024, EV_KEYS = 40960;      // keys a CTA holds in shared memory (160 KiB)
__device__ __forceinline__ unsigned evict_key(float acc, int pos, int n_sink, int recent_from) {
    if (pos < n_sink || pos >= recent_from) return 0xFFFFFFFFu;
    if (acc != acc) return 0u;
    const unsigned b = __float_as_uint(acc + 0.f);
    return b >> 31 ? ~b : b | 0x80000000u;
}
// Grid (CL, n_kv). Writes to[], from[] (rows, ascending both) and the number of moves of each head, and
// acc_out / pos_out of the kept rows that stay where they are.
__global__ void __cluster_dims__(CL, 1, 1) __launch_bounds__(EV_THREADS) k_evict_choose(const CacheEvict e) {
    pdl_enter();
    extern __shared__ unsigned s_key[];
    __shared__ unsigned hist[2][256];
    __shared__ unsigned long long s_warp[EV_THREADS / 32];
    __shared__ Exchange s_ex;
    cg::cluster_group cl = cg::this_cluster();
    const int kv = blockIdx.y, rank = (int)cl.block_rank(), tid = threadIdx.x;
    const float* acc = e.acc + (int64_t)kv * e.max_rows;
    const int32_t* pos = e.pos + (int64_t)kv * e.max_rows;
    const int first = (int)((int64_t)e.n_rows * rank / CL), last = (int)((int64_t)e.n_rows * (rank + 1) / CL);
    const int n = last - first;
    const bool held = n <= EV_KEYS;
    auto fresh = [&](int i) { return evict_key(acc[first + i], pos[first + i], e.n_sink, e.recent_from); };
    if (held)
        for (int i = tid; i < n; i += EV_THREADS) s_key[i] = fresh(i);
    __syncthreads();
    auto key = [&](int i) { return held ? s_key[i] : fresh(i); };
    const Threshold th = cluster_threshold<EV_THREADS, 32>(cl, key, n, e.n_keep, hist, s_warp);

    // a thread owns a run of rows (odd length: the runs' first words fall in different banks)
    const int len = (n + EV_THREADS - 1) / EV_THREADS | 1, i0 = min(n, tid * len), i1 = min(n, i0 + len);
    unsigned long long eq = 0, total;
    for (int i = i0; i < i1; ++i) eq += (unsigned long long)(key(i) >> th.shift) == th.prefix;
    unsigned long long eq_rank = block_scan<EV_THREADS>(eq, s_warp, total);
    eq_rank += cluster_before(cl, &s_ex, 0, total);
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
    unsigned long long at = block_scan<EV_THREADS>(counts, s_warp, total);
    const unsigned long long before = cluster_before(cl, &s_ex, 1, total);
    at += before;
    if (rank == CL - 1 && tid == 0) e.n_moves[kv] = (int)((before + total) & 0xFFFFFFFFu);
    eq_rank = eq_rank0;
    int32_t* to = e.to + (int64_t)kv * e.max_rows;
    int32_t* from = e.from + (int64_t)kv * e.max_rows;
    int n_to = (int)(at & 0xFFFFFFFFu), n_from = (int)(at >> 32);
    for (int i = i0; i < i1; ++i) {
        const bool k = kept(i);
        const int row = first + i;
        if (row < e.n_keep) {
            if (!k) {
                to[n_to++] = row;
            } else {
                e.acc_out[(int64_t)kv * e.max_rows + row] = acc[row];
                e.pos_out[(int64_t)kv * e.max_rows + row] = pos[row];
            }
        } else if (k) {
            from[n_from++] = row;
        }
    }
    cl.sync();                                         // no CTA leaves while its counts may be read
}
// One warp per move: lanes take the K row's 16-byte pieces, then the V row's. Rows read are at or above n_keep,
// rows written below it.
__global__ void __launch_bounds__(256) k_evict_move(const CacheEvict e) {
    pdl_enter();
    const int kv = blockIdx.y, i = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (i >= e.n_moves[kv]) return;
    const int64_t hb = (int64_t)kv * e.max_rows;
    const int to = e.to[hb + i], from = e.from[hb + i];
    const int c16 = e.hd / 8;
    const int64_t src = ((int64_t)from * e.rs + (int64_t)kv * e.hs) * 2, dst = ((int64_t)to * e.rs + (int64_t)kv * e.hs) * 2;
    for (int p = lane; p < 2 * c16; p += 32) {
        char* c = static_cast<char*>(p < c16 ? e.kc : e.vc) + (p < c16 ? p : p - c16) * 16;
        *reinterpret_cast<uint4*>(c + dst) = *reinterpret_cast<const uint4*>(c + src);
    }
    if (lane == 0) {
        e.acc_out[hb + to] = e.acc[hb + from];
        e.pos_out[hb + to] = e.pos[hb + from];
    }
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
#pragma unroll 4
        for (int r = gi + groups; r < block; r += groups) {
            V x;
            x.u = *reinterpret_cast<const uint4*>(base + r * rs);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                lo.h[i] = min2(lo.h[i], x.h[i]);
                hi.h[i] = max2(hi.h[i], x.h[i]);
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
// its warps share out the dims and their sums are added in warp order. A value is converted once for the
// eight rows, since conversions to f64 run at a quarter of the rate of its multiply-adds.
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
    uint32_t* sb = reinterpret_cast<uint32_t*>(red + 8 * SC_ROWS * 32);         // [32][hd + 1] words
    for (int i = tid; i < SC_ROWS * c.hd; i += SC_THREADS) {
        const int r = i / c.hd, d = i - r * c.hd, row = row0 + r;
        sq[i] = row < R ? (double)c.q[(row / c.g) * c.q_ts + (kv * c.g + row % c.g) * c.q_hs + d] : 0.0;
    }
    const int n = min(SC_BLOCKS, n_cand - b0);
    const uint32_t* src = reinterpret_cast<const uint32_t*>(c.bounds) +
                          ((int64_t)kv * (c.max_rows / c.block) + cd.first + b0) * c.hd;      // hd words a block
    for (int i = tid; i < n * c.hd; i += SC_THREADS) {
        const int b = i / c.hd, w = i - b * c.hd;
        sb[b * (c.hd + 1) + w] = src[i];
    }
    __syncthreads();
    double acc[SC_ROWS];
#pragma unroll
    for (int r = 0; r < SC_ROWS; ++r) acc[r] = 0.0;
    const uint32_t* mine = sb + min(lane, n - 1) * (c.hd + 1);
    for (int p = warp; p < c.hd / 2; p += 8) {
        const double2 lo = to_double2<KT>(mine[p]), hi = to_double2<KT>(mine[c.hd / 2 + p]);
#pragma unroll
        for (int r = 0; r < SC_ROWS; ++r) {
            const double2 q = *reinterpret_cast<const double2*>(sq + r * c.hd + 2 * p);
            acc[r] = fma(q.x, q.x > 0.0 ? hi.x : lo.x, acc[r]);
            acc[r] = fma(q.y, q.y > 0.0 ? hi.y : lo.y, acc[r]);
        }
    }
#pragma unroll
    for (int r = 0; r < SC_ROWS; ++r) red[(warp * SC_ROWS + r) * 32 + lane] = acc[r];
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += red[(w * SC_ROWS + warp) * 32 + lane];     // thread = (row, block)
    if (lane < n && row0 + warp < R) c.u[((int64_t)kv * R + row0 + warp) * nb_cap + b0 + lane] = s;
}

// ---- selection: one cluster per (KV head, token) -----------------------------------------------------------------
constexpr int BS_THREADS = 256, BS_MAX_G = 64;
__device__ __forceinline__ unsigned long long order_key(double v) {
    if (v != v) return 0ull;
    const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__global__ void __cluster_dims__(CL, 1, 1) __launch_bounds__(BS_THREADS) k_block_choose(const CacheSelect c, int nb_cap) {
    pdl_enter();
    extern __shared__ unsigned long long s_keys[];
    __shared__ unsigned hist[2][256];
    __shared__ unsigned long long s_warp[BS_THREADS / 32];
    __shared__ double s_max[BS_MAX_G], s_top[BS_MAX_G];
    __shared__ Exchange s_ex;
    cg::cluster_group cl = cg::this_cluster();
    const int kv = blockIdx.y, t = blockIdx.z, rank = (int)cl.block_rank(), tid = threadIdx.x;
    const int lane = tid & 31, warp = tid >> 5;
    const Candidates cd = candidates(c);
    const int n_cand = cd.last - cd.first, n_take = min(n_cand, c.n_sel);
    const int prob = kv * c.m + t;
    int32_t* list = c.list + (int64_t)prob * c.list_cap;
    int32_t* sel = c.sel_out ? c.sel_out + ((int64_t)t * c.n_kv + kv) * c.n_sel : nullptr;
    // the blocks that are always attended, and the tail of sel
    const int gtid = rank * BS_THREADS + tid, gn = CL * BS_THREADS;
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
    const int i0 = (int)((int64_t)n_cand * rank / CL), i1 = (int)((int64_t)n_cand * (rank + 1) / CL), n = i1 - i0;
    const double* u = c.u + ((int64_t)kv * c.m + t) * c.g * nb_cap + i0;
    for (int h = warp; h < c.g; h += BS_THREADS / 32) {
        double mx = -INFINITY;
        for (int i = lane; i < n; i += 32) mx = fmax(mx, u[(int64_t)h * nb_cap + i]);
        for (int o = 16; o > 0; o >>= 1) mx = fmax(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        if (lane == 0) s_max[h] = mx;
    }
    cl.sync();
    if (tid < c.g) {
        double mx = -INFINITY;
        for (int r = 0; r < CL; ++r) mx = fmax(mx, cl.map_shared_rank(s_max, r)[tid]);
        s_top[tid] = mx;
    }
    __syncthreads();
    for (int i = tid; i < n; i += BS_THREADS) {
        double best = -INFINITY;
        for (int h = 0; h < c.g; ++h) best = fmax(best, u[(int64_t)h * nb_cap + i] - s_top[h]);
        s_keys[i] = order_key(best);
    }
    __syncthreads();
    auto key = [&](int i) { return s_keys[i]; };
    const Threshold th = cluster_threshold<BS_THREADS, 64>(cl, key, n, n_take, hist, s_warp);
    const int len = (n + BS_THREADS - 1) / BS_THREADS | 1, a0 = min(n, tid * len), a1 = min(n, a0 + len);
    unsigned long long eq = 0, total;
    for (int i = a0; i < a1; ++i) eq += (s_keys[i] >> th.shift) == th.prefix;
    unsigned long long eq_rank = block_scan<BS_THREADS>(eq, s_warp, total);
    eq_rank += cluster_before(cl, &s_ex, 0, total);
    unsigned long long count = 0;
    const unsigned long long eq_rank0 = eq_rank;
    auto kept = [&](int i) {
        const unsigned long long k = s_keys[i] >> th.shift;
        return k > th.prefix || (k == th.prefix && eq_rank++ < (unsigned long long)th.eq_need);
    };
    for (int i = a0; i < a1; ++i) count += kept(i);
    unsigned long long at = block_scan<BS_THREADS>(count, s_warp, total);
    at += cluster_before(cl, &s_ex, 1, total);
    eq_rank = eq_rank0;
    for (int i = a0; i < a1; ++i)
        if (kept(i)) {
            const int b = cd.first + i0 + i;
            list[cd.first + at] = b;
            if (sel) sel[at] = b;
            ++at;
        }
    cl.sync();
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
    const int n = (int)(((int64_t)e.n_rows + CL - 1) / CL);
    const size_t smem = n <= EV_KEYS ? (size_t)n * 4 : 0;
    cudaError_t rc = cudaFuncSetAttribute(k_evict_choose, cudaFuncAttributeMaxDynamicSharedMemorySize, EV_KEYS * 4);
    if (rc != cudaSuccess) return rc;
    rc = launch_pdl(k_evict_choose, dim3(CL, e.n_kv), EV_THREADS, smem, s, e);
    if (rc != cudaSuccess) return rc;
    const int most = e.n_keep < e.n_rows - e.n_keep ? e.n_keep : e.n_rows - e.n_keep;
    if (most == 0) return cudaSuccess;
    return launch_pdl(k_evict_move, dim3((most + 7) / 8, e.n_kv), 256, 0, s, e);
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
        const size_t smem = (size_t)SC_ROWS * c.hd * 8 + 8 * SC_ROWS * 32 * 8 + (size_t)SC_BLOCKS * (c.hd + 1) * 4;
        auto fn = c.bf16 ? k_block_score<__nv_bfloat16> : k_block_score<__half>;
        e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, 72 * 1024);
        if (e != cudaSuccess) return e;
        e = launch_pdl(fn, grid, SC_THREADS, smem, s, c, nb_cap);
        if (e != cudaSuccess) return e;
    }
    const size_t smem = (size_t)((n_cand + CL - 1) / CL) * 8;
    e = cudaFuncSetAttribute(k_block_choose, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 * 1024);
    if (e != cudaSuccess) return e;
    return launch_pdl(k_block_choose, dim3(CL, c.n_kv, c.m), BS_THREADS, smem, s, c, nb_cap);
}

cudaError_t launch_cache_take(void* kc, void* vc, int64_t rs, int64_t hs, int n_kv, int hd, int row0,
                              const TakePath& path, int n, cudaStream_t s) {
    return launch_pdl(k_cache_take, dim3(n_kv, 2), 32, 0, s, (char*)kc, (char*)vc, rs, hs, hd, row0, path, n);
}

}  // namespace hoard
