// kernels_cache.cu -- attention of several query tokens over a KV cache, split over the cache's rows.
//
//   s_rj = scale * q_r . K_j,  out_r = sum_j exp(s_rj - M_r) V_j / sum_j exp(s_rj - M_r),  M_r = max_j s_rj
//
// For the R query rows of a KV head (tokens x query heads of the head) the cache's K and V are read once
// and every product is a matrix instruction (m16n8k16): S^T[16 rows j x 8 query rows] = K q^T, and
// O^T[dims x 8 query rows] += V^T P^T. Eight query rows are the N of the instruction, so one token of a
// model with eight heads per KV head wastes nothing. The sums over j are split over CTAs, and inside a
// CTA over warps: a warp takes 16-row chunks of the cache through a ring of its own (cp.async, no barrier
// between warps), with its own running maximum and total, and the partial results are joined once at the
// end of the CTA and once after all CTAs (k_cache_combine).
//
// Bound by: latency over short caches (one CTA's chain of loads, products and joins: 4.5 us over 40 rows), the warps' chains of
// products over middle ones (a 16-row chunk of a warp 1.1 to 1.4 us at 64 and 128 dims, 2.6 at 256), DRAM over long ones: 16
// heads of 128, one token each, over 30000 rows 245 MB in 42 us, 5.8 TB/s. At 256 dims the registers allow eight warps, whose
// chains do not cover the loads: 2 heads over 32769 rows 67 MB in 18.5 us, 3.6 TB/s.
//
// Precision. K and V enter the products as they are stored. q (f32) and the weights p (f32) are written as
// sums of f16 or bf16 terms (kv_terms.cuh), whatever the cache's type is, so a product is f32-accurate; sums, maxima
// and totals are f32.
#include "common.cuh"
#include "kernels_cache.h"
#include "async_copy.cuh"
#include "kv_terms.cuh"

#include <cmath>
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace hoard {

namespace {

template <typename KT>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if constexpr (sizeof(KT) == 2 && Terms<KT>::N == 2)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldm4(uint32_t* r, unsigned addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t* r, unsigned addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// 16 bytes global -> shared, or 16 zero bytes where !there (the source is not read)
__device__ __forceinline__ void cp16z(unsigned dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
template <int N> __device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// Warps and ring slots of one CTA (one CTA per SM). A slot is the K or the V of 16 rows; the warps with all but one of their
// slots in flight keep 128 to 170 KiB per SM on the way. Eight warps; tiles of 8 rows of 64 dims have registers and slots for
// twelve: 8 heads over 100000 cache rows 63.3 us with 8, 39.0 with 12, 37.9 with 16; over 40 rows 4.1, 4.5, 4.7. At 128 dims
// twelve are slower over few rows and no faster over many (4 heads, 8 rows: 7.8 / 9.0 over 2300, 36.7 / 39.1 over
// 100000), at 256 dims slower everywhere (9.2 / 10.8, 39.6 / 41.5).
constexpr int MAX_CLUSTER = 4;           // CTAs of a cluster: with a CTA per SM, eight rarely fit in a GPC at once
constexpr int plan_warps(int hd, int nt) { return hd == 64 && nt == 1 ? 12 : 8; }
template <int HD, int NT> struct Plan {
    static constexpr int W = plan_warps(HD, NT), NS = HD == 256 ? 3 : W == 12 ? 8 : 6;
    static constexpr int SLOT = KV_CHUNK * HD * 2;                 // bytes
    static constexpr int RING = W * NS * SLOT;
};
template <typename KT, int HD, int NT> constexpr int q_bytes() { return HD / 16 * NT * Terms<KT>::N * 32 * 8; }
template <typename KT, int HD, int NT> constexpr int attn_smem() {
    constexpr int ring = Plan<HD, NT>::RING + q_bytes<KT, HD, NT>(), join = Plan<HD, NT>::W * 8 * NT * (HD + 4) * 4;
    return ring > join ? ring : join;
}

__device__ __forceinline__ int past_rows(const CacheAttn& a) {
    return a.n_past_dev ? max(0, min(*a.n_past_dev, a.max_rows - a.m)) : a.n_past;
}

template <typename KT, int HD, int KS, int NT, bool BLOCKS>
__global__ void __launch_bounds__(Plan<HD, NT>::W * 32, 1) k_cache_attention(const CacheAttn a) {
    constexpr int W = Plan<HD, NT>::W, NS = Plan<HD, NT>::NS, SLOT = Plan<HD, NT>::SLOT, TN = Terms<KT>::N;
    static_assert(KS <= HD / 16, "K steps of q . K = M tiles of V^T, as many as the dims need");
    constexpr int RT = 8 * NT;                         // query rows of the tile
    constexpr int PITCH = HD * 2;                      // bytes of a staged row
    constexpr int C16 = HD / 8;                        // 16-byte pieces of a row
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ float s_scale[RT];                      // per query row: scale, log2(e) and the row's power of two
    __shared__ uint64_t s_vis[RT];
    __shared__ float s_m[W][RT], s_l[W][RT];
    __shared__ float2 s_ml[RT];                        // the CTA's maxima and totals
    __shared__ float s_fac[MAX_CLUSTER][RT], s_top[RT], s_inv[RT];
    pdl_enter();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = blockIdx.x, tile = blockIdx.y, prob = blockIdx.z;
    const int n_past = past_rows(a);
    const int kv = BLOCKS ? prob / a.m : prob;
    const int t0 = BLOCKS ? prob - kv * a.m : 0;       // first token of the problem's rows
    uint32_t* qf = reinterpret_cast<uint32_t*>(smem + Plan<HD, NT>::RING);

    // chunks of this CTA: past rows (or the listed blocks' rows), then the tokens' own rows
    const int sub_shift = BLOCKS ? __ffs(a.block / KV_CHUNK) - 1 : 0;         // chunks of a block: a power of two
    const int n_pc = BLOCKS ? a.list_n[prob] << sub_shift : (n_past + KV_CHUNK - 1) / KV_CHUNK;
    const int n_chunks = n_pc + (a.m + KV_CHUNK - 1) / KV_CHUNK;
    const Share share_of(n_chunks, gridDim.x);
    const int c_end = share_of.first(split + 1), c_first = share_of.first(split) + warp;
    const int32_t* list = BLOCKS ? a.list + (int64_t)prob * a.list_cap : nullptr;
    auto chunk_row = [&](int c) {                      // first cache row of chunk c
        if (c >= n_pc) return n_past + (c - n_pc) * KV_CHUNK;
        if (BLOCKS) return list[c >> sub_shift] * a.block + (c & ((1 << sub_shift) - 1)) * KV_CHUNK;
        return c * KV_CHUNK;
    };
    auto chunk_end = [&](int c) { return c >= n_pc ? n_past + a.m : n_past; };

    // the warp's ring; lane -> (row of the piece, 16-byte piece) with consecutive lanes on consecutive pieces
    const unsigned ring = smem_u32(smem) + warp * NS * SLOT;
    const int n_mine = c_first < c_end ? (c_end - c_first + W - 1) / W : 0;      // chunks of this warp
    // slot load i: K (i even) or V of the warp's chunk i / 2, into ring slot i % NS
    int load = 0, load_slot = 0;
    auto issue = [&]() {
        if (load < 2 * n_mine) {
            const int c = c_first + (load >> 1) * W, row0 = chunk_row(c), end = chunk_end(c);
            const char* base = static_cast<const char*>(load & 1 ? a.vc : a.kc) + (int64_t)kv * a.hs * 2;
            const unsigned dst = ring + load_slot * SLOT;
#pragma unroll
            for (int i = 0; i < KV_CHUNK * C16 / 32; ++i) {
                const int p = i * 32 + lane, r = p / C16, c16 = p % C16;
                const bool there = row0 + r < end && c16 * 8 < a.hd;
                cp16z(dst + r * PITCH + ((c16 ^ (r & 7)) << 4),
                      there ? base + (int64_t)(row0 + r) * a.rs * 2 + c16 * 16 : base, there);
            }
        }
        cp_async_commit();
        ++load;
        load_slot = load_slot == NS - 1 ? 0 : load_slot + 1;
    };
#pragma unroll 1
    for (int i = 0; i < NS - 1; ++i) issue();

    // the tile's q rows as fragments of the B operand: [K step][8-row tile][term][lane] of 8 bytes. A warp takes
    // every W-th row and loads all of them before it uses the first
    constexpr int QR = (RT + W - 1) / W;
    float x[QR][HD / 32];
#pragma unroll
    for (int i = 0; i < QR; ++i) {
        const int row = tile * RT + warp + i * W;      // row = (token - t0) * g + head of the KV head
        const bool live = warp + i * W < RT && row < a.R;
        const int t = t0 + (live ? row / a.g : 0), h = kv * a.g + (live ? row % a.g : 0);
        const float* q = a.q + t * a.q_ts + h * a.q_hs;
#pragma unroll
        for (int k = 0; k < HD / 32; ++k) x[i][k] = live && k * 32 + lane < a.hd ? q[k * 32 + lane] : 0.f;
    }
    if (tid < RT) {
        const int row = tile * RT + tid, t = t0 + row / a.g;
        s_vis[tid] = row >= a.R ? 0 : a.vis ? a.vis[t] : t >= 63 ? ~0ull : (1ull << (t + 1)) - 1;
    }
#pragma unroll
    for (int i = 0; i < QR; ++i) {
        const int r = warp + i * W;
        if (RT % W && r >= RT) break;
        float am = 0.f;
        bool bad = false;
#pragma unroll
        for (int k = 0; k < HD / 32; ++k) {
            bad |= !(fabsf(x[i][k]) < INFINITY);
            am = fmaxf(am, fabsf(x[i][k]));
        }
        am = warp_max(am);
        bad = __any_sync(0xffffffffu, bad);
        const RowScale rs = row_scale<KT>(am, bad);
        if (lane == 0) s_scale[r] = a.scale_log2 * rs.down;
#pragma unroll
        for (int k = 0; k < HD / 32; ++k) {
            // lanes 2c, 2c + 1 hold the pair of dims that one fragment register packs
            float lo = x[i][k] * rs.up;
            float hi = __shfl_down_sync(0xffffffffu, lo, 1);
            const int d = k * 32 + lane, kk = d >> 4, reg = (d >> 3) & 1, c = (d & 7) >> 1;
#pragma unroll
            for (int u = 0; u < TN; ++u) {
                const uint32_t w = take_term<KT>(lo, hi);
                if (!(lane & 1))
                    qf[((((kk * NT + (r >> 3)) * TN + u) * 32) + ((r & 7) << 2) + c) * 2 + reg] = w;
            }
        }
    }
    __syncthreads();

    // fragment addresses inside a stage
    const int k_r = (lane & 7) + ((lane >> 3) & 1) * 8, k_c = lane >> 4;         // K: rows j, dims
    const int v_r = (lane & 7) + (lane >> 4) * 8, v_c = (lane >> 3) & 1;         // V transposed: keys, dims
    const int cq = lane & 3;                            // query rows 2 cq, 2 cq + 1 of each 8-row tile

    float o[KS][NT][4];
    float mx[NT][2], tot[NT][2], sc[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            mx[n][i] = -INFINITY;
            tot[n][i] = 0.f;
            sc[n][i] = s_scale[8 * n + 2 * cq + i];
        }
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[k][n][i] = 0.f;
    }

    int slot = 0;                                      // ring slot of the next K or V
    // the next slot's bytes have arrived; the slot before it is free and takes the next load
    auto next_slot = [&]() {
        cp_wait<NS - 2>();
        __syncwarp();
        issue();
        const unsigned at = ring + slot * SLOT;
        slot = slot == NS - 1 ? 0 : slot + 1;
        return at;
    };
#pragma unroll 1
    for (int c = c_first; c < c_end; c += W) {
        const unsigned ks = next_slot();
        // ---- S^T = K q^T: each K step's products by matrix instructions, added with rounding (the instructions
        // truncate as they accumulate), which also leaves no chain of instructions longer than the terms ----
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[n][i] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            uint32_t af[4];
            ldm4(af, ks + k_r * PITCH + (((2 * k + k_c) ^ (k_r & 7)) << 4));
#pragma unroll
            for (int n = 0; n < NT; ++n)
            {
                float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int u = TN - 1; u >= 0; --u) {
                    const uint2 b = *reinterpret_cast<const uint2*>(qf + ((((k * NT + n) * TN + u) * 32) + lane) * 2);
                    mma16816<KT>(x, af, b.x, b.y);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) s[n][i] += x[i];
            }
        }
        // ---- scores in log2 units; masked ones -inf ----
        const int row0 = chunk_row(c), left = chunk_end(c) - row0;               // rows of the chunk that exist
        const bool own = c >= n_pc;
        const int j0 = lane >> 2, j1 = j0 + 8;                                   // this thread's rows of the chunk
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[n][i] = __fmul_rn(s[n][i], sc[n][i & 1]);      // a score: rounded once, nowhere fused
        if (left < KV_CHUNK || own) {
            const int sh = own ? row0 - n_past : 0;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = i < 2 ? j0 : j1;
                    const bool see = j < left && (!own || (s_vis[8 * n + 2 * cq + (i & 1)] >> (sh + j) & 1));
                    if (!see) s[n][i] = -INFINITY;
                }
        }
        if (!BLOCKS && a.logits) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = tile * RT + 8 * n + 2 * cq + (i & 1), j = i < 2 ? j0 : j1;
                    if (row < a.R && j < left) a.logits[((int64_t)kv * a.R + row) * a.logits_ld + row0 + j] = s[n][i];
                }
        }
        // ---- running maximum; earlier sums are rescaled only when one rises ----
        bool rises = false;
        float top[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float v = fmaxf(s[n][i], s[n][i + 2]);
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
                top[n][i] = fmaxf(mx[n][i], v);
                rises |= top[n][i] > mx[n][i];
            }
        if (__any_sync(0xffffffffu, rises)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float f[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    f[i] = top[n][i] > mx[n][i] ? ex2f(mx[n][i] - top[n][i]) : 1.f;
                    mx[n][i] = top[n][i];
                    tot[n][i] *= f[i];
                }
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    o[k][n][0] *= f[0];
                    o[k][n][1] *= f[1];
                    o[k][n][2] *= f[0];
                    o[k][n][3] *= f[1];
                }
            }
        }
        // ---- weights, their terms as B fragments ----
        uint32_t pf[NT][TN][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) b[i] = mx[n][i] == -INFINITY ? 0.f : mx[n][i];
#pragma unroll
            for (int i = 0; i < 4; ++i) s[n][i] = weight<KT>(s[n][i], b[i & 1]);
            tot[n][0] += s[n][0] + s[n][2];
            tot[n][1] += s[n][1] + s[n][3];
        }
        const unsigned vs = next_slot();
        // masked own rows may hold infinities or NaN (0 * inf): such a chunk takes its products one by one
        bool odd = false;
        if (own) {
            for (int i = lane; i < KV_CHUNK * C16; i += 32) {
                uint32_t w[4];
                asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                             : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(vs + i * 16) : "memory");
#pragma unroll
                for (int k = 0; k < 4; ++k) odd |= odd_pair<KT>(w[k]);
            }
            odd = __any_sync(0xffffffffu, odd);
        }
        if (!odd) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float r[4] = {s[n][0], s[n][1], s[n][2], s[n][3]};
#pragma unroll
                for (int u = 0; u < TN; ++u) {
                    pf[n][u][0] = transpose8(take_term<KT>(r[0], r[1]));
                    pf[n][u][1] = transpose8(take_term<KT>(r[2], r[3]));
                }
            }
            // ---- O^T += V^T P^T, added likewise: left in the instructions' accumulators over 8192 rows the sums
            // were 2e-5 off ----
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t af[4];
                ldm4t(af, vs + v_r * PITCH + (((2 * k + v_c) ^ (v_r & 7)) << 4));
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int u = TN - 1; u >= 0; --u) mma16816<KT>(x, af, pf[n][u][0], pf[n][u][1]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[k][n][i] += x[i];
                }
            }
        } else {
            for (int j = 0; j < KV_CHUNK; ++j) {
                const int src = ((j & 7) << 2) + cq;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float p0 = __shfl_sync(0xffffffffu, j < 8 ? s[n][0] : s[n][2], src);
                    const float p1 = __shfl_sync(0xffffffffu, j < 8 ? s[n][1] : s[n][3], src);
#pragma unroll
                    for (int k = 0; k < KS; ++k)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int d = 16 * k + 8 * i + (lane >> 2);
                            unsigned short hv;
                            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(hv)
                                         : "r"(vs + j * PITCH + (((d >> 3) ^ (j & 7)) << 4) + (d & 7) * 2) : "memory");
                            const float v = kv_lo<KT>(hv);
                            if (p0 != 0.f) o[k][n][2 * i] += p0 * v;
                            if (p1 != 0.f) o[k][n][2 * i + 1] += p1 * v;
                        }
                }
            }
        }
    }
    cp_async_wait_all();

    // ---- join the warps: totals over the four lanes' rows, then sums relative to the CTA's maximum ----
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float v = tot[n][i];
            v += __shfl_xor_sync(0xffffffffu, v, 4);
            v += __shfl_xor_sync(0xffffffffu, v, 8);
            v += __shfl_xor_sync(0xffffffffu, v, 16);
            // a total of NaN without a maximum (every score NaN) has to reach the output: any finite maximum does
            if (v != v && mx[n][i] == -INFINITY) mx[n][i] = 0.f;
            if (lane < 4) {
                s_m[warp][8 * n + 2 * cq + i] = mx[n][i];
                s_l[warp][8 * n + 2 * cq + i] = v;
            }
        }
    __syncthreads();                                   // every warp has left its ring
    constexpr int OP = HD + 4;                         // floats of a row in the join buffer (over the ring)
    static_assert(W * RT * OP * 4 <= attn_smem<KT, HD, NT>(), "join buffer");
    float* joined = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = 8 * n + 2 * cq + i;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < W; ++w) top = fmaxf(top, s_m[w][r]);
            const float f = mx[n][i] == -INFINITY ? 0.f : ex2f(mx[n][i] - top);
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                joined[(warp * RT + r) * OP + 16 * k + (lane >> 2)] = mx[n][i] == -INFINITY ? 0.f : o[k][n][i] * f;
                joined[(warp * RT + r) * OP + 16 * k + 8 + (lane >> 2)] = mx[n][i] == -INFINITY ? 0.f : o[k][n][i + 2] * f;
            }
        }
    __syncthreads();
    // the rows' maxima and totals over the warps, then the sums: to the output where nothing is to be joined, to the
    // partial results, or for the cluster in place of the first warp's
    const bool single = a.cluster && a.splits == 1;
    if (tid < RT) {
        float top = -INFINITY, l = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) top = fmaxf(top, s_m[w][tid]);
#pragma unroll
        for (int w = 0; w < W; ++w) l += s_m[w][tid] == -INFINITY ? 0.f : s_l[w][tid] * ex2f(s_m[w][tid] - top);
        s_ml[tid] = make_float2(top, l);
        s_top[tid] = top;
        s_inv[tid] = l == 0.f ? 0.f : 1.f / l;
        if (!a.cluster && tile * RT + tid < a.R)
            a.part_ml[((int64_t)prob * a.splits + split) * a.R + tile * RT + tid] = make_float2(top, l);
    }
    if (single) __syncthreads();
    auto put = [&](int r, int d, float4 v) {           // the output of row r of the tile, dims d ..
        const int row = tile * RT + r, tt = row / a.g, t = t0 + tt, h = kv * a.g + row - tt * a.g;
        const float inv = s_inv[r];
        float y[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
        if (a.gate) {
            const float* gp = a.gate + t * a.gate_ts + h * a.gate_hs + d;
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] *= sigmoid_f(gp[i]);
        }
        store4(a.out + ((int64_t)t * a.n_head + h) * a.hd + d, y);
    };
    float* sums = joined;
    for (int x = tid; x < RT * (HD / 4); x += W * 32) {
        const int r = x / (HD / 4), d = (x - r * (HD / 4)) * 4;
        const int row = tile * RT + r;
        if (row >= a.R || d >= a.hd) continue;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float4 u = *reinterpret_cast<const float4*>(joined + (w * RT + r) * OP + d);
            v.x += u.x;
            v.y += u.y;
            v.z += u.z;
            v.w += u.w;
        }
        if (single) put(r, d, v);
        else if (a.cluster) *reinterpret_cast<float4*>(sums + r * OP + d) = v;
        else *reinterpret_cast<float4*>(a.part_o + ((((int64_t)prob * a.splits + split) * a.R) + row) * HD + d) = v;
    }
    if (!a.cluster) return;

    // ---- the splits are the CTAs of a cluster: each has every split's maximum and total of the rows, joins its share of
    // the rows' sums and, with weights to accumulate, adds those of its own cache rows ----
    cg::cluster_group cl = cg::this_cluster();
    if (!single) {
        cl.sync();
        if (tid < RT) {
            float2 ml[MAX_CLUSTER];
            float top = -INFINITY, l = 0.f;
#pragma unroll
            for (int c = 0; c < MAX_CLUSTER; ++c) {
                ml[c] = make_float2(-INFINITY, 0.f);
                if (c < a.splits) ml[c] = *cl.map_shared_rank(&s_ml[tid], c);
                top = fmaxf(top, ml[c].x);
            }
#pragma unroll
            for (int c = 0; c < MAX_CLUSTER; ++c) {
                const float f = ml[c].x == -INFINITY ? 0.f : ex2f(ml[c].x - top);
                s_fac[c][tid] = f;
                l += f == 0.f ? 0.f : f * ml[c].y;
            }
            s_top[tid] = top;
            s_inv[tid] = l == 0.f ? 0.f : 1.f / l;
        }
        const int share = (RT + a.splits - 1) / a.splits, r0 = split * share;
        for (int x0 = 0; x0 < share * (HD / 4); x0 += W * 32) {
            const int x = x0 + tid, rr = x / (HD / 4), r = r0 + rr, d = (x - rr * (HD / 4)) * 4;
            const bool mine = rr < share && r < RT && tile * RT + r < a.R && d < a.hd;
            float4 u[MAX_CLUSTER];
#pragma unroll
            for (int c = 0; c < MAX_CLUSTER; ++c)
                if (mine && c < a.splits) u[c] = *reinterpret_cast<const float4*>(cl.map_shared_rank(sums, c) + r * OP + d);
            if (x0 == 0) __syncthreads();              // the factors are known
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (mine) {
#pragma unroll
                for (int c = 0; c < MAX_CLUSTER; ++c) {
                    const float f = s_fac[c][r];
                    if (c < a.splits && f != 0.f) {
                        v.x += f * u[c].x;
                        v.y += f * u[c].y;
                        v.z += f * u[c].z;
                        v.w += f * u[c].w;
                    }
                }
                put(r, d, v);
            }
        }
    }
    if (!BLOCKS && a.logits) {                         // one row tile: these are all the query rows of the KV head
        const float* lg = a.logits + (int64_t)kv * a.R * a.logits_ld;
        float* acc = a.acc + (int64_t)kv * a.max_rows;
        const int c0 = c_first - warp;                 // this CTA's first chunk
        for (int x = tid; x < (c_end - c0) * KV_CHUNK; x += W * 32) {
            const int c = c0 + x / KV_CHUNK, j = chunk_row(c) + x % KV_CHUNK;
            if (j >= chunk_end(c)) continue;
            const float before = acc[j];
            float lv[RT], w = 0.f;
#pragma unroll
            for (int r = 0; r < RT; ++r) lv[r] = r < a.R ? lg[(int64_t)r * a.logits_ld + j] : -INFINITY;
#pragma unroll
            for (int r = 0; r < RT; ++r)
                if (r < a.R && s_inv[r] != 0.f) w += weight<KT>(lv[r], s_top[r]) * s_inv[r];
            acc[j] = before + w;
        }
    }
    if (!single) cl.sync();                            // no CTA leaves while its sums may be read
}

// ---- joins the splits of every query row, and with acc adds the rows' weights to the accumulated ones -------
// Grid y: the problem. A CTA per query row (token, head) and block of columns (one block where there are rows enough):
// the factors 2^(m_s - M) of the splits, one split per thread, then float4 columns x split groups, eight partial rows in
// flight per thread. The CTAs after them take 1024 cache rows of a KV head each: w = sum over the head's query rows of
// 2^(s - M) / L in row order, four cache rows per thread. Bound by latency, three dependent rounds of loads: 3 us for 512
// rows of 33 splits; with a warp per row and its splits in sequence it was 29, and integer divisions before the loads
// cost 0.6.
constexpr int CB = 256, ACC_PER = 4, ACC_ROWS = CB * ACC_PER, ACC_MAX_R = 512;
static_assert(KV_SMS + 1 <= CB, "one split per thread");
__global__ void __launch_bounds__(CB) k_cache_combine(const CacheAttn a, int hdt, int col_shift, int v4, unsigned v4_inv) {
    pdl_enter();
    __shared__ float s_f[CB];
    __shared__ float s_red[2][CB / 32];
    __shared__ float4 s_o[CB];
    __shared__ float s_mr[ACC_MAX_R], s_ir[ACC_MAX_R];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int prob = blockIdx.y, n_rows = a.R << col_shift;
    if ((int)blockIdx.x < n_rows) {
        const int row = blockIdx.x >> col_shift;
        const int64_t part = (int64_t)prob * a.splits * a.R + row;       // + split * R
        // this CTA's float4 columns, shared out over split groups. The first round of sums is on its way before the
        // factors are known (what a split without weight left there is not used)
        const int groups = CB * v4_inv >> 16, gi = tid * v4_inv >> 16;                 // divided by v4
        const int lc = tid - gi * v4, c = (blockIdx.x - (row << col_shift)) * v4 + lc;
        const bool mine = gi < groups && 4 * c < a.hd;
        const float* po = a.part_o + part * hdt + 4 * c;
        float4 u[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int s = gi + k * groups;
            u[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (mine && s < a.splits) u[k] = *reinterpret_cast<const float4*>(po + (int64_t)s * a.R * hdt);
        }
        const float2 ml = tid < a.splits ? a.part_ml[part + (int64_t)tid * a.R] : make_float2(-INFINITY, 0.f);
        const float wm = warp_max(ml.x);
        if (lane == 0) s_red[0][warp] = wm;
        __syncthreads();
        float top = s_red[0][0];
#pragma unroll
        for (int w = 1; w < CB / 32; ++w) top = fmaxf(top, s_red[0][w]);
        const float f = ml.x == -INFINITY ? 0.f : ex2f(ml.x - top);
        s_f[tid] = f;
        const float wl = warp_sum(ml.x == -INFINITY ? 0.f : f * ml.y);
        if (lane == 0) s_red[1][warp] = wl;
        __syncthreads();
        float l = s_red[1][0];
#pragma unroll
        for (int w = 1; w < CB / 32; ++w) l += s_red[1][w];
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (mine) {
            for (int s0 = gi;;) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int s = s0 + k * groups;
                    const float w = s < a.splits ? s_f[s] : 0.f;
                    if (w != 0.f) {
                        v.x += w * u[k].x;
                        v.y += w * u[k].y;
                        v.z += w * u[k].z;
                        v.w += w * u[k].w;
                    }
                }
                s0 += 8 * groups;
                if (s0 >= a.splits) break;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int s = s0 + k * groups;
                    if (s < a.splits) u[k] = *reinterpret_cast<const float4*>(po + (int64_t)s * a.R * hdt);
                }
            }
            s_o[tid] = v;
        }
        __syncthreads();
        if (gi == 0 && 4 * c < a.hd) {
            for (int k = 1; k < groups; ++k) {
                const float4 u = s_o[k * v4 + lc];
                v.x += u.x;
                v.y += u.y;
                v.z += u.z;
                v.w += u.w;
            }
            const bool blocks = a.list != nullptr;
            const int kv = blocks ? prob / a.m : prob;
            const int t = (blocks ? prob - kv * a.m : 0) + row / a.g, h = kv * a.g + row % a.g;
            const float inv = l == 0.f ? 0.f : 1.f / l;
            float y[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
            if (a.gate) {
                const float* gp = a.gate + t * a.gate_ts + h * a.gate_hs + 4 * c;
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] *= sigmoid_f(gp[i]);
            }
            store4(a.out + ((int64_t)t * a.n_head + h) * a.hd + 4 * c, y);
        }
        return;
    }
    // accumulation
    const int n = past_rows(a) + a.m;
    const int kv = prob, j0 = (blockIdx.x - n_rows) * ACC_ROWS;
    if (j0 >= n) return;
    const float* lg = a.logits + (int64_t)kv * a.R * a.logits_ld;
    float* acc = a.acc + (int64_t)kv * a.max_rows;
    float w[ACC_PER];
#pragma unroll
    for (int i = 0; i < ACC_PER; ++i) w[i] = j0 + i * CB + tid < n ? acc[j0 + i * CB + tid] : 0.f;
    // a warp per query row: its maximum and total over the splits
    for (int row = warp; row < a.R; row += CB / 32) {
        const float2* ml = a.part_ml + (int64_t)kv * a.splits * a.R + row;
        float2 v[(KV_SMS + 32) / 32];
        float top = -INFINITY, l = 0.f;
#pragma unroll
        for (int k = 0; k < (KV_SMS + 32) / 32; ++k) {
            const int s = lane + 32 * k;
            v[k] = s < a.splits ? ml[(int64_t)s * a.R] : make_float2(-INFINITY, 0.f);
            top = fmaxf(top, v[k].x);
        }
        top = warp_max(top);
#pragma unroll
        for (int k = 0; k < (KV_SMS + 32) / 32; ++k) l += v[k].x == -INFINITY ? 0.f : ex2f(v[k].x - top) * v[k].y;
        l = warp_sum(l);
        if (lane == 0) {
            s_mr[row] = top;
            s_ir[row] = l == 0.f ? 0.f : 1.f / l;
        }
    }
    __syncthreads();
    const float pe = a.bf16 ? Terms<__nv_bfloat16>::P_EXP : Terms<__half>::P_EXP;      // l holds 2^P_EXP sum p
    float sum[ACC_PER] = {};
    for (int r0 = 0; r0 < a.R; r0 += 4) {
        float s[4][ACC_PER];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int i = 0; i < ACC_PER; ++i) {
                const int j = j0 + i * CB + tid;
                s[k][i] = r0 + k < a.R && j < n ? lg[(r0 + k) * a.logits_ld + j] : -INFINITY;
            }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (r0 + k < a.R && s_ir[r0 + k] != 0.f)
#pragma unroll
                for (int i = 0; i < ACC_PER; ++i) sum[i] += ex2f((s[k][i] - s_mr[r0 + k]) + pe) * s_ir[r0 + k];
    }
#pragma unroll
    for (int i = 0; i < ACC_PER; ++i)
        if (j0 + i * CB + tid < n) acc[j0 + i * CB + tid] = w[i] + sum[i];
}

template <typename KT, int HD, int KS, int NT, bool BLOCKS>
cudaError_t attention_go(const CacheAttn& a, cudaStream_t s) {
    constexpr int smem = attn_smem<KT, HD, NT>();
    constexpr int W = Plan<HD, NT>::W;
    static SmemLimit limit;
    cudaError_t e = limit.raise((const void*)k_cache_attention<KT, HD, KS, NT, BLOCKS>, smem);
    if (e != cudaSuccess) return e;
    const dim3 grid(a.splits, a.row_tiles, a.problems);
    if (!a.cluster) return launch_pdl(k_cache_attention<KT, HD, KS, NT, BLOCKS>, grid, W * 32, smem, s, a);
    return launch_pdl_cluster(k_cache_attention<KT, HD, KS, NT, BLOCKS>, a.splits, grid, W * 32, smem, s, a);
}
template <typename KT, int HD, int KS, int NT> cudaError_t attention_form(const CacheAttn& a, cudaStream_t s) {
    return a.list ? attention_go<KT, HD, KS, NT, true>(a, s) : attention_go<KT, HD, KS, NT, false>(a, s);
}
template <typename KT> cudaError_t attention_type(const CacheAttn& a, cudaStream_t s) {
    const bool one = a.tile_rows == 8;
    // up to 96 dims run six K steps in rows of 128: 4 heads of 96 with 12 rows over 100000 cache rows 43.0 us, 48.2 with eight
    if (a.hd <= 64) return one ? attention_form<KT, 64, 4, 1>(a, s) : attention_form<KT, 64, 4, 2>(a, s);
    if (a.hd <= 96) return one ? attention_form<KT, 128, 6, 1>(a, s) : attention_form<KT, 128, 6, 2>(a, s);
    if (a.hd <= 128) return one ? attention_form<KT, 128, 8, 1>(a, s) : attention_form<KT, 128, 8, 2>(a, s);
    return one ? attention_form<KT, 256, 16, 1>(a, s) : attention_form<KT, 256, 16, 2>(a, s);
}

}  // namespace

int cache_tile_dims(int hd) { return hd <= 64 ? 64 : hd <= 128 ? 128 : 256; }

// The plan of a call: query rows of a tile (8 or 16), splits of the chunks and who joins them, or the tensor-core form.
// The choice is by time, from what the parts were measured to take in microseconds, for f16 (bf16 takes a tenth more in either
// form, which the choice leaves out):
//
//   - a CTA's start and end, and a chunk of each of its warps (a CTA has as many in turn as its fullest warp):
//     tiles of 16 cost more of both and halve the reads of the cache where there are more than 8 rows
//   - joining: nothing for one CTA; 1.2 for a cluster of 2 or 4, which joins in shared memory; a second kernel takes 2.5
//     and, up to 128 query rows, 0.01 for each
//   - the tensor-core form: its start, 1 / 256 for each query row (staged, split into terms, stored) and a tile of 64 cache
//     rows. It takes 128 query rows at once, so that its time hardly depends on them
//
// Both sides, measured: 4 heads of 128 with 32 rows each over 250 cache rows: one CTA 7.4, cluster of 4 6.4, second kernel
// 8.4; over 1000 with 8 rows: 10.5 for 2 CTAs, 8.0 for a cluster of 4, 7.4 for eight splits; heads of 256 over 1400: cluster
// 13.3, sixteen splits 9.0. Tiles of 8 against 16: 4 heads of 128 with 64 rows 11.0 / 12.1 over 2000 cache rows, 47 / 34 over
// 16000. Tensor cores against the best of these: 4 heads of 128 with 24 rows 13.2 / 11.5 over 4000 cache rows, 15.1 / 15.0
// over 8000, 35.5 / 58.0 over 64000; with 512 rows 20.3 / 15.6 over 600, 31.8 / 115 over 8000; 16 heads with 33 rows 13.1 /
// 11.7 over 600, 15.3 / 18.9 over 2000. Up to 16 rows a tile of 16 reads the cache once as well, and they are not asked for.
struct TileCost {
    float base, chunk;
};
constexpr TileCost TILE_COST[3][2] = {{{3.4f, 1.15f}, {4.3f, 1.15f}}, {{3.2f, 1.4f}, {4.4f, 1.8f}}, {{3.9f, 2.6f}, {5.5f, 3.9f}}};
constexpr TileCost TC_COST[2] = {{8.6f, 0.7f}, {10.f, 1.f}};
// CTAs up to which clusters of four all run at once (a CTA per SM, and SMs of a GPC left over)
constexpr int CLUSTERED_CTAS = 128;

inline int64_t up_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

void cache_plan(CacheAttn& a, int n_chunks, int64_t past_rows) {
    const int dims = cache_tile_dims(a.hd), di = dims == 64 ? 0 : dims == 128 ? 1 : 2;
    const int64_t rows = (int64_t)a.problems * a.R;
    const float second = 2.5f + 0.01f * (rows < 128 ? rows : 128);
    float best = INFINITY;
    a.tc_splits = 0;
    for (int rt = 8; rt <= (a.R > 8 ? 16 : 8); rt += 8) {
        const TileCost& cost = TILE_COST[di][rt / 16];
        const int W = plan_warps(dims, rt / 8);
        const int64_t row_tiles = up_div(a.R, rt), ctas = a.problems * row_tiles, useful = up_div(n_chunks, W);
        const int64_t fit = KV_SMS / ctas, most = useful < fit ? useful : fit;
        auto offer = [&](int64_t splits, bool cluster, float join) {
            const int64_t waves = up_div(ctas * splits, KV_SMS);
            const float t = join + waves * (cost.base + cost.chunk * up_div(up_div(n_chunks, splits), W));
            if (t >= best) return;
            best = t;
            a.tile_rows = rt;
            a.row_tiles = (int)row_tiles;
            a.splits = (int)splits;
            a.cluster = cluster;
        };
        // the weights of a call that accumulates are added by the cluster if one tile has all rows of a KV head
        const bool joins = !a.logits || row_tiles == 1;
        offer(1, joins, joins ? 0.f : second);
        if (joins && ctas * 2 <= CLUSTERED_CTAS) offer(2, true, 1.2f);
        if (joins && ctas * 4 <= CLUSTERED_CTAS) offer(4, true, 1.2f);
        if (most > 1) offer(most, false, second);
    }
    if (a.logits || a.list || a.R <= TC_MIN_R || di == 2) return;
    // one CTA per SM over KV heads and tiles of 128 query rows, two tiles of cache rows each at least
    const int64_t tiles = up_div(past_rows, 64) + 1, ctas = a.problems * up_div(a.R, 128);
    int64_t splits = KV_SMS / ctas;
    if (splits > up_div(tiles, 2)) splits = up_div(tiles, 2);
    if (splits < 1) splits = 1;
    const float t = TC_COST[di].base + rows * (1.f / 256) + TC_COST[di].chunk * up_div(tiles, splits) * up_div(ctas * splits, KV_SMS);
    if (t < best) a.tc_splits = a.splits = (int)splits;
}

cudaError_t launch_cache_attention(const CacheAttn& a, cudaStream_t s) {
    const cudaError_t e = a.tc_splits ? launch_cache_attention_tc(a, s)
                          : a.bf16    ? attention_type<__nv_bfloat16>(a, s)
                                      : attention_type<__half>(a, s);
    if (e != cudaSuccess || (a.tc_splits ? a.splits == 1 : a.cluster)) return e;
    const int rows = a.n_past_dev ? a.max_rows : a.n_past + a.m;
    const int per = (rows + ACC_ROWS - 1) / ACC_ROWS;                  // accumulating CTAs of a KV head
    const int n_rows = a.problems * a.R;
    const int col_shift = a.hd % 64 || n_rows > KV_SMS || a.hd == 192 ? 0 : a.hd / 128;     // blocks of 64 dims
    const int v4 = a.hd / 4 >> col_shift;
    const unsigned v4_inv = (65536 + v4 - 1) / v4;     // exact for x <= 256: x * (v4 - 1) < 65536
    return launch_pdl(k_cache_combine, dim3((a.R << col_shift) + (a.logits ? per : 0), a.problems), CB, 0, s, a,
                      cache_tile_dims(a.hd), col_shift, v4, v4_inv);
}

}  // namespace hoard
