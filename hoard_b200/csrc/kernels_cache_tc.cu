// kernels_cache_tc.cu -- attention of many query rows over a KV cache on the 5th-generation
// tensor cores (tcgen05, accumulators and one operand in tensor memory).
//
//   S[128 query rows x 64 keys] = Q K^T,  P = 2^(S - M),  O[128 x head_dim] += P V
//
// A CTA takes 128 query rows of a KV head and a share of the cache's rows in tiles of 64. Q, as its two f16 or
// three bf16 terms (see kernels_cache.cu for the precision), stays in tensor memory for the whole CTA; a tile's
// K and V come to shared memory as they lie in the cache and are operands as they are: K as the K-major B of S,
// V as the MN-major B of O. S is read by the softmax threads, one query row per thread, and P's terms are written back
// over it as the A operand of the second product. Roles of the 384 threads:
//   warp 0       issues the products
//   warps 1-3    copy K and V tiles into a ring (cp.async, rows past the end as zeros)
//   warps 4-7, 8-11   two softmax groups, even and odd tiles: each has its own running maximum, total and f32 sums
//                (head_dim registers per thread) and the two are joined at the end.
// The products of one group's tile run while the other group works on its own: PV(j), S(j+NSB), PV(j+1), .. Three
// tiles of S are in flight for f16 (two for bf16, whose terms leave no room), so that a group finds its next scores
// ready; the tile of a steady state took 1500 cycles with two and 1170 are the products'.
// The tensor cores truncate as they accumulate, so a tile's O leaves tensor memory after every tile and is added
// with rounding, sums scaled to a risen maximum in the same multiply-add.
// The last tile is the tokens' own rows, with their masks. k_cache_combine joins the splits.
// Bound by power in long calls: 64 tokens of 8 heads x 4 KV heads over 131008 rows are 2 x 137 GFLOP in 240 us, 1.14 PFLOP/s of
// products, and 275 when repeated (the clock falls to 1.4 GHz). In short ones by what does not depend on the cache's length:
// tensor memory, q staged and split, the first tile, the end, 10 us together.
// Every wait is bounded; a CTA whose wait ran out reports totals of NaN, which reach the output.
#include "common.cuh"
#include "kernels_cache.h"
#include "async_copy.cuh"
#include "kv_terms.cuh"

#include <type_traits>

namespace hoard {

namespace {

constexpr int TM = 128, TK = 64;                       // query rows, keys of a tile
constexpr int TC_THREADS = 384, LOADERS = 96, GROUP = 128;
constexpr float LARGE_SCORE = 1 << 20;                 // steps of f32 up to there: 2^-4
constexpr int Q_PAD = 4;                               // floats added to a staged q row: rows start in other banks

__device__ __forceinline__ bool wait_or_give_up(uint64_t* bar, unsigned parity, volatile int* give_up) {
    if (mbar_try_wait(bar, parity)) return true;
    const unsigned long long t0 = gtimer();
    while (!mbar_try_wait(bar, parity)) {
        if (*give_up) return false;
        if (gtimer() - t0 > WAIT_NS) {
            *give_up = 1;
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Issued by the whole warp with one lane elected, so that the operands stay in uniform registers.
__device__ __forceinline__ uint32_t elect_lane() {
    uint32_t e;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(e));
    return e;
}
__device__ __forceinline__ void tc_commit(uint64_t* bar, uint32_t elected) {
    asm volatile("{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
                 " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n"
                 ::"r"(smem_u32(bar)), "r"(elected) : "memory");
}
// D[128 x N] (+)= A (tensor memory) * B (shared memory)
__device__ __forceinline__ void tc_mma(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, bool add,
                                       uint32_t elected) {
    asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
                 " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
                 ::"r"(d), "r"(a), "l"(b_desc), "r"(idesc), "r"((uint32_t)add), "r"(elected) : "memory");
}
// 32 consecutive columns of this warp's 32 lanes: thread = lane, register = column
__device__ __forceinline__ void tc_ld32(uint32_t addr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
                   "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
                   "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
                   "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr));
}
__device__ __forceinline__ uint32_t tc_ld1(uint32_t addr) {
    uint32_t r;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n tcgen05.wait::ld.sync.aligned;" : "=r"(r) : "r"(addr) : "memory");
    return r;
}
__device__ __forceinline__ void tc_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_st32(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
                 "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
                   "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
                   "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
                 : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tc_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory descriptors of 128B-swizzled operands (rows of 128 bytes, eight-row atoms of 1024 bytes, version 1):
// K-major (K): stride between eight-row groups 1024, the leading offset unused. MN-major (V: rows are keys, the
// dims of a row contiguous): stride between eight-key groups 1024, leading offset between blocks of 64 dims.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr, uint32_t lead_bytes) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(lead_bytes >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
// Instruction descriptor: D f32, A and B of the cache's type, M = 128, N, B MN-major or K-major
template <typename KT> constexpr uint32_t tc_idesc(int n, bool b_mn) {
    const uint32_t ty = Terms<KT>::N == 2 ? 0u : 1u;   // f16 : bf16
    return (1u << 4) | (ty << 7) | (ty << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(TM >> 4) << 24);
}

template <typename KT, int HD> struct TcPlan {
    static constexpr int TN = Terms<KT>::N;
    static constexpr int SUB = TK * 128;               // bytes of 64 keys x 64 dims
    static constexpr int STAGE = 2 * (HD / 64) * SUB;  // K, then V
    static constexpr int STAGES = HD == 128 ? 6 : 8;
    static constexpr int FIRST = 3;                    // stages that are filled while q is staged over the others
    static constexpr int Q_OFF = FIRST * STAGE;
    static constexpr int RING = STAGES * STAGE;
    static_assert(Q_OFF + TM * (HD + Q_PAD) * 4 <= RING, "staged q over the ring's later stages");
    static_assert(TM * (HD + 4) * 4 <= RING, "join buffer");
    // tensor memory, in columns: Q terms, tiles of S (P's terms over it; what fits beside the other two), O
    static constexpr int NSB = TN == 2 ? 3 : 2;
    static constexpr int Q_COLS = HD / 2, P_COLS = TK / 2;
    static constexpr int SP = TN * P_COLS > TK ? TN * P_COLS : TK;
    static constexpr int C_Q = 0, C_S = TN * Q_COLS, C_O = C_S + NSB * SP;
    static_assert(C_O + HD <= 512, "tensor memory");
};

// HD: dims of the layout; ND: dims of the products (96 of 128: 4 heads of 96, 64 tokens of 6 heads each over 100000 cache rows
// 123.9 us, 131.9 with all 128)
template <typename KT, int HD, int ND>
__global__ void __launch_bounds__(TC_THREADS, 1) k_cache_attention_tc(const CacheAttn a) {
    using P = TcPlan<KT, HD>;
    constexpr int TN = P::TN, ST = P::STAGES, NSB = P::NSB;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[ST], empty[ST], s_full[NSB], p_full[NSB], o_full[2], o_empty, q_full, done;
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_give_up;
    __shared__ float s_mx[2][TM], s_tot[2][TM];
    __shared__ int64_t s_q[TM];                        // a query row's offset in q, its (token, head) index
    __shared__ int s_o[TM];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int split = blockIdx.x, tile = blockIdx.y, kv = blockIdx.z;

    if (tid == 0) {
        for (int i = 0; i < ST; ++i) {
            mbar_init(&full[i], LOADERS);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < NSB; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], GROUP);
        }
        for (int i = 0; i < 2; ++i) mbar_init(&o_full[i], 1);
        mbar_init(&o_empty, GROUP);
        mbar_init(&q_full, 2 * GROUP);
        mbar_init(&done, 1);
        s_give_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    pdl_enter();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    const int n_past = __shfl_sync(0xffffffffu, a.n_past_dev ? max(0, min(*a.n_past_dev, a.max_rows - a.m)) : a.n_past, 0);
    const int n_tiles = (n_past + TK - 1) / TK + 1;    // the last: the tokens' own rows
    const Share share(n_tiles, a.tc_splits);
    const int t_first = share.first(split), T = share.first(split + 1) - t_first;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 0) {
            if (T > 0) {
                const uint32_t elected = elect_lane(), ring = smem_u32(smem);
                // the warp goes on or gives up as a whole
                auto wait = [&](uint64_t* bar, unsigned parity) {
                    return __all_sync(0xffffffffu, wait_or_give_up(bar, parity, &s_give_up)) != 0;
                };
                bool ok = wait(&q_full, 0);
                tc_after();
                int st_s = 0, ph_s = 0, st_o = 0;      // ring stages of the next S and the next O
                auto score = [&](int b) {              // S = Q K^T of the next tile into buffer b
                    if (!ok || !(ok = wait(&full[st_s], ph_s))) return;
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    tc_after();
                    const uint32_t kt = ring + st_s * P::STAGE, d = tmem + P::C_S + b * P::SP;
                    const uint64_t kd = desc_sw128(kt, 16);
#pragma unroll
                    for (int u = TN - 1; u >= 0; --u)
#pragma unroll
                        for (int k = 0; k < ND / 16; ++k)
                            tc_mma(d, tmem + P::C_Q + u * P::Q_COLS + 8 * k,
                                   kd + (((k >> 2) * P::SUB + (k & 3) * 32) >> 4), tc_idesc<KT>(TK, false),
                                   u != TN - 1 || k != 0, elected);
                    tc_commit(&s_full[b], elected);
                    if (++st_s == ST) {
                        st_s = 0;
                        ph_s ^= 1;
                    }
                };
                for (int j = 0; j < NSB && j < T; ++j) score(j);
                int b = 0, ph_b = 0;                   // buffer of S(j), the phase of its uses
                for (int j = 0; j < T && ok; ++j) {
                    ok = wait(&p_full[b], ph_b) && (j == 0 || wait(&o_empty, (j - 1) & 1));
                    if (!ok) break;
                    tc_after();
                    const uint64_t vd = desc_sw128(ring + st_o * P::STAGE + (HD / 64) * P::SUB, P::SUB);
#pragma unroll
                    for (int u = TN - 1; u >= 0; --u)
#pragma unroll
                        for (int k = 0; k < TK / 16; ++k)
                            tc_mma(tmem + P::C_O, tmem + P::C_S + b * P::SP + u * P::P_COLS + 8 * k, vd + (k * 2048 >> 4),
                                   tc_idesc<KT>(ND, true), u != TN - 1 || k != 0, elected);
                    tc_commit(&o_full[j & 1], elected);
                    tc_commit(&empty[st_o], elected);
                    if (++st_o == ST) st_o = 0;
                    if (j + NSB < T) score(b);
                    if (++b == NSB) {
                        b = 0;
                        ph_b ^= 1;
                    }
                }
                // nothing of this warp's is in flight when tensor memory is freed
                tc_commit(&done, elected);
                const unsigned long long t0 = gtimer();
                while (!mbar_try_wait(&done, 0) && gtimer() - t0 < WAIT_NS) {}
            }
            __syncwarp();
        } else {
            // ---- K and V tiles: 16-byte pieces, consecutive threads on consecutive pieces of a row ----
            constexpr int C16 = HD / 8, STEP = LOADERS / C16;        // pieces of a row, rows of one round
            const int lt = tid - 32, c = lt % C16, r0 = lt / C16;
            const int64_t step = (int64_t)STEP * a.rs * 2;
            const int64_t at0 = ((int64_t)r0 * a.rs + (int64_t)kv * a.hs) * 2 + c * 16;
            const bool dim = c * 8 < a.hd;
            const uint32_t dst0 = smem_u32(smem) + (c >> 3) * P::SUB;
            int stage = 0, phase = 1;                  // phase of `empty` to wait for (the first round passes)
            bool ok = true;
            for (int j = 0; j < T && ok; ++j) {
                if (j == P::FIRST) named_sync(1, LOADERS + 2 * GROUP);           // q has left the later stages
                if (j >= ST && !(ok = wait_or_give_up(&empty[stage], phase, &s_give_up))) break;
                const uint32_t dst = dst0 + stage * P::STAGE;
                const bool own = t_first + j == n_tiles - 1;
                const int row0 = own ? n_past : (t_first + j) * TK;
                const int left = own ? a.m : n_past - row0;                     // rows of the tile that exist
                const char* kp = static_cast<const char*>(a.kc) + at0 + (int64_t)row0 * a.rs * 2;
                const char* vp = static_cast<const char*>(a.vc) + at0 + (int64_t)row0 * a.rs * 2;
#pragma unroll
                for (int i = 0; i < (TK + STEP - 1) / STEP; ++i) {
                    const int r = r0 + i * STEP;
                    const uint32_t o = dst + r * 128 + (((c & 7) ^ (r & 7)) << 4);
                    if (r < TK) {
                        const bool there = dim && r < left;
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(o),
                                     "l"(there ? kp : static_cast<const char*>(a.kc)), "r"(there ? 16 : 0) : "memory");
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(o + (HD / 64) * P::SUB),
                                     "l"(there ? vp : static_cast<const char*>(a.vc)), "r"(there ? 16 : 0) : "memory");
                    }
                    kp += step;
                    vp += step;
                }
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[stage])) : "memory");
                if (++stage == ST) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            if (T <= P::FIRST) named_sync(1, LOADERS + 2 * GROUP);
            cp_async_wait_all();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        const int grp = (warp - 4) >> 2, row = tid - GROUP - grp * GROUP;        // this thread's query row
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        // ---- q: rows staged as they are, each row's largest magnitude, then the row as scaled terms. The two groups
        // take half of a row's dims each ----
        float* sq = reinterpret_cast<float*>(smem + P::Q_OFF);
        constexpr int QP = HD + Q_PAD, V4 = HD / 4, ROUND = 2 * GROUP / V4;      // rows that the threads copy at once
        const int gt = tid - GROUP, col = 4 * (gt % V4), rows = min(TM, a.R - tile * TM);
        if (grp == 0) {                                // query row -> token and head, once per row
            const int g = tile * TM + min(row, rows - 1), t = g / a.g, h = kv * a.g + (g - t * a.g);
            s_q[row] = t * a.q_ts + h * a.q_hs;
            s_o[row] = t * a.n_head + h;
        }
        named_sync(2, 2 * GROUP);
        {
            const bool wide = ((reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)(a.q_ts * 4) | (uintptr_t)(a.q_hs * 4)) & 15) == 0;
#pragma unroll
            for (int i = 0; i < TM / ROUND; ++i) {
                const int r = gt / V4 + i * ROUND;
                const bool live = r < rows && col < a.hd;
                const float* q = a.q + (live ? s_q[r] + col : 0);
                const uint32_t dst = smem_u32(sq + r * QP + col);
                if (wide) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(q), "r"(live ? 16 : 0) : "memory");
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + 4 * k), "l"(live ? q + k : q),
                                     "r"(live ? 4 : 0) : "memory");
                }
            }
            cp_async_commit();
            cp_async_wait_all();
        }
        named_sync(2, 2 * GROUP);
        constexpr int HALF = HD / 2;
        float4 xq[HALF / 4];
        {
            float am = 0.f, odd = 0.f;                 // NaN where the row has an infinity or NaN
#pragma unroll
            for (int i = 0; i < HALF / 4; ++i) {
                const float4 x = xq[i] = *reinterpret_cast<const float4*>(sq + row * QP + grp * HALF + 4 * i);
                am = fmaxf(am, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
                odd = fmaf(x.x, 0.f, fmaf(x.y, 0.f, fmaf(x.z, 0.f, fmaf(x.w, 0.f, odd))));
            }
            s_mx[grp][row] = odd == 0.f ? am : INFINITY;
        }
        named_sync(2, 2 * GROUP);
        const float am = fmaxf(s_mx[0][row], s_mx[1][row]);
        const RowScale rs = row_scale<KT>(am, am == INFINITY);
        // a factor that vanishes (a tiny scale beside a row that was scaled up) must not make NaN of a masked -inf; scores vanish
        // as well with the least normal number
        const float sc = fmaxf(a.scale_log2 * rs.down, rs.down < 1.f ? 1.17549435e-38f : 0.f);
#pragma unroll
        for (int h = 0; h < HALF; h += 32) {           // 32 dims are 16 columns
            uint32_t w[TN][16];
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float4 x = xq[(h + 2 * i) / 4];
                float v[4] = {x.x * rs.up, x.y * rs.up, x.z * rs.up, x.w * rs.up};
#pragma unroll
                for (int u = 0; u < TN; ++u) {
                    w[u][i] = take_term<KT>(v[0], v[1]);
                    w[u][i + 1] = take_term<KT>(v[2], v[3]);
                }
            }
#pragma unroll
            for (int u = 0; u < TN; ++u) tc_st16(tmem + lanes + P::C_Q + u * P::Q_COLS + (grp * HALF + h) / 2, w[u]);
        }
        tc_st_wait();
        tc_before();
        mbar_arrive(&q_full);
        named_sync(1, LOADERS + 2 * GROUP);
        // which own rows this thread's query row sees
        uint64_t vis = 0;
        if (tile * TM + row < a.R) {
            const int t = (tile * TM + row) / a.g;
            vis = a.vis ? a.vis[t] : t >= 63 ? ~0ull : (1ull << (t + 1)) - 1;
            if (a.m < 64) vis &= (1ull << a.m) - 1;
        }

        float acc[ND];
#pragma unroll
        for (int i = 0; i < ND; ++i) acc[i] = 0.f;
        float mx = -INFINITY, tot = 0.f;
        bool ok = true;
        // a warp goes on or gives up as a whole: what follows is collective
        auto group_wait = [&](uint64_t* bar, unsigned parity) {
            return __all_sync(0xffffffffu, wait_or_give_up(bar, parity, &s_give_up)) != 0;
        };
        for (int j = grp; j < T; j += 2) {
            const int buf = j % NSB;
            if (!(ok = group_wait(&s_full[buf], (j / NSB) & 1))) break;
            tc_after();
            const uint32_t sp = tmem + lanes + P::C_S + buf * P::SP;
            uint32_t sr[TK];
            tc_ld32(sp, sr);
            tc_ld32(sp + 32, sr + 32);
            tc_ld_wait();
            const bool own = t_first + j == n_tiles - 1;
            const int left = n_past - (t_first + j) * TK;                       // past keys of the tile that exist
            if (own || left < TK) {
                const uint64_t sees = own ? vis : (1ull << left) - 1;
#pragma unroll
                for (int i = 0; i < TK; ++i)
                    if (!(sees >> i & 1)) sr[i] = 0xFF800000u;                  // -inf
            }
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < TK; ++i) top = fmaxf(top, __uint_as_float(sr[i]));
            top = fmaxf(mx, __fmul_rn(top, sc));
            const float f = top > mx ? ex2f(mx - top) : 1.f;
            // weights 2^(s sc - top + P_EXP), their exponents by one multiply-add each. Where the roundings of s sc and of top
            // may come to more than 2^-4, s sc - top is formed first, in the order that makes the largest weight 2^P_EXP exactly
            const float base = top == -INFINITY ? 0.f : top;
            float mul = sc, add = Terms<KT>::P_EXP - base;
            if (__any_sync(0xffffffffu, fabsf(base) > LARGE_SCORE)) {
#pragma unroll
                for (int i = 0; i < TK; ++i)
                    sr[i] = __float_as_uint(__fsub_rn(__fmul_rn(__uint_as_float(sr[i]), sc), base));
                mul = 1.f;
                add = Terms<KT>::P_EXP;
            }
            mx = top;
            float sum = 0.f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t w[TN][16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float p0 = ex2f(fmaf(__uint_as_float(sr[32 * h + 2 * i]), mul, add));
                    float p1 = ex2f(fmaf(__uint_as_float(sr[32 * h + 2 * i + 1]), mul, add));
                    sum += p0 + p1;
#pragma unroll
                    for (int u = 0; u < TN; ++u) w[u][i] = take_term<KT>(p0, p1);
                }
#pragma unroll
                for (int u = 0; u < TN; ++u) tc_st16(sp + u * P::P_COLS + 16 * h, w[u]);
            }
            tot = tot * f + sum;
            tc_st_wait();
            // masked own rows may hold infinities or NaN (0 * inf): that tile's products are then taken one by one
            bool odd = false;
            if (own) {
                const uint8_t* vt = smem + (j % ST) * P::STAGE + (HD / 64) * P::SUB;
                uint32_t any = 0;
                for (int i = lane; i < HD / 64 * P::SUB / 16; i += 32) {         // each warp for itself
                    const uint4 v = *reinterpret_cast<const uint4*>(vt + 16 * i);
                    any |= odd_pair<KT>(v.x) | odd_pair<KT>(v.y) | odd_pair<KT>(v.z) | odd_pair<KT>(v.w);
                }
                odd = __any_sync(0xffffffffu, any != 0);
            }
            if (odd) {
                // two keys at a time, their weights put together again from the terms
#pragma unroll
                for (int i = 0; i < ND; ++i) acc[i] *= f;
                const uint8_t* vt = smem + (j % ST) * P::STAGE + (HD / 64) * P::SUB;
#pragma unroll 1
                for (int i = 0; i < a.m; i += 2) {
                    float p0 = 0.f, p1 = 0.f;
#pragma unroll
                    for (int u = TN - 1; u >= 0; --u) {
                        const uint32_t w = tc_ld1(sp + u * P::P_COLS + (i >> 1));
                        p0 += kv_lo<KT>(w);
                        p1 += kv_lo<KT>(w >> 16);
                    }
#pragma unroll
                    for (int c = 0; c < ND / 2; ++c) {
                        const uint32_t o = (c >> 5) * P::SUB + (c & 3) * 4, q = (c & 31) >> 2;
                        const uint32_t v0 = *reinterpret_cast<const uint32_t*>(vt + o + i * 128 + ((q ^ (i & 7)) << 4));
                        const uint32_t v1 = *reinterpret_cast<const uint32_t*>(vt + o + (i + 1) * 128 + ((q ^ ((i + 1) & 7)) << 4));
                        if (p0 != 0.f) {
                            acc[2 * c] += p0 * kv_lo<KT>(v0);
                            acc[2 * c + 1] += p0 * kv_lo<KT>(v0 >> 16);
                        }
                        if (p1 != 0.f) {
                            acc[2 * c] += p1 * kv_lo<KT>(v1);
                            acc[2 * c + 1] += p1 * kv_lo<KT>(v1 >> 16);
                        }
                    }
                }
            }
            tc_before();
            mbar_arrive(&p_full[buf]);
            if (!(ok = group_wait(&o_full[grp], (j >> 1) & 1))) break;
            tc_after();
            if (!odd) {
#pragma unroll
                for (int c = 0; c < ND; c += 32) {
                    uint32_t r[32];
                    tc_ld32(tmem + lanes + P::C_O + c, r);
                    tc_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) acc[c + i] = fmaf(acc[c + i], f, __uint_as_float(r[i]));
                }
            }
            tc_before();
            mbar_arrive(&o_empty);
        }
        if (!ok) tot = __int_as_float(0x7FC00000);     // a wait ran out: the total says so
        if (tot != tot && mx == -INFINITY) mx = 0.f;
        // ---- join the groups through shared memory (the ring is idle now): each hands the other half of its sums and
        // joins the half it keeps; then rows are stored by consecutive threads ----
        float* joined = reinterpret_cast<float*>(smem);
        constexpr int JP = HD + 4, JH = ND / 2;        // floats of a row, of a group's half
        named_sync(2, 2 * GROUP);                      // both groups have seen their last tile's products complete
        const bool whole = a.splits == 1;              // nothing to join with: the output itself
        s_mx[grp][row] = mx;
        s_tot[grp][row] = tot;
        auto hand = [&](auto first) {                  // columns [first, first + JH)
            constexpr int F = decltype(first)::value;
#pragma unroll
            for (int c = F; c < F + JH; c += 4)
                *reinterpret_cast<float4*>(joined + row * JP + c) = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
        };
        if (grp == 0) hand(std::integral_constant<int, JH>());
        else hand(std::integral_constant<int, 0>());
        named_sync(2, 2 * GROUP);
        const float m1 = s_mx[grp ^ 1][row], l1 = s_tot[grp ^ 1][row], top = fmaxf(mx, m1);
        const float f0 = mx == -INFINITY ? 0.f : ex2f(mx - top), f1 = m1 == -INFINITY ? 0.f : ex2f(m1 - top);
        const float l = (mx == -INFINITY ? 0.f : tot * f0) + (m1 == -INFINITY ? 0.f : l1 * f1);
        const float inv = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l;
        const int64_t part0 = ((int64_t)kv * a.splits + split) * a.R + tile * TM;
        if (!whole && grp == 0 && row < rows) a.part_ml[part0 + row] = make_float2(top, l);
        auto keep = [&](auto first) {
            constexpr int F = decltype(first)::value;
#pragma unroll
            for (int c = F; c < F + JH; c += 4) {
                float4* at = reinterpret_cast<float4*>(joined + row * JP + c);
                const float4 u = *at;
                *at = make_float4((acc[c] * f0 + u.x * f1) * inv, (acc[c + 1] * f0 + u.y * f1) * inv,
                                  (acc[c + 2] * f0 + u.z * f1) * inv, (acc[c + 3] * f0 + u.w * f1) * inv);
            }
        };
        if (grp == 0) keep(std::integral_constant<int, 0>());
        else keep(std::integral_constant<int, JH>());
        named_sync(2, 2 * GROUP);
#pragma unroll 4
        for (int r = gt / V4; r < rows; r += ROUND) {
            const float4 y = *reinterpret_cast<const float4*>(joined + r * JP + col);
            if (!whole) {
                *reinterpret_cast<float4*>(a.part_o + (part0 + r) * HD + col) = y;
            } else if (col < a.hd) {
                float v[4] = {y.x, y.y, y.z, y.w};
                if (a.gate) {
                    const int t = (tile * TM + r) / a.g, h = s_o[r] - t * a.n_head;
                    const float* gp = a.gate + t * a.gate_ts + h * a.gate_hs + col;
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[k] *= sigmoid_f(gp[k]);
                }
                store4(a.out + (int64_t)s_o[r] * a.hd + col, v);
            }
        }
    }
    tc_before();
    __syncthreads();
    tc_after();
    if (warp == 0)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

template <typename KT, int HD, int ND> cudaError_t tc_go(const CacheAttn& a, cudaStream_t s) {
    constexpr int smem = TcPlan<KT, HD>::RING + 1024;
    static SmemLimit limit;
    const cudaError_t e = limit.raise((const void*)k_cache_attention_tc<KT, HD, ND>, smem);
    if (e != cudaSuccess) return e;
    return launch_pdl(k_cache_attention_tc<KT, HD, ND>, dim3(a.tc_splits, (a.R + TM - 1) / TM, a.n_kv), TC_THREADS, smem, s, a);
}
template <typename KT> cudaError_t tc_type(const CacheAttn& a, cudaStream_t s) {
    return a.hd <= 64 ? tc_go<KT, 64, 64>(a, s) : a.hd <= 96 ? tc_go<KT, 128, 96>(a, s) : tc_go<KT, 128, 128>(a, s);
}

}  // namespace

cudaError_t launch_cache_attention_tc(const CacheAttn& a, cudaStream_t s) {
    return a.bf16 ? tc_type<__nv_bfloat16>(a, s) : tc_type<__half>(a, s);
}

}  // namespace hoard
