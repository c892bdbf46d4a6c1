// kernels_cache_tc.cu -- attention of many query rows over the past rows of a KV cache on the 5th-generation
// tensor cores (tcgen05, accumulators and one operand in tensor memory).
//
//   S[128 query rows x 64 keys] = Q K^T,  P = 2^(S - M),  O[128 x head_dim] += P V
//
// A CTA takes 128 query rows of a KV head and a share of the cache's past rows in tiles of 64. Q, as its two f16 or
// three bf16 terms (see kernels_cache.cu for the precision), stays in tensor memory for the whole CTA; a tile's
// K and V come to shared memory as they lie in the cache and are operands as they are: K as the K-major B of S,
// V as the MN-major B of O. S is read by the softmax threads, one query row per thread, and P's terms are written back
// over it as the A operand of the second product. Roles of the 384 threads:
//   warp 0       one thread issues the products
//   warps 1-3    copy K and V tiles into a ring (cp.async, rows past the end as zeros)
//   warps 4-7, 8-11   two softmax groups, even and odd tiles: each has its own running maximum, total and f32 sums
//                (head_dim registers per thread) and the two are joined at the end.
// The products of one group's tile run while the other group works on its own: PV(j), S(j+2), PV(j+1), S(j+3), ..
// The tensor cores truncate as they accumulate, so a tile's O leaves tensor memory after every tile and is added
// with rounding, sums scaled to a risen maximum in the same multiply-add.
// The tokens' own rows, with their masks, are another split's work (k_cache_attention); k_cache_combine joins all.
// Every wait is bounded; a CTA whose wait ran out reports totals of NaN, which reach the output.
#include "common.cuh"
#include "kernels_cache.h"
#include "async_copy.cuh"
#include "kv_terms.cuh"

namespace hoard {

namespace {

constexpr int TM = 128, TK = 64;                       // query rows, keys of a tile
constexpr int TC_THREADS = 384, LOADERS = 96, GROUP = 128;
constexpr int Q_PITCH_PAD = 1;                         // floats added to a staged q row

__device__ __forceinline__ bool wait_or_give_up(uint64_t* bar, unsigned parity, volatile int* give_up) {
    if (mbar_try_wait(bar, parity)) return !*give_up;
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
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// D[128 x N] (+)= A (tensor memory) * B (shared memory)
__device__ __forceinline__ void tc_mma(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, bool add) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
                 ::"r"(d), "r"(a), "l"(b_desc), "r"(idesc), "r"((uint32_t)add) : "memory");
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
    static_assert(Q_OFF + TM * (HD + Q_PITCH_PAD) * 4 <= RING, "staged q over the ring's later stages");
    static_assert(TM * (HD + 4) * 4 <= RING, "join buffer");
    // tensor memory, in columns: Q terms, two tiles of S (P's terms over it), O
    static constexpr int Q_COLS = HD / 2, P_COLS = TK / 2;
    static constexpr int SP = TN * P_COLS > TK ? TN * P_COLS : TK;
    static constexpr int C_Q = 0, C_S = TN * Q_COLS, C_O = C_S + 2 * SP;
    static_assert(C_O + HD <= 512, "tensor memory");
};

template <typename KT, int HD>
__global__ void __launch_bounds__(TC_THREADS, 1) k_cache_attention_tc(const CacheAttn a) {
    using P = TcPlan<KT, HD>;
    constexpr int TN = P::TN, ST = P::STAGES;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[ST], empty[ST], s_full[2], p_full[2], o_full[2], o_empty, q_full, done;
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_give_up;
    __shared__ float s_scale[TM], s_mx[TM], s_tot[TM];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = blockIdx.x, tile = blockIdx.y, kv = blockIdx.z;

    if (tid == 0) {
        for (int i = 0; i < ST; ++i) {
            mbar_init(&full[i], LOADERS);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], GROUP);
            mbar_init(&o_full[i], 1);
        }
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
    const uint32_t tmem = s_tmem;
    const int n_past = a.n_past_dev ? max(0, min(*a.n_past_dev, a.max_rows - a.m)) : a.n_past;
    const int n_tiles = (n_past + TK - 1) / TK;
    const int t_first = (int)((int64_t)n_tiles * split / a.tc_splits), t_end = (int)((int64_t)n_tiles * (split + 1) / a.tc_splits);
    const int T = t_end - t_first;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 0) {
            if (lane == 0 && T > 0) {
                bool ok = wait_or_give_up(&q_full, 0, &s_give_up);
                tc_after();
                auto score = [&](int j) {              // S(j) = Q K(j)^T into buffer j & 1
                    if (!ok || !(ok = wait_or_give_up(&full[j % ST], (j / ST) & 1, &s_give_up))) return;
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    tc_after();
                    const uint32_t kt = smem_u32(smem) + (j % ST) * P::STAGE, d = tmem + P::C_S + (j & 1) * P::SP;
#pragma unroll
                    for (int u = TN - 1; u >= 0; --u)
#pragma unroll
                        for (int k = 0; k < HD / 16; ++k)
                            tc_mma(d, tmem + P::C_Q + u * P::Q_COLS + 8 * k,
                                   desc_sw128(kt + (k >> 2) * P::SUB + (k & 3) * 32, 16), tc_idesc<KT>(TK, false),
                                   u != TN - 1 || k != 0);
                    tc_commit(&s_full[j & 1]);
                };
                score(0);
                if (T > 1) score(1);
                for (int j = 0; j < T && ok; ++j) {
                    ok = wait_or_give_up(&p_full[j & 1], (j >> 1) & 1, &s_give_up) &&
                         (j == 0 || wait_or_give_up(&o_empty, (j - 1) & 1, &s_give_up));
                    if (!ok) break;
                    tc_after();
                    const uint32_t vt = smem_u32(smem) + (j % ST) * P::STAGE + (HD / 64) * P::SUB;
#pragma unroll
                    for (int u = TN - 1; u >= 0; --u)
#pragma unroll
                        for (int k = 0; k < TK / 16; ++k)
                            tc_mma(tmem + P::C_O, tmem + P::C_S + (j & 1) * P::SP + u * P::P_COLS + 8 * k,
                                   desc_sw128(vt + k * 2048, P::SUB), tc_idesc<KT>(HD, true), u != TN - 1 || k != 0);
                    tc_commit(&o_full[j & 1]);
                    tc_commit(&empty[j % ST]);
                    if (j + 2 < T) score(j + 2);
                }
                // nothing of this thread's is in flight when tensor memory is freed
                tc_commit(&done);
                const unsigned long long t0 = gtimer();
                while (!mbar_try_wait(&done, 0) && gtimer() - t0 < WAIT_NS) {}
            }
            __syncwarp();
        } else {
            // ---- K and V tiles: 16-byte pieces, consecutive threads on consecutive pieces of a row ----
            const int lt = tid - 32;
            constexpr int C16 = HD / 8;                // pieces of a row
            const char* kb = reinterpret_cast<const char*>(a.kc) + (int64_t)kv * a.hs * 2;
            const char* vb = reinterpret_cast<const char*>(a.vc) + (int64_t)kv * a.hs * 2;
            bool ok = true;
            for (int j = 0; j < T && ok; ++j) {
                if (j == P::FIRST) named_sync(1, LOADERS + 2 * GROUP);           // q has left the later stages
                if (j >= ST && !(ok = wait_or_give_up(&empty[j % ST], (j / ST - 1) & 1, &s_give_up))) break;
                const int row0 = (t_first + j) * TK;
                const uint32_t dst = smem_u32(smem) + (j % ST) * P::STAGE;
#pragma unroll 4
                for (int i = lt; i < TK * C16; i += LOADERS) {
                    const int r = i / C16, c = i - r * C16;
                    const bool there = row0 + r < n_past && c * 8 < a.hd;
                    const int64_t off = there ? (int64_t)(row0 + r) * a.rs * 2 + c * 16 : 0;
                    const uint32_t o = (c >> 3) * P::SUB + r * 128 + (((c & 7) ^ (r & 7)) << 4);
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + o), "l"(kb + off),
                                 "r"(there ? 16 : 0) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + (HD / 64) * P::SUB + o),
                                 "l"(vb + off), "r"(there ? 16 : 0) : "memory");
                }
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[j % ST])) : "memory");
            }
            if (T <= P::FIRST) named_sync(1, LOADERS + 2 * GROUP);
            cp_async_wait_all();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        const int grp = (warp - 4) >> 2, row = tid - GROUP - grp * GROUP;        // this thread's query row
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        // ---- q: rows scaled by a power of two, staged, then this thread's row (half of the dims) as terms ----
        float* sq = reinterpret_cast<float*>(smem + P::Q_OFF);
        constexpr int QP = HD + Q_PITCH_PAD;
        for (int i0 = 0; i0 < TM / 8; i0 += 4) {
            float x[4][HD / 32];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = (warp - 4) * (TM / 8) + i0 + i, g = tile * TM + r;
                const bool live = g < a.R;
                const float* q = a.q + (live ? g / a.g : 0) * a.q_ts + (kv * a.g + (live ? g % a.g : 0)) * a.q_hs;
#pragma unroll
                for (int k = 0; k < HD / 32; ++k) x[i][k] = live && k * 32 + lane < a.hd ? q[k * 32 + lane] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = (warp - 4) * (TM / 8) + i0 + i;
                float am = 0.f;
                bool bad = false;
#pragma unroll
                for (int k = 0; k < HD / 32; ++k) {
                    bad |= !(fabsf(x[i][k]) <= 3.4e38f);
                    am = fmaxf(am, fabsf(x[i][k]));
                }
                const RowScale rs = row_scale<KT>(warp_max(am), __any_sync(0xffffffffu, bad));
                if (lane == 0) s_scale[r] = a.scale_log2 * rs.down;
#pragma unroll
                for (int k = 0; k < HD / 32; ++k) sq[r * QP + k * 32 + lane] = x[i][k] * rs.up;
            }
        }
        named_sync(2, 2 * GROUP);
        if (grp * 64 < HD) {
            uint32_t w[TN][32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                float lo = sq[row * QP + grp * 64 + 2 * i], hi = sq[row * QP + grp * 64 + 2 * i + 1];
#pragma unroll
                for (int u = 0; u < TN; ++u) w[u][i] = take_term<KT>(lo, hi);
            }
#pragma unroll
            for (int u = 0; u < TN; ++u) tc_st32(tmem + lanes + P::C_Q + u * P::Q_COLS + grp * 32, w[u]);
            tc_st_wait();
        }
        tc_before();
        mbar_arrive(&q_full);
        named_sync(1, LOADERS + 2 * GROUP);
        const float sc = s_scale[row];

        float acc[HD];
#pragma unroll
        for (int i = 0; i < HD; ++i) acc[i] = 0.f;
        float mx = -INFINITY, tot = 0.f;
        bool ok = true;
        // a warp goes on or gives up as a whole: what follows is collective
        auto group_wait = [&](uint64_t* bar, unsigned parity) {
            return __all_sync(0xffffffffu, wait_or_give_up(bar, parity, &s_give_up)) != 0;
        };
        for (int j = grp; j < T; j += 2) {
            if (!(ok = group_wait(&s_full[grp], (j >> 1) & 1))) break;
            tc_after();
            const uint32_t sp = tmem + lanes + P::C_S + grp * P::SP;
            uint32_t sr[TK];
            tc_ld32(sp, sr);
            tc_ld32(sp + 32, sr + 32);
            tc_ld_wait();
            const int left = n_past - (t_first + j) * TK;                       // keys of the tile that exist
            if (left < TK) {
#pragma unroll
                for (int i = 0; i < TK; ++i)
                    if (i >= left) sr[i] = 0xFF800000u;                         // -inf
            }
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < TK; ++i) top = fmaxf(top, __uint_as_float(sr[i]));
            top = fmaxf(mx, top * sc);
            const float f = top > mx ? ex2f(mx - top) : 1.f;
            const float b = Terms<KT>::P_EXP - (top == -INFINITY ? 0.f : top);
            mx = top;
            float sum = 0.f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t w[TN][16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float p0 = ex2f(fmaf(__uint_as_float(sr[32 * h + 2 * i]), sc, b));
                    float p1 = ex2f(fmaf(__uint_as_float(sr[32 * h + 2 * i + 1]), sc, b));
                    sum += p0 + p1;
#pragma unroll
                    for (int u = 0; u < TN; ++u) w[u][i] = take_term<KT>(p0, p1);
                }
#pragma unroll
                for (int u = 0; u < TN; ++u) tc_st16(sp + u * P::P_COLS + 16 * h, w[u]);
            }
            tot = tot * f + sum;
            tc_st_wait();
            tc_before();
            mbar_arrive(&p_full[grp]);
            if (!(ok = group_wait(&o_full[grp], (j >> 1) & 1))) break;
            tc_after();
#pragma unroll
            for (int c = 0; c < HD; c += 32) {
                uint32_t r[32];
                tc_ld32(tmem + lanes + P::C_O + c, r);
                tc_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; ++i) acc[c + i] = fmaf(acc[c + i], f, __uint_as_float(r[i]));
            }
            tc_before();
            mbar_arrive(&o_empty);
        }
        if (!ok) tot = __int_as_float(0x7FC00000);     // a wait ran out: the total says so
        if (tot != tot && mx == -INFINITY) mx = 0.f;
        // ---- join the groups: the odd tiles' sums through shared memory (the ring is idle now) ----
        float* joined = reinterpret_cast<float*>(smem);
        constexpr int JP = HD + 4;                     // floats of a row
        named_sync(2, 2 * GROUP);                      // both groups have seen their last tile's products complete
        if (grp == 1) {
            s_mx[row] = mx;
            s_tot[row] = tot;
#pragma unroll
            for (int c = 0; c < HD; c += 4)
                *reinterpret_cast<float4*>(joined + row * JP + c) = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
        }
        named_sync(2, 2 * GROUP);
        if (grp == 0) {
            const float m1 = s_mx[row], l1 = s_tot[row], top = fmaxf(mx, m1);
            const float f0 = mx == -INFINITY ? 0.f : ex2f(mx - top), f1 = m1 == -INFINITY ? 0.f : ex2f(m1 - top);
            const int g = tile * TM + row;
            if (g < a.R) {
                const int64_t part = ((int64_t)kv * a.splits + split) * a.R + g;
                a.part_ml[part] = make_float2(top, (mx == -INFINITY ? 0.f : tot * f0) + (m1 == -INFINITY ? 0.f : l1 * f1));
#pragma unroll
                for (int c = 0; c < HD; c += 4) {
                    const float4 u = *reinterpret_cast<const float4*>(joined + row * JP + c);
                    *reinterpret_cast<float4*>(a.part_o + part * HD + c) =
                        make_float4(acc[c] * f0 + u.x * f1, acc[c + 1] * f0 + u.y * f1, acc[c + 2] * f0 + u.z * f1,
                                    acc[c + 3] * f0 + u.w * f1);
                }
            }
        }
    }
    tc_before();
    __syncthreads();
    tc_after();
    if (warp == 0)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

template <typename KT, int HD> cudaError_t tc_go(const CacheAttn& a, cudaStream_t s) {
    constexpr int smem = TcPlan<KT, HD>::RING + 1024;
    static SmemLimit limit;
    const cudaError_t e = limit.raise((const void*)k_cache_attention_tc<KT, HD>, smem);
    if (e != cudaSuccess) return e;
    return launch_pdl(k_cache_attention_tc<KT, HD>, dim3(a.tc_splits, (a.R + TM - 1) / TM, a.n_kv), TC_THREADS, smem, s, a);
}

}  // namespace

cudaError_t launch_cache_attention_tc(const CacheAttn& a, cudaStream_t s) {
    if (cache_tile_dims(a.hd) == 64) return a.bf16 ? tc_go<__nv_bfloat16, 64>(a, s) : tc_go<__half, 64>(a, s);
    return a.bf16 ? tc_go<__nv_bfloat16, 128>(a, s) : tc_go<__half, 128>(a, s);
}

}  // namespace hoard
