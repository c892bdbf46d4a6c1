// kernels_cache.h -- launch interface of the cache operators (kernels_cache.cu, kernels_cache_select.cu),
// called by cache_api.cpp after its argument checks.
#pragma once
#include <atomic>
#include <cuda_runtime.h>
#include <stdint.h>

namespace hoard {

constexpr int KV_SMS = 148;              // B200: one split CTA per SM
constexpr int KV_CHUNK = 16;             // rows of one step of a warp (the M of m16n8k16)
constexpr int TC_MIN_R = 16;             // the tensor-core form runs where a KV head has more query rows than these

// Dynamic shared memory above 48 KiB has to be allowed once for each kernel and device; asking again costs a
// launch's time in every call.
struct SmemLimit {
    std::atomic<uint64_t> done{0};       // devices 0..63
    cudaError_t raise(const void* fn, int bytes) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        const uint64_t bit = dev < 64 ? 1ull << dev : 0;
        if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
        e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
        return e;
    }
};

// a programmatic dependent launch in clusters of `cl` CTAs along x
template <typename... KArgs, typename... Args>
inline cudaError_t launch_pdl_cluster(void (*kernel)(KArgs...), int cl, dim3 grid, dim3 block, size_t smem, cudaStream_t s,
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

// The cache and the query side of one attention call. Strides in elements (caches) and floats (q, gate).
struct CacheAttn {
    const float* q;
    int64_t q_ts, q_hs;
    const void *kc, *vc;
    int64_t rs, hs;
    const uint64_t* vis;
    const float* gate;
    int64_t gate_ts, gate_hs;
    float* out;
    int n_head, n_kv, g, hd, m, n_past, max_rows;
    const int32_t* n_past_dev;
    bool bf16;
    float scale_log2;                    // scale * log2(e): scores are kept in units of log2
    // A problem is the set of query rows that read the same cache rows: a KV head with the R = m * g rows of
    // its query heads, or with a block list a (token, KV head) with R = g.
    int problems, R, tile_rows, row_tiles, splits;
    int tc_splits;                       // splits of the tensor-core form, 0 where it does not run
    bool cluster;                        // the splits are a cluster's CTAs and are joined by it
    // partial results of each (problem, split, query row): unnormalised sums, running maxima and totals
    float* part_o;                       // [problems][splits][R][tile dims]
    float2* part_ml;                     // [problems][splits][R]
    float* logits;                       // optional [n_kv][R][logits_ld], in log2 units
    int64_t logits_ld;
    float* acc;                          // optional [n_kv][max_rows]
    // block lists (sparse form): ascending block ids of each problem, and their number
    const int32_t* list;
    const int32_t* list_n;
    int list_cap, block;
};

int cache_tile_dims(int hd);             // dims of the instantiation that runs a head_dim
// sets tile_rows, row_tiles, splits, cluster, tc_splits for n_chunks chunks (past_rows rows of the past among them) a problem
void cache_plan(CacheAttn& a, int n_chunks, int64_t past_rows);
cudaError_t launch_cache_attention(const CacheAttn& a, cudaStream_t s);
cudaError_t launch_cache_attention_tc(const CacheAttn& a, cudaStream_t s);

struct CacheEvict {
    void *kc, *vc;
    int64_t rs, hs;
    const float* acc;
    const int32_t* pos;
    float* acc_out;
    int32_t* pos_out;
    int n_kv, hd, max_rows, n_rows, n_keep, n_sink, recent_from;
    int32_t *to, *from, *n_moves;        // [n_kv][max_rows] twice, [n_kv]
};
cudaError_t launch_cache_evict(const CacheEvict& e, cudaStream_t s);

cudaError_t launch_cache_bounds(const void* kc, int64_t rs, int64_t hs, bool bf16, int n_kv, int hd, int max_rows,
                                int block, int row0, int row1, const int32_t* row1_dev, void* bounds, cudaStream_t s);

// Scores of the candidate blocks, their selection, and the ascending lists that launch_cache_attention reads.
struct CacheSelect {
    const float* q;
    int64_t q_ts, q_hs;
    const void* bounds;
    bool bf16;
    int n_head, n_kv, g, hd, m, n_past, max_rows, block, n_sink, n_local, n_sel;
    int block_shift;                     // log2(block), set by the launcher
    const int32_t* n_past_dev;
    double* u;                           // [n_kv][m * g][max_rows / block]
    double* u_top;                       // [n_kv][m * g][ceil of that / 32]
    int32_t *list, *list_n, *sel_out;
    int list_cap;
};
cudaError_t launch_cache_select(const CacheSelect& c, cudaStream_t s);
// who chooses among n_cand candidates of each of `problems` problems: one CTA; one CTA, the keys formed by a cluster; a cluster
enum ChooseForm { CHOOSE_ONE, CHOOSE_GATHER, CHOOSE_CLUSTER };
ChooseForm choose_form(int n_cand, int problems);

struct TakePath {
    int32_t row[64];
};
cudaError_t launch_cache_take(void* kc, void* vc, int64_t rs, int64_t hs, int n_kv, int hd, int row0,
                              const TakePath& path, int n, cudaStream_t s);

}  // namespace hoard

// The form that a call runs, for tests and measurements, by the rules the calls themselves go by (cache_api.cpp).
// form: {1 where the tensor-core kernel runs, query rows of a tile, splits, 1 where a cluster (or one CTA) joins them}.
// n_blocks: blocks that each problem of hoard_kv_block_attention attends, -1 for hoard_kv_attention; acc: weights accumulated
struct hoard_kv_desc;
extern "C" int hoard_kv_attention_form(const hoard_kv_desc* d, int m, int n_past, int n_blocks, int acc, int32_t* form);
extern "C" int hoard_kv_choose_form(int n_cand, int problems);
