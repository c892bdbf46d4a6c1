/* hoard_cache.h -- operators on a layer's KV cache for several query tokens, long contexts and bounded
 * caches: attention of a tree of drafted tokens, attention that accumulates its weights, eviction by
 * those weights, and attention over blocks of the cache that a score selects.
 *
 * They stand beside hoard_hx_attention (hoard_harness.h), which attends one token over the whole cache
 * with its scores in shared memory. hoard's speculative loop (src/run_specloop.cpp:189-210) verifies a
 * chain of drafts with a causal mask (:86-95); a tree of drafts is its generalisation.
 *
 * A cache holds rows of f16 or bf16 values, one row per stored token: element (row, kv head, d) is at
 * row * row_stride + kv * head_stride + d. Past rows are [0, n_past); the m query tokens' own keys and
 * values are rows n_past .. n_past + m - 1 and have been stored before the call. n_past comes from the
 * host, or with n_past_dev from device memory (clamped to [0, max_rows - m]), so that a captured CUDA
 * graph can be replayed at growing positions. Rows at or past n_past + m are never read.
 *
 * Every call is asynchronous on `stream` and runs on the current device, which has to be the pointers'.
 * A call uses the workspace `ws` (hoard_kv_ws_bytes, any contents, 16-byte aligned) until it has
 * completed: calls that may overlap, captured graphs among them, need workspaces of their own. Status
 * codes are those of hoard_moe.h; bad arguments are refused (HOARD_EINVAL) before anything is launched. */
#ifndef HOARD_CACHE_H
#define HOARD_CACHE_H

#include <stdint.h>
#include "hoard_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

#define HOARD_KV_MAX_TOKENS 64      /* query tokens of one call: the bits of a visibility word */

typedef struct hoard_kv_desc {
    int n_head, n_head_kv;  /* n_head a multiple of n_head_kv, at most 64 query heads per KV head */
    int head_dim;           /* a multiple of 8, 8 .. 256 */
    int kv_type;            /* HOARD_TYPE_F16 or HOARD_TYPE_BF16 */
    int max_rows;           /* rows of the caches */
    int max_tokens;         /* most query tokens of a call, 1 .. HOARD_KV_MAX_TOKENS (sizes the workspace) */
    int max_acc_tokens;     /* most query tokens of a call that accumulates weights, 0 .. max_tokens */
    int block;              /* rows of a block for the block operators: 16, 32, 64 or 128 (max_rows / block at most
                               131072, n_head_kv * max_tokens 65535); 0: not used */
    int64_t row_stride, head_stride; /* in elements, multiples of 8; both 0: [row][n_head_kv][head_dim] */
    float scale;            /* of the scores, finite and > 0 */
} hoard_kv_desc;

/* Bytes of the workspace of every call with this descriptor; -1 where the descriptor is refused. */
int64_t hoard_kv_ws_bytes(const hoard_kv_desc* d);

/* The query side of an attention call. */
typedef struct hoard_kv_query {
    const float* q;              /* head h of token t at q + t * q_token_stride + h * q_head_stride */
    int64_t q_token_stride, q_head_stride;       /* in floats; token after token or head after head, none overlapping */
    const void* k_cache;         /* 16-byte aligned */
    const void* v_cache;
    const uint64_t* visible;     /* [m]: bit i of word t: token t sees token i's row. NULL: rows of tokens <= t */
    const float* gate;           /* optional: head h of token t's output times sigmoid(gate[...]) */
    int64_t gate_token_stride, gate_head_stride;
    float* out;                  /* [m][n_head][head_dim]; may be q where q has this layout */
    int m, n_past;
    const int32_t* n_past_dev;   /* optional, overrides n_past */
} hoard_kv_query;

/* out[t][h] = sum_j p_j V[j], p = softmax over the rows that token t sees of scale * q[t][h] . K[j]: every past
 * row and its visible own rows. A token that sees nothing gets 0; what masked rows hold, infinities and
 * NaN among it, does not reach the result. Of a row that is seen an infinity may come out as NaN. Sums are
 * f32 and weights at most 1 in them (2^14 over f16): |V| times the rows has to stay below the largest float. acc (optional, f32 [n_head_kv][max_rows], m <= max_acc_tokens):
 * acc[kv][j] += sum of p_j over the tokens and the heads of KV head kv, in a fixed order. */
int hoard_kv_attention(const hoard_kv_desc* d, const hoard_kv_query* a, float* acc, void* ws, hoard_stream stream);

/* Keeps n_keep of the rows [0, n_rows) of each KV head, by accumulated weight, in rows [0, n_keep):
 * kept are first the rows whose position row_pos is < n_sink or >= recent_from, then those of the largest
 * acc (NaN ranks below everything), the lower row first where equal. The i-th row below n_keep that is
 * not kept takes the contents (K, V, acc, row_pos) of the i-th kept row at or above n_keep; no other row
 * of the caches is written, so after an eviction a head's rows are no longer in the order of positions.
 * acc, row_pos: [n_head_kv][max_rows]. acc_out / pos_out receive entries [0, n_keep) of each head and may
 * be acc / row_pos themselves. 1 <= n_keep <= n_rows <= max_rows. */
int hoard_kv_evict(const hoard_kv_desc* d, void* k_cache, void* v_cache, const float* acc, const int32_t* row_pos,
                   int n_rows, int n_keep, int n_sink, int recent_from, float* acc_out, int32_t* pos_out, void* ws,
                   hoard_stream stream);

/* bounds[kv][b] = elementwise minimum and maximum of the keys of block b, rows [b * block, (b + 1) * block),
 * [n_head_kv][max_rows / block][2][head_dim] of the cache's type, for the complete blocks that end in
 * (row0, row1]. row1_dev (optional): row1 = *row1_dev + 1 (clamped to max_rows), row0 = *row1_dev; for the
 * token a captured decode step has stored. */
int hoard_kv_block_bounds(const hoard_kv_desc* d, const void* k_cache, void* bounds, int row0, int row1,
                          const int32_t* row1_dev, hoard_stream stream);

/* hoard_kv_attention over a choice of past rows. With nb = ceil(n_past / block): each token and KV head
 * attends the blocks below n_sink, the last n_local (>= 1), and of the others the n_sel whose score is
 * largest (the lower block where equal), beside the token's visible own rows. The score of block b is
 * max over the KV head's query heads of U_h(b) - max_b' U_h(b'), U_h(b) = sum_d max(q_d kmin_d, q_d kmax_d), an
 * upper bound of q . k over the block's keys; formed and compared in 64 bits, the NaN of a NaN in q ranking
 * lowest and infinite keys counting as one step above the largest finite value.
 * What keys of NaN count as is not defined. bounds have to be those of the complete blocks of [0, n_past). sel_out (optional, [m][n_head_kv][n_sel]):
 * the chosen blocks in ascending order, then -1. */
int hoard_kv_block_attention(const hoard_kv_desc* d, const hoard_kv_query* a, const void* bounds, int n_sink,
                             int n_local, int n_sel, int32_t* sel_out, void* ws, hoard_stream stream);

/* Rows row0 + path[i] of both caches to rows row0 + i, i < n: the accepted path of a drafted tree, path
 * a host array, strictly ascending, 0 <= path[i] < HOARD_KV_MAX_TOKENS, row0 + path[n - 1] < max_rows. */
int hoard_kv_take(const hoard_kv_desc* d, void* k_cache, void* v_cache, int row0, const int32_t* path, int n,
                  hoard_stream stream);

/* hoard_hx_qknorm_rope_store_ex for m tokens whose rows need not be their positions: token t's rotation
 * is that of position pos[t] (device memory) and its k, v go to row row0 + t (row0_dev optional, overrides
 * row0; a row outside [0, max_rows) is not written). q: heads q_head_stride floats apart, tokens
 * q_token_stride; k, v: [m][n_head_kv * head_dim]; q_out [m][n_head][head_dim], not q. With acc / row_pos
 * ([n_head_kv][max_rows], optional) a stored row starts with weight 0 and its position. */
int hoard_kv_store(const hoard_kv_desc* d, const float* q, int64_t q_token_stride, int64_t q_head_stride,
                   const float* k, const float* v, const float* q_norm, const float* k_norm, int mode, float eps,
                   int rope_dim, float freq_base, const int32_t* pos, int m, int row0, const int32_t* row0_dev,
                   float* q_out, void* k_cache, void* v_cache, float* acc, int32_t* row_pos, hoard_stream stream);

#ifdef __cplusplus
}
#endif

#endif
