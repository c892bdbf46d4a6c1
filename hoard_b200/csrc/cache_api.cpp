// cache_api.cpp -- the C ABI of include/hoard_cache.h: argument checks, the workspace's layout and the
// launches of the cache operators (kernels_cache.cu, kernels_cache_select.cu). Stateless; status codes as
// hoard_moe.h.
#include "../../include/hoard_cache.h"
#include "kernels.h"
#include "kernels_cache.h"

#include <cmath>

using namespace hoard;

namespace {

constexpr float LOG2E = 1.4426950408889634f;

inline int64_t al256(int64_t v) { return (v + 255) / 256 * 256; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline int st(cudaError_t e) {
    if (e == cudaSuccess) return HOARD_OK;
    cudaGetLastError();
    return e == cudaErrorInvalidValue ? HOARD_EINVAL : HOARD_ECUDA;
}

inline int64_t row_stride(const hoard_kv_desc* d) {
    return d->row_stride ? d->row_stride : (int64_t)d->n_head_kv * d->head_dim;
}
inline int64_t head_stride(const hoard_kv_desc* d) { return d->row_stride ? d->head_stride : d->head_dim; }

bool desc_ok(const hoard_kv_desc* d) {
    if (!d || d->n_head <= 0 || d->n_head_kv <= 0 || d->n_head % d->n_head_kv || d->n_head / d->n_head_kv > 64 ||
        d->n_head > 4096 || d->head_dim < 8 || d->head_dim > 256 || d->head_dim % 8)
        return false;
    if (d->kv_type != HOARD_TYPE_F16 && d->kv_type != HOARD_TYPE_BF16) return false;
    if (d->max_rows <= 0 || d->max_rows > (1 << 30) || d->max_tokens < 1 || d->max_tokens > HOARD_KV_MAX_TOKENS ||
        d->max_tokens > d->max_rows || d->max_acc_tokens < 0 || d->max_acc_tokens > d->max_tokens ||
        d->max_acc_tokens * (d->n_head / d->n_head_kv) > 512)
        return false;
    if (d->block != 0 && d->block != 16 && d->block != 32 && d->block != 64 && d->block != 128) return false;
    if (d->block && d->max_rows / d->block > 131072) return false;
    // the block form's problems, (token, KV head), are the third dimension of its grid
    if (d->block && (int64_t)d->max_tokens * d->n_head_kv > 65535) return false;
    if (!(d->scale > 0) || !std::isfinite(d->scale * LOG2E)) return false;
    // either [row][head][dim]-like (heads inside a row) or [head][row][dim]-like, elements of a head contiguous
    if (d->row_stride == 0 && d->head_stride == 0) return true;
    if (d->row_stride < d->head_dim || d->head_stride < d->head_dim || d->row_stride % 8 || d->head_stride % 8)
        return false;
    return d->row_stride >= d->head_stride * (d->n_head_kv - 1) + d->head_dim ||
           d->head_stride >= d->row_stride * ((int64_t)d->max_rows - 1) + d->head_dim;
}

// The workspace: the splits' partial results, the logits that accumulation needs, and the block operators'
// scores and lists; an eviction's lists take the same bytes, no call needs both.
struct Ws {
    int64_t part_o, part_ml, logits, u, u_top, list, list_n, attn_end;
    int64_t to, from, n_moves, evict_end;
    int64_t logits_ld;
    int list_cap;
};
Ws ws_plan(const hoard_kv_desc* d) {
    Ws w{};
    const int g = d->n_head / d->n_head_kv, hdt = cache_tile_dims(d->head_dim);
    // partial results exist where there are splits: then problems x row tiles x splits is at most one CTA per SM, with
    // tiles of 16 query rows or in the tensor-core form 128; a call that accumulates has them without splits too
    const int64_t R = (int64_t)d->max_tokens * g;
    int64_t rows = KV_SMS * 16;
    if (R > TC_MIN_R && hdt <= 128) rows = KV_SMS * 128;
    if (rows < (int64_t)d->max_acc_tokens * d->n_head) rows = (int64_t)d->max_acc_tokens * d->n_head;
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t o = at;
        at += al256(bytes);
        return o;
    };
    w.part_o = take(rows * hdt * 4);
    w.part_ml = take(rows * 8);
    w.logits_ld = ceil_div(d->max_rows, 8) * 8;
    w.logits = take((int64_t)d->max_acc_tokens * d->n_head * w.logits_ld * 4);
    if (d->block) {
        w.list_cap = (int)ceil_div(d->max_rows, d->block);
        w.u = take((int64_t)d->max_tokens * d->n_head * (d->max_rows / d->block) * 8);
        w.u_top = take((int64_t)d->max_tokens * d->n_head * ceil_div(d->max_rows / d->block, 32) * 8);
        w.list = take((int64_t)d->max_tokens * d->n_head_kv * w.list_cap * 4);
        w.list_n = take((int64_t)d->max_tokens * d->n_head_kv * 4);
    }
    w.attn_end = at;
    at = 0;
    w.to = take((int64_t)d->n_head_kv * d->max_rows * 4);
    w.from = take((int64_t)d->n_head_kv * d->max_rows * 4);
    w.n_moves = take((int64_t)d->n_head_kv * 4);
    w.evict_end = at;
    return w;
}

// Heads of hd floats, one token's after another's or one head's tokens after another's, none over the next
bool heads_ok(int64_t ts, int64_t hs, int m, int n_head, int hd) {
    if (hs < hd || ts < 0) return false;
    return m == 1 || ts >= hs * (n_head - 1) + hd || (ts >= hd && hs >= ts * (m - 1) + hd);
}

bool query_ok(const hoard_kv_desc* d, const hoard_kv_query* a) {
    if (!a || !a->q || !a->k_cache || !a->v_cache || !a->out || !aligned16(a->k_cache) || !aligned16(a->v_cache))
        return false;
    if (a->m < 1 || a->m > d->max_tokens || !heads_ok(a->q_token_stride, a->q_head_stride, a->m, d->n_head, d->head_dim))
        return false;
    if (a->gate && (a->gate_head_stride < d->head_dim || a->gate_token_stride < 0)) return false;
    if (!a->n_past_dev && (a->n_past < 0 || a->n_past > d->max_rows - a->m)) return false;
    return true;
}

CacheAttn attn_of(const hoard_kv_desc* d, const hoard_kv_query* a) {
    CacheAttn c{};
    c.q = a->q;
    c.q_ts = a->q_token_stride;
    c.q_hs = a->q_head_stride;
    c.kc = a->k_cache;
    c.vc = a->v_cache;
    c.rs = row_stride(d);
    c.hs = head_stride(d);
    c.vis = a->visible;
    c.gate = a->gate;
    c.gate_ts = a->gate_token_stride;
    c.gate_hs = a->gate_head_stride;
    c.out = a->out;
    c.n_head = d->n_head;
    c.n_kv = d->n_head_kv;
    c.g = d->n_head / d->n_head_kv;
    c.hd = d->head_dim;
    c.m = a->m;
    c.n_past = a->n_past;
    c.max_rows = d->max_rows;
    c.n_past_dev = a->n_past_dev;
    c.bf16 = d->kv_type == HOARD_TYPE_BF16;
    c.scale_log2 = d->scale * LOG2E;
    return c;
}
// most chunks of a problem, for the number of splits
int chunks_of(const CacheAttn& c, int64_t past_rows) {
    return (int)(ceil_div(past_rows, KV_CHUNK) + ceil_div(c.m, KV_CHUNK));
}
// A problem is a KV head with the rows of all its tokens, or with a block list one token of it
void plan_dense(CacheAttn& c) {
    const int64_t past = c.n_past_dev ? c.max_rows - c.m : c.n_past;
    c.problems = c.n_kv;
    c.R = c.m * c.g;
    cache_plan(c, chunks_of(c, past), past);
}
void plan_blocks(CacheAttn& c, int64_t blocks) {
    c.problems = c.n_kv * c.m;
    c.R = c.g;
    cache_plan(c, chunks_of(c, blocks * c.block), blocks * c.block);
}
}  // namespace

extern "C" {

int64_t hoard_kv_ws_bytes(const hoard_kv_desc* d) {
    if (!desc_ok(d)) return -1;
    const Ws w = ws_plan(d);
    return w.attn_end > w.evict_end ? w.attn_end : w.evict_end;
}

int hoard_kv_attention(const hoard_kv_desc* d, const hoard_kv_query* a, float* acc, void* ws, hoard_stream stream) {
    if (!desc_ok(d) || !query_ok(d, a) || !ws || !aligned16(ws) || (acc && a->m > d->max_acc_tokens)) return HOARD_EINVAL;
    const Ws w = ws_plan(d);
    char* b = static_cast<char*>(ws);
    CacheAttn c = attn_of(d, a);
    c.part_o = reinterpret_cast<float*>(b + w.part_o);
    c.part_ml = reinterpret_cast<float2*>(b + w.part_ml);
    if (acc) {
        c.acc = acc;
        c.logits = reinterpret_cast<float*>(b + w.logits);
        c.logits_ld = w.logits_ld;
    }
    plan_dense(c);
    return st(launch_cache_attention(c, (cudaStream_t)stream));
}

int hoard_kv_evict(const hoard_kv_desc* d, void* k_cache, void* v_cache, const float* acc, const int32_t* row_pos,
                   int n_rows, int n_keep, int n_sink, int recent_from, float* acc_out, int32_t* pos_out, void* ws,
                   hoard_stream stream) {
    if (!desc_ok(d) || !k_cache || !v_cache || !acc || !row_pos || !acc_out || !pos_out || !ws || !aligned16(ws) ||
        !aligned16(k_cache) || !aligned16(v_cache) || n_rows > d->max_rows || n_keep < 1 || n_keep > n_rows)
        return HOARD_EINVAL;
    const Ws w = ws_plan(d);
    char* b = static_cast<char*>(ws);
    CacheEvict e{};
    e.kc = k_cache;
    e.vc = v_cache;
    e.rs = row_stride(d);
    e.hs = head_stride(d);
    e.acc = acc;
    e.pos = row_pos;
    e.acc_out = acc_out;
    e.pos_out = pos_out;
    e.n_kv = d->n_head_kv;
    e.hd = d->head_dim;
    e.max_rows = d->max_rows;
    e.n_rows = n_rows;
    e.n_keep = n_keep;
    e.n_sink = n_sink;
    e.recent_from = recent_from;
    e.to = reinterpret_cast<int32_t*>(b + w.to);
    e.from = reinterpret_cast<int32_t*>(b + w.from);
    e.n_moves = reinterpret_cast<int32_t*>(b + w.n_moves);
    return st(launch_cache_evict(e, (cudaStream_t)stream));
}

int hoard_kv_block_bounds(const hoard_kv_desc* d, const void* k_cache, void* bounds, int row0, int row1,
                          const int32_t* row1_dev, hoard_stream stream) {
    if (!desc_ok(d) || !d->block || !k_cache || !bounds || !aligned16(k_cache) || !aligned16(bounds)) return HOARD_EINVAL;
    if (!row1_dev && (row0 < 0 || row1 < row0 || row1 > d->max_rows)) return HOARD_EINVAL;
    return st(launch_cache_bounds(k_cache, row_stride(d), head_stride(d), d->kv_type == HOARD_TYPE_BF16, d->n_head_kv,
                                  d->head_dim, d->max_rows, d->block, row0, row1, row1_dev, bounds,
                                  (cudaStream_t)stream));
}

int hoard_kv_block_attention(const hoard_kv_desc* d, const hoard_kv_query* a, const void* bounds, int n_sink,
                             int n_local, int n_sel, int32_t* sel_out, void* ws, hoard_stream stream) {
    if (!desc_ok(d) || !d->block || !query_ok(d, a) || !bounds || !aligned16(bounds) || !ws || !aligned16(ws) ||
        n_sink < 0 || n_local < 1 || n_sel < 0)
        return HOARD_EINVAL;
    const Ws w = ws_plan(d);
    char* b = static_cast<char*>(ws);
    CacheAttn c = attn_of(d, a);
    const int nb_most = (int)ceil_div(c.n_past_dev ? c.max_rows - c.m : c.n_past, d->block);
    CacheSelect s{};
    s.q = c.q;
    s.q_ts = c.q_ts;
    s.q_hs = c.q_hs;
    s.bounds = bounds;
    s.bf16 = c.bf16;
    s.n_head = c.n_head;
    s.n_kv = c.n_kv;
    s.g = c.g;
    s.hd = c.hd;
    s.m = c.m;
    s.n_past = c.n_past;
    s.max_rows = c.max_rows;
    s.block = d->block;
    s.n_sink = n_sink < w.list_cap ? n_sink : w.list_cap;
    s.n_local = n_local < w.list_cap ? n_local : w.list_cap;
    s.n_sel = n_sel;
    s.n_past_dev = c.n_past_dev;
    s.u = reinterpret_cast<double*>(b + w.u);
    s.u_top = reinterpret_cast<double*>(b + w.u_top);
    s.list = reinterpret_cast<int32_t*>(b + w.list);
    s.list_n = reinterpret_cast<int32_t*>(b + w.list_n);
    s.list_cap = w.list_cap;
    s.sel_out = sel_out;
    int rc = st(launch_cache_select(s, (cudaStream_t)stream));
    if (rc != HOARD_OK) return rc;
    c.part_o = reinterpret_cast<float*>(b + w.part_o);
    c.part_ml = reinterpret_cast<float2*>(b + w.part_ml);
    c.list = s.list;
    c.list_n = s.list_n;
    c.list_cap = s.list_cap;
    c.block = d->block;
    int64_t blocks = (int64_t)s.n_sink + s.n_local + n_sel;
    if (blocks > nb_most) blocks = nb_most;
    plan_blocks(c, blocks);
    return st(launch_cache_attention(c, (cudaStream_t)stream));
}

int hoard_kv_take(const hoard_kv_desc* d, void* k_cache, void* v_cache, int row0, const int32_t* path, int n,
                  hoard_stream stream) {
    if (!desc_ok(d) || !k_cache || !v_cache || !aligned16(k_cache) || !aligned16(v_cache) || row0 < 0 || n < 0 ||
        n > HOARD_KV_MAX_TOKENS || (n && !path))
        return HOARD_EINVAL;
    TakePath p{};
    bool moves = false;
    for (int i = 0; i < n; ++i) {
        if (path[i] < (i ? path[i - 1] + 1 : 0) || path[i] >= HOARD_KV_MAX_TOKENS || path[i] >= d->max_rows - row0)
            return HOARD_EINVAL;
        p.row[i] = path[i];
        moves |= path[i] != i;
    }
    if (!moves) return HOARD_OK;
    return st(launch_cache_take(k_cache, v_cache, row_stride(d), head_stride(d), d->n_head_kv, d->head_dim, row0, p, n,
                                (cudaStream_t)stream));
}

int hoard_kv_store(const hoard_kv_desc* d, const float* q, int64_t q_token_stride, int64_t q_head_stride,
                   const float* k, const float* v, const float* q_norm, const float* k_norm, int mode, float eps,
                   int rope_dim, float freq_base, const int32_t* pos, int m, int row0, const int32_t* row0_dev,
                   float* q_out, void* k_cache, void* v_cache, float* acc, int32_t* row_pos, hoard_stream stream) {
    if (!desc_ok(d) || !q || !k || !v || !pos || !q_out || q_out == q || !k_cache || !v_cache || m < 1 ||
        m > HOARD_KV_MAX_TOKENS || mode < 0 || mode > 2 || (mode && (!q_norm || !k_norm)) || rope_dim < 2 ||
        rope_dim > d->head_dim || rope_dim % 2 || !(freq_base > 0) ||
        !heads_ok(q_token_stride, q_head_stride, m, d->n_head, d->head_dim) ||
        (mode == 1 && q_head_stride != d->head_dim) || (!row0_dev && row0 < 0))
        return HOARD_EINVAL;
    return st(launch_qknorm_rope_store_rows(q, q_token_stride, q_head_stride, k, v, q_norm, k_norm, mode, eps, d->n_head,
                                            d->n_head_kv, d->head_dim, rope_dim, pos, m, row0, row0_dev, d->max_rows,
                                            freq_base, q_out, k_cache, v_cache, row_stride(d), head_stride(d),
                                            d->kv_type == HOARD_TYPE_BF16, acc, row_pos, (cudaStream_t)stream));
}

int hoard_kv_attention_form(const hoard_kv_desc* d, int m, int n_past, int n_blocks, int acc, int32_t* form) {
    if (!desc_ok(d) || !form || m < 1 || m > d->max_tokens || n_past < 0 || n_past > d->max_rows - m) return HOARD_EINVAL;
    hoard_kv_query a{};
    a.m = m;
    a.n_past = n_past;
    CacheAttn c = attn_of(d, &a);
    // what is not null says what the call does; nothing is read
    if (acc) c.logits = reinterpret_cast<float*>(form);
    if (n_blocks >= 0) c.list = form;
    c.block = d->block;
    if (n_blocks >= 0) plan_blocks(c, n_blocks);
    else plan_dense(c);
    form[0] = c.tc_splits != 0;
    form[1] = c.tile_rows;
    form[2] = c.splits;
    form[3] = !c.tc_splits && c.cluster;
    return HOARD_OK;
}

int hoard_kv_choose_form(int n_cand, int problems) { return choose_form(n_cand, problems); }

}  // extern "C"
