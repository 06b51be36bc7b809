// pk_attention.hip — attention of packed prompts (pk_attention_packed) and of
// new rows over paged caches (pk_attention_paged): the calls' checks and the
// choice of kernel.
#include "pk_attention.h"

#include <math.h>

namespace {

constexpr int MAX_REQ = 1 << 17;                             // (every workgroup looks through all of them)

int check_common(const pk_engine *e, int H, int KVH, int hd, int n_tokens, int n_req, int max_q, int window, float scale) {
    PK_CHECK(n_tokens >= 0 && n_req >= 0 && max_q >= 0 && window >= 0, PK_ERR_ARG,
             "attention: %d rows, %d requests of up to %d rows, window %d", n_tokens, n_req, max_q, window);
    PK_CHECK(H > 0 && KVH > 0 && H % KVH == 0, PK_ERR_ARG, "attention: %d heads over %d", H, KVH);
    PK_CHECK(H <= 1024, PK_ERR_UNSUPPORTED, "attention: %d heads (supported: up to 1024)", H);
    PK_CHECK(hd >= 16 && hd <= 128 && hd % 16 == 0, PK_ERR_UNSUPPORTED,
             "head_dim %d (supported: multiples of 16 up to 128)", hd);
    PK_CHECK(scale >= 0.0f && scale <= 3.4e38f, PK_ERR_ARG, "attention: scale %g", (double)scale);
    PK_CHECK(n_req <= MAX_REQ, PK_ERR_UNSUPPORTED, "attention: %d requests (supported: up to %d)", n_req, MAX_REQ);
    // (the kernels count columns, and positions before the first, in 32 bits)
    PK_CHECK((int64_t)n_tokens * (H / KVH) <= 1 << 30, PK_ERR_UNSUPPORTED, "attention: %d rows of %d heads per key head", n_tokens, H / KVH);
    return PK_OK;
}

}  // namespace

int pk_attn_workspace(pk_engine *e, int64_t floats, int64_t counts) {
    if (floats <= e->att_ws_floats && counts <= e->att_ws_counts) return PK_OK;
    PK_CHECK(!e->capturing, PK_ERR_ARG, "attention: the workspace would grow while capturing; run the call once before");
    floats = std::max(floats, e->att_ws_floats);
    counts = std::max(counts, e->att_ws_counts);
    const pk_buf_bytes b[] = {{(void **)&e->att_ws, floats * 4}, {(void **)&e->att_cnt, counts * 4}};
    const int rc = pk_regrow(e, e->att_use, b, 2);
    if (rc != PK_OK) {                                       // (the old ones are kept for a graph, or are gone)
        if (!e->att_ws || !e->att_cnt) e->att_ws_floats = e->att_ws_counts = 0;
        return rc;
    }
    e->att_ws_floats = e->att_ws_counts = 0;
    PK_HIP(hipMemsetAsync(e->att_cnt, 0, (size_t)counts * 4, e->stream));
    e->att_ws_floats = floats;
    e->att_ws_counts = counts;
    return PK_OK;
}

extern "C" int pk_attention_packed(pk_engine *e, const pk_attn_packed *p) {
    PK_CHECK(e && p, PK_ERR_ARG, "null argument");
    PK_CHECK(pk_type_size(p->type), PK_ERR_ARG, "type %d", p->type);
    PK_TRY(check_common(e, p->n_heads, p->n_kv_heads, p->head_dim, p->n_tokens, p->n_seq, p->max_len, p->window, p->scale));
    if (p->n_tokens == 0 || p->n_seq == 0 || p->max_len == 0) return PK_OK;
    PK_CHECK(p->cu_dev, PK_ERR_ARG, "attention_packed: null argument");
    PK_TRY(pk_check_rows(p->q_dev, p->q_stride, p->n_heads, p->head_dim, "q"));
    PK_TRY(pk_check_rows(p->k_dev, p->k_stride, p->n_kv_heads, p->head_dim, "k"));
    PK_TRY(pk_check_rows(p->v_dev, p->v_stride, p->n_kv_heads, p->head_dim, "v"));
    PK_TRY(pk_check_rows(p->out_dev, p->out_stride, p->n_heads, p->head_dim, "out"));
    pk_attn_args a{};
    a.q = p->q_dev, a.k = p->k_dev, a.v = p->v_dev, a.out = p->out_dev;
    a.q_stride = p->q_stride, a.k_stride = p->k_stride, a.v_stride = p->v_stride, a.out_stride = p->out_stride;
    a.cu = p->cu_dev, a.sinks = p->sinks_dev, a.lse = p->lse_dev;
    a.n_tokens = p->n_tokens, a.n_req = p->n_seq, a.max_q = p->max_len;
    a.window = p->window < p->n_tokens ? p->window : 0;
    a.H = p->n_heads, a.KVH = p->n_kv_heads, a.hd = p->head_dim;
    a.scale2 = (p->scale > 0.0f ? p->scale : 1.0f / sqrtf((float)p->head_dim)) * PK_LOG2E;
    a.type = a.cache_type = p->type;
    pk_device_scope dev(e->device);
    PK_TRY(dev.rc);
    return pk_launch_attn_tile(e, a, 0, p->max_len);
}

extern "C" int pk_attention_paged(pk_engine *e, const pk_attn_paged *p) {
    PK_CHECK(e && p, PK_ERR_ARG, "null argument");
    PK_TRY(pk_check_pages(p->pages, p->type));
    const pk_pages &g = p->pages;
    PK_TRY(check_common(e, p->n_heads, g.n_kv_heads, g.head_dim, p->n_tokens, p->n_req, p->max_q, p->window, p->scale));
    PK_CHECK(p->max_kv >= 0 && p->max_blocks > 0 && (int64_t)p->max_blocks * g.page_size <= 1 << 30, PK_ERR_ARG,
             "attention_paged: tables of %d pages of %d, max_kv %d", p->max_blocks, g.page_size, p->max_kv);
    if (p->n_tokens == 0 || p->n_req == 0 || p->max_q == 0) return PK_OK;
    PK_CHECK(p->cu_q_dev && p->kv_len_dev && p->table_dev, PK_ERR_ARG, "attention_paged: null argument");
    PK_TRY(pk_check_rows(p->q_dev, p->q_stride, p->n_heads, g.head_dim, "q"));
    PK_TRY(pk_check_rows(p->out_dev, p->out_stride, p->n_heads, g.head_dim, "out"));
    pk_attn_args a{};
    a.q = p->q_dev, a.k = g.k_dev, a.v = g.v_dev, a.out = p->out_dev;
    a.q_stride = p->q_stride, a.out_stride = p->out_stride;
    a.cu = p->cu_q_dev, a.kv_len = p->kv_len_dev, a.table = p->table_dev, a.sinks = p->sinks_dev, a.lse = p->lse_dev;
    a.n_tokens = p->n_tokens, a.n_req = p->n_req, a.max_q = p->max_q;
    a.H = p->n_heads, a.KVH = g.n_kv_heads, a.hd = g.head_dim;
    a.n_pages = g.n_pages, a.page_shift = __builtin_ctz((unsigned)g.page_size), a.max_blocks = p->max_blocks;
    a.scale2 = (p->scale > 0.0f ? p->scale : 1.0f / sqrtf((float)g.head_dim)) * PK_LOG2E;
    a.type = p->type, a.cache_type = g.type;
    pk_device_scope dev(e->device);
    PK_TRY(dev.rc);
    const int64_t cap = (int64_t)p->max_blocks * g.page_size;
    a.window = p->window < cap ? p->window : 0;
    const int max_kv = (int)(p->max_kv > 0 ? std::min<int64_t>(p->max_kv, cap) : cap);
    // Few rows of every request: k_attn_few, bound by the reads of K and V. Else the
    // requests with few rows there (a tile of 128 or 256 columns would be
    // mostly empty for them), the others in tiles.
    const int G = a.H / a.KVH;
    if ((int64_t)a.max_q * G <= PK_FEW_ROWS) return pk_launch_attn_few(e, a);
    int cut = 0;
    if (a.n_req > 1 && G <= PK_FEW_ROWS) {
        cut = G <= 16 ? 16 : PK_FEW_ROWS;
        pk_attn_args few = a;
        few.max_q = cut / G, few.few_only = 1;
        PK_TRY(pk_launch_attn_few(e, few));
    }
    return pk_launch_attn_tile(e, a, cut, max_kv);
}
