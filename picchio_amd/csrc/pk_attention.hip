// pk_attention.hip — attention of packed prompts (pk_attention_packed) and of
// new rows over paged caches (pk_attention_paged): the calls' checks and the
// choice of kernel.
#include "pk_attention.h"

#include <math.h>

namespace {

template <typename A, typename C, bool PAGED>
__global__ __launch_bounds__(64) void k_attn_rows(pk_attn_args a) {
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, hd = a.hd;
    const int kvh = h / (a.H / a.KVH);
    int lo = 0, hi = a.n_req - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.cu[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    const pk_span s = pk_request(a, lo);
    const int i = t - s.row0;
    if (i < 0 || i >= s.rows || i >= a.max_q) return;
    const int p = s.kv - s.rows + i;
    const int first = a.window > 0 ? max(p - a.window + 1, 0) : 0;
    __shared__ float q[128];
    for (int c = lane; c < hd; c += 64) q[c] = (float)((const A *)a.q)[(int64_t)t * a.q_stride + h * hd + c];
    __syncthreads();
    const float c2 = a.scale2;
    float m = a.sinks ? a.sinks[h] * 1.4426950408889634f : -INFINITY, l = a.sinks ? 1.0f : 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int j0 = first; j0 <= p; j0 += 64) {
        const int j = j0 + lane;
        int64_t at = -1;
        int64_t vat = -1;
        if (j <= p) {
            if (PAGED) {
                const int page = a.table[(int64_t)lo * a.max_blocks + (j >> a.page_shift)];
                if (page >= 0 && page < a.n_pages)
                    at = vat = ((((int64_t)page * a.KVH + kvh) << a.page_shift) + (j & ((1 << a.page_shift) - 1))) * hd;
            } else {
                at = (int64_t)(s.row0 + j) * a.k_stride + kvh * hd;
                vat = (int64_t)(s.row0 + j) * a.v_stride + kvh * hd;
            }
        }
        float sc = -INFINITY;
        if (at >= 0) {
            sc = 0.0f;
            for (int c = 0; c < hd; ++c) sc = __builtin_fmaf(q[c], (float)((const C *)a.k)[at + c], sc);
            sc *= c2;
        }
        const float mn = fmaxf(m, pk_wave_max_f(sc));
        if (mn == -INFINITY) continue;
        const float r = exp2f(m - mn), pr = at >= 0 ? exp2f(sc - mn) : 0.0f;
        l = l * r + pk_wave_sum_f(pr);
        o0 *= r, o1 *= r;
        for (int k = 0; k < 64; ++k) {
            const int64_t b = __shfl(vat, k);
            const float w = __shfl(pr, k);
            if (b < 0) continue;
            if (lane < hd) o0 = __builtin_fmaf(w, (float)((const C *)a.v)[b + lane], o0);
            if (lane + 64 < hd) o1 = __builtin_fmaf(w, (float)((const C *)a.v)[b + lane + 64], o1);
        }
        m = mn;
    }
    const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
    A *dst = (A *)a.out + (int64_t)t * a.out_stride + h * hd;
    if (lane < hd) dst[lane] = (A)(o0 * inv);
    if (lane + 64 < hd) dst[lane + 64] = (A)(o1 * inv);
    if (a.lse && lane == 0) a.lse[(int64_t)t * a.H + h] = m * 0.6931471805599453f + logf(l);
}

int check_common(const pk_engine *e, int H, int KVH, int hd, int n_tokens, int n_req, int max_q, int window, float scale) {
    PK_CHECK(n_tokens >= 0 && n_req >= 0 && max_q >= 0 && window >= 0, PK_ERR_ARG,
             "attention: %d rows, %d requests of up to %d rows, window %d", n_tokens, n_req, max_q, window);
    PK_CHECK(H > 0 && KVH > 0 && H % KVH == 0, PK_ERR_ARG, "attention: %d heads over %d", H, KVH);
    PK_CHECK(H <= 1024, PK_ERR_UNSUPPORTED, "attention: %d heads (supported: up to 1024)", H);
    PK_CHECK(hd >= 16 && hd <= 128 && hd % 16 == 0, PK_ERR_UNSUPPORTED,
             "head_dim %d (supported: multiples of 16 up to 128)", hd);
    PK_CHECK(scale >= 0.0f && scale <= 3.4e38f, PK_ERR_ARG, "attention: scale %g", (double)scale);
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
    a.n_tokens = p->n_tokens, a.n_req = p->n_seq, a.max_q = p->max_len, a.window = p->window;
    a.H = p->n_heads, a.KVH = p->n_kv_heads, a.hd = p->head_dim;
    a.scale2 = (p->scale > 0.0f ? p->scale : 1.0f / sqrtf((float)p->head_dim)) * PK_LOG2E;
    a.type = a.cache_type = p->type;
    pk_device_scope dev(e->device);
    PK_TRY(dev.rc);
    const dim3 grid((unsigned)a.n_tokens, (unsigned)a.H);
    if (p->type == PK_T_F32) k_attn_rows<float, float, false><<<grid, 64, 0, e->stream>>>(a);
    else if (p->type == PK_T_F16) k_attn_rows<pk_f16, pk_f16, false><<<grid, 64, 0, e->stream>>>(a);
    else k_attn_rows<pk_bf16, pk_bf16, false><<<grid, 64, 0, e->stream>>>(a);
    PK_HIP(hipGetLastError());
    return PK_OK;
}

extern "C" int pk_attention_paged(pk_engine *e, const pk_attn_paged *p) {
    PK_CHECK(e && p, PK_ERR_ARG, "null argument");
    PK_TRY(pk_check_pages(p->pages, p->type));
    const pk_pages &g = p->pages;
    PK_TRY(check_common(e, p->n_heads, g.n_kv_heads, g.head_dim, p->n_tokens, p->n_req, p->max_q, p->window, p->scale));
    PK_CHECK(p->max_kv >= 0 && p->max_blocks > 0 && (int64_t)p->max_blocks * g.page_size <= INT32_MAX, PK_ERR_ARG,
             "attention_paged: tables of %d pages of %d, max_kv %d", p->max_blocks, g.page_size, p->max_kv);
    if (p->n_tokens == 0 || p->n_req == 0 || p->max_q == 0) return PK_OK;
    PK_CHECK(p->cu_q_dev && p->kv_len_dev && p->table_dev, PK_ERR_ARG, "attention_paged: null argument");
    PK_TRY(pk_check_rows(p->q_dev, p->q_stride, p->n_heads, g.head_dim, "q"));
    PK_TRY(pk_check_rows(p->out_dev, p->out_stride, p->n_heads, g.head_dim, "out"));
    pk_attn_args a{};
    a.q = p->q_dev, a.k = g.k_dev, a.v = g.v_dev, a.out = p->out_dev;
    a.q_stride = p->q_stride, a.out_stride = p->out_stride;
    a.cu = p->cu_q_dev, a.kv_len = p->kv_len_dev, a.table = p->table_dev, a.sinks = p->sinks_dev, a.lse = p->lse_dev;
    a.n_tokens = p->n_tokens, a.n_req = p->n_req, a.max_q = p->max_q, a.window = p->window;
    a.H = p->n_heads, a.KVH = g.n_kv_heads, a.hd = g.head_dim;
    a.n_pages = g.n_pages, a.page_shift = __builtin_ctz((unsigned)g.page_size), a.max_blocks = p->max_blocks;
    a.scale2 = (p->scale > 0.0f ? p->scale : 1.0f / sqrtf((float)g.head_dim)) * PK_LOG2E;
    a.type = p->type, a.cache_type = g.type;
    pk_device_scope dev(e->device);
    PK_TRY(dev.rc);
    const int64_t cap = (int64_t)p->max_blocks * g.page_size;
    const int max_kv = (int)(p->max_kv > 0 ? std::min<int64_t>(p->max_kv, cap) : cap);
    if ((int64_t)a.max_q * (a.H / a.KVH) <= PK_FEW_ROWS) return pk_launch_attn_few(e, a, max_kv);
    const dim3 grid((unsigned)a.n_tokens, (unsigned)a.H);
#define PK_ATTN(A, C) k_attn_rows<A, C, true><<<grid, 64, 0, e->stream>>>(a)
    PK_BY_TYPES(p->type, g.type, PK_ATTN);
#undef PK_ATTN
    PK_HIP(hipGetLastError());
    return PK_OK;
}
