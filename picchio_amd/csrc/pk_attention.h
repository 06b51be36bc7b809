// pk_attention.h — what the attention kernels of packed prompts and paged
// caches share (pk_attention.hip: the calls; pk_attn_few.hip: few rows over
// many positions; pk_attn_tile.hip: many rows).
//
// Row i of a request at position p sees the positions j in (p - window, p]:
// s_j = scale q . k_j, m = max(max_j s_j, sink), l = sum_j exp(s_j - m) +
// exp(sink - m), o = sum_j exp(s_j - m) v_j / l, lse = m + ln l. One pass over
// the positions carries the running m, l and o, rescaled where m grows; runs
// over parts of the positions are joined by the same rule. Exponentials are
// taken to the base 2 (log2 e is part of the scale).
#pragma once

#include "pk_engine.h"
#include "pk_types.h"

// What both calls hand to a kernel: the requests' rows of q, and where their
// positions' keys and values lie (rows of k and v, or pages).
struct pk_attn_args {
    const void *q, *k, *v;
    void *out;
    int64_t q_stride, k_stride, v_stride, out_stride;
    const int32_t *cu, *kv_len, *table;          // kv_len, table: null for packed prompts
    const float *sinks;
    float *lse;
    int n_tokens, n_req, max_q, window;
    int few_only;                                // requests of more than max_q rows: left to another launch
    int H, KVH, hd;
    int n_pages, page_shift, max_blocks;
    float scale2;                                // scale * log2 e
    int type, cache_type;
};

constexpr float PK_LOG2E = 1.4426950408889634f, PK_LN2 = 0.6931471805599453f;

// Request r's first row, number of rows and of positions, within the buffers
// whatever cu and kv_len hold.
struct pk_span {
    int row0, rows, kv;
};
__device__ __forceinline__ pk_span pk_request(const pk_attn_args &a, int r) {
    pk_span s;
    s.row0 = min(max(a.cu[r], 0), a.n_tokens);
    s.rows = max(min(max(a.cu[r + 1], 0), a.n_tokens) - s.row0, 0);
    s.kv = a.kv_len ? min(max(a.kv_len[r], 0), a.max_blocks << a.page_shift) : s.rows;
    return s;
}

// A workspace of `floats` and `counts` zeroed counters that kernels hand
// partial results through (and leave zeroed), grown outside captures.
int pk_attn_workspace(pk_engine *e, int64_t floats, int64_t counts);

// Rows of a request times query heads per KV head that one launch of k_attn_few
// holds; the launchers.
constexpr int PK_FEW_ROWS = 32;
int pk_launch_attn_few(pk_engine *e, const pk_attn_args &a);
// Requests with more than `cut` of these (the rest is k_attn_few's).
int pk_launch_attn_tile(pk_engine *e, const pk_attn_args &a, int cut, int max_kv);

// ───────── moves between the lanes of a wave ─────────
// Maximum and sum over the four lanes l, l ^ 16, l ^ 32, l ^ 48: a 32 x 32 or 16 x 16
// product leaves a column's rows in those.
__device__ __forceinline__ float pk_max_rows4(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float pk_sum_rows4(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
