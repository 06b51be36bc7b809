// pk_paged.hip — the paged KV cache: pages handed out to requests and the
// slots of a step's rows (pk_plan_pages), and the rows' rotation and way into
// the slots (pk_store_pages).
#include "pk_engine.h"
#include "pk_types.h"

pk_device_scope::pk_device_scope(int device) {
    int d = 0;
    if (hipGetDevice(&d) != hipSuccess || (d != device && hipSetDevice(device) != hipSuccess)) {
        pk_set_error("device %d cannot be made current", device);
        rc = PK_ERR_HIP;
    } else if (d != device) {
        cur = d;
    }
}
pk_device_scope::~pk_device_scope() {
    if (cur >= 0) (void)hipSetDevice(cur);
}

int pk_check_pages(const pk_pages &p, int act_type) {
    PK_CHECK(p.k_dev && p.v_dev, PK_ERR_ARG, "pages: null argument");
    PK_CHECK(pk_type_size(p.type) && pk_type_size(act_type), PK_ERR_ARG, "types %d, %d", act_type, p.type);
    PK_CHECK(act_type == PK_T_F32 || act_type == p.type, PK_ERR_UNSUPPORTED,
             "activations of type %d over pages of type %d (supported: the same type, or fp32 activations)", act_type,
             p.type);
    PK_CHECK(p.page_size >= 8 && p.page_size <= 256 && (p.page_size & (p.page_size - 1)) == 0, PK_ERR_UNSUPPORTED,
             "page_size %d (supported: powers of two from 8 to 256)", p.page_size);
    PK_CHECK(p.n_pages > 0 && (int64_t)p.n_pages * p.page_size <= INT32_MAX, PK_ERR_ARG, "%d pages of %d positions",
             p.n_pages, p.page_size);
    PK_CHECK(p.n_kv_heads > 0, PK_ERR_ARG, "n_kv_heads %d", p.n_kv_heads);
    PK_CHECK(p.head_dim >= 16 && p.head_dim <= 128 && p.head_dim % 16 == 0, PK_ERR_UNSUPPORTED,
             "head_dim %d (supported: multiples of 16 up to 128)", p.head_dim);
    PK_CHECK((((uintptr_t)p.k_dev | (uintptr_t)p.v_dev) & 15) == 0, PK_ERR_ARG, "pages: pointer not 16-byte aligned");
    return PK_OK;
}

int pk_check_rows(const void *p, int64_t stride, int heads, int hd, const char *what) {
    PK_CHECK(p, PK_ERR_ARG, "%s is null", what);
    PK_CHECK(((uintptr_t)p & 15) == 0, PK_ERR_ARG, "%s: pointer not 16-byte aligned", what);
    // (kernels take offsets of up to eight rows in 32 bits)
    PK_CHECK(stride % 8 == 0 && stride >= (int64_t)heads * hd && stride <= 1 << 26, PK_ERR_ARG,
             "%s: row stride %lld (a multiple of 8, at least %d heads of %d, at most 2^26)", what, (long long)stride, heads, hd);
    return PK_OK;
}

namespace {

// ───────────────────────── pages of a step ─────────────────────────
// One launch: bound by its latency (a step of 32 requests 6.3 us) and, for long
// prompts, by the write of the rows. Every workgroup adds up the requests' pages
// and rows for itself (three running sums over at most 4096 requests, ~1 us) and
// keeps row starts, page places and old lengths in LDS; then it moves the pages of
// its share of the requests and writes its share of the rows, four neighbours per
// thread, which find their request once and write 16 bytes (1000 requests, 1.3 M
// rows: 11.4 us, one row per thread 15.3). Two launches, sums first, would save the
// repeated sums but cost a launch more than those. What a workgroup reads of the
// table and the ring (pages below ceil(old / page_size); the ring's free entries)
// no other one writes; the ring's state is written by the workgroup that arrives
// last, when all have read it.
constexpr int PLAN_THREADS = 512, PLAN_REQ = 4096, PLAN_PER = PLAN_REQ / PLAN_THREADS, PLAN_ROWS = 4 * PLAN_THREADS;

// Sums that stay at 2^31 - 1 once they would pass it (more than any count they are
// compared with).
__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) { return min(a + b, 0x7fffffffu); }
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_sat_add(uint32_t v) {
    return sat_add(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, true));
}
// Sums over the block's threads up to this one.
template <int N>
__device__ __forceinline__ void block_sums(uint32_t (&v)[N], uint32_t (*part)[N]) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
        v[k] = dpp_sat_add<0x111, 0xf>(v[k]);                  // row_shr 1, 2, 4, 8
        v[k] = dpp_sat_add<0x112, 0xf>(v[k]);
        v[k] = dpp_sat_add<0x114, 0xf>(v[k]);
        v[k] = dpp_sat_add<0x118, 0xf>(v[k]);
        v[k] = dpp_sat_add<0x142, 0xa>(v[k]);                  // lane 15 of a row to the next row, 31 to the upper half
        v[k] = dpp_sat_add<0x143, 0xc>(v[k]);
    }
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 63)
#pragma unroll
        for (int k = 0; k < N; ++k) part[wave][k] = v[k];
    __syncthreads();
#pragma unroll
    for (int w = 0; w < PLAN_THREADS / 64; ++w)
        if (w < wave)
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] = sat_add(v[k], part[w][k]);
}

__global__ __launch_bounds__(PLAN_THREADS) void k_plan_pages(
    int n_req, int max_blocks, int n_pages, int shift, int max_tokens, const int32_t *__restrict__ old_len,
    const int32_t *__restrict__ new_len, int32_t *table, int32_t *ring, int32_t *state, int32_t *len, int32_t *cu_q,
    int32_t *__restrict__ slot, int32_t *__restrict__ pos, uint32_t *arrivals) {
    __shared__ int32_t cu[PLAN_REQ + 1], place[PLAN_REQ], old[PLAN_REQ];    // row starts; ring places of pages; old lengths
    __shared__ uint32_t part[PLAN_THREADS / 64][3];
    __shared__ int32_t stop, moved[2];                          // first request not served; pages taken, given
    const int t = threadIdx.x, most = max_blocks << shift, up = (1 << shift) - 1;
    const int count = min(max(state[1], 0), n_pages);
    const int head = (int)((uint32_t)state[0] % (uint32_t)n_pages);
    if (t == 0) stop = n_req;
    // a thread's requests are neighbours
    const int per = (n_req + PLAN_THREADS - 1) / PLAN_THREADS, r0 = t * per;
    uint32_t sum[3] = {0, 0, 0};                                // pages taken, rows, pages given
    int a[PLAN_PER], b[PLAN_PER];
#pragma unroll
    for (int i = 0; i < PLAN_PER; ++i) {
        a[i] = b[i] = 0;
        if (i >= per) break;
        if (r0 + i < n_req) {
            a[i] = min(max(old_len[r0 + i], 0), most);
            b[i] = min(max(new_len[r0 + i], 0), most);
        }
        const int d = ((b[i] + up) >> shift) - ((a[i] + up) >> shift);
        sum[0] = sat_add(sum[0], max(d, 0));
        sum[1] = sat_add(sum[1], max(b[i] - a[i], 0));
        sum[2] = sat_add(sum[2], max(-d, 0));
    }
    // sums before this thread's requests: those up to the thread before
    uint32_t at[3] = {sum[0], sum[1], sum[2]};
    block_sums(at, part);                                       // (its barrier also covers `stop`)
    uint32_t at0[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        at0[k] = (uint32_t)__shfl_up((int)at[k], 1);
        if ((t & 63) == 0) {
            at0[k] = 0;
            for (int w = 0; w < t >> 6; ++w) at0[k] = sat_add(at0[k], part[w][k]);
        }
        at[k] = at0[k];
    }
    // the sums only grow: from the first request that does not fit on, none that grows does
#pragma unroll
    for (int i = 0; i < PLAN_PER; ++i) {
        if (i >= per) break;
        const int d = ((b[i] + up) >> shift) - ((a[i] + up) >> shift);
        at[0] = sat_add(at[0], max(d, 0));
        at[1] = sat_add(at[1], max(b[i] - a[i], 0));
        if (r0 + i < n_req && (at[0] > (uint32_t)count || at[1] > (uint32_t)max_tokens)) atomicMin(&stop, r0 + i);
    }
    __syncthreads();
    const int last = stop;
#pragma unroll
    for (int k = 0; k < 3; ++k) at[k] = at0[k];
#pragma unroll
    for (int i = 0; i < PLAN_PER; ++i) {
        const int r = r0 + i;
        if (i >= per) break;
        if (r >= n_req) continue;
        old[r] = a[i];
        if (r <= last) cu[r] = (int32_t)at[1];
        if (r == last) moved[0] = (int32_t)at[0];
        const int d = ((b[i] + up) >> shift) - ((a[i] + up) >> shift);
        // (served requests' pages are at most `count` from the head; head, count < 2^28)
        const uint32_t x = (uint32_t)head + (d < 0 ? (uint32_t)count + at[2] : min(at[0], (uint32_t)count));
        place[r] = (int32_t)(x % (uint32_t)n_pages);
        at[0] = sat_add(at[0], max(d, 0));
        at[1] = sat_add(at[1], max(b[i] - a[i], 0));
        at[2] = sat_add(at[2], max(-d, 0));
        if (r == n_req - 1) {
            if (last == n_req) cu[n_req] = (int32_t)at[1], moved[0] = (int32_t)at[0];
            moved[1] = (int32_t)min(at[2], (uint32_t)n_pages);
        }
    }
    if (n_req == 0 && t == 0) cu[0] = moved[0] = moved[1] = 0;
    __syncthreads();
    // (requests behind the last one served have no rows)
    if (last < n_req) {
        for (int r = last + 1 + t; r <= n_req; r += PLAN_THREADS) cu[r] = cu[last];
        __syncthreads();
    }
    // The state is read; the last workgroup to have done so writes it, by a wave while the others
    // go on. Many arrive in two steps, at 16 words and then one (650 on one word take 10 us).
    if (t == PLAN_THREADS - 64) {
        const auto arrive = [&](uint32_t *c, uint32_t of) {
            if (of == 1) return true;
            const bool last_in = __hip_atomic_fetch_add(c, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u == of;
            if (last_in) __hip_atomic_store(c, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            return last_in;
        };
        const uint32_t group = blockIdx.x & 15;
        if (gridDim.x <= 32 ? arrive(arrivals, gridDim.x)
                            : arrive(arrivals + 16 * (1 + group), (gridDim.x + 15 - group) >> 4) && arrive(arrivals, 16)) {
            state[0] = (int32_t)(((uint32_t)head + (uint32_t)moved[0]) % (uint32_t)n_pages);
            state[1] = min(count - moved[0] + moved[1], n_pages);
        }
    }
    // entry k of the ring from a place on (k < n_pages)
    const auto from = [&](int place, int k) {
        const uint32_t x = (uint32_t)place + (uint32_t)k;
        return x >= (uint32_t)n_pages ? x - (uint32_t)n_pages : x;
    };

    // the pages: a wave per request
    const int lane = t & 63, waves = gridDim.x * (PLAN_THREADS / 64);
    for (int r = blockIdx.x * (PLAN_THREADS / 64) + (t >> 6); r < n_req; r += waves) {
        const int o = old[r], n = min(max(new_len[r], 0), most);
        const int ob = (o + up) >> shift, nb = (n + up) >> shift;
        int32_t *row = table + (int64_t)r * max_blocks;
        if (n > o) {
            if (r < last)
                for (int k = ob + lane; k < nb; k += 64) row[k] = ring[from(place[r], k - ob)];
        } else {
            for (int k = nb + lane; k < ob; k += 64) {
                ring[((uint32_t)place[r] + (uint32_t)(k - nb)) % (uint32_t)n_pages] = row[k];
                row[k] = -1;
            }
        }
        if (lane == 0) {
            len[r] = n > o && r >= last ? o : n;
            cu_q[r] = cu[r];
        }
    }
    if (blockIdx.x == 0 && t == 0) cu_q[n_req] = cu[n_req];

    // the rows
    const int total = cu[n_req];
    const bool wide = (((uintptr_t)slot | (uintptr_t)pos) & 15) == 0;
    // the last of the requests lo .. hi that starts at or before row i
    const auto find = [&](int i, int lo, int hi) {
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (cu[mid] <= i) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    };
    for (int64_t base = (int64_t)blockIdx.x * PLAN_ROWS; base < max_tokens; base += (int64_t)gridDim.x * PLAN_ROWS) {
        const int64_t i0 = base + t * 4;
        int p[4], s[4];
        const int32_t *src[4];                                  // the entry that names the row's page
        int r = -1, end = 0, off = 0, ob = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int64_t i = i0 + q;
            p[q] = 0;
            src[q] = nullptr;
            if (i >= total) continue;
            if (r < 0 || i >= end) {                            // (often the next request's)
                r = r >= 0 && cu[r + 2] > i ? r + 1 : find((int)i, r + 1, n_req - 1);
                end = cu[r + 1];
                const int o = old[r];
                off = o - cu[r];
                ob = (o + up) >> shift;
            }
            p[q] = off + (int)i;
            const int k = p[q] >> shift;
            src[q] = k < ob ? table + (int64_t)r * max_blocks + k : ring + from(place[r], k - ob);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) s[q] = src[q] ? *src[q] : -1;
#pragma unroll
        for (int q = 0; q < 4; ++q) s[q] = s[q] >= 0 && s[q] < n_pages ? (s[q] << shift) + (p[q] & up) : -1;
        if (wide && i0 + 3 < max_tokens) {
            *reinterpret_cast<int4 *>(slot + i0) = int4{s[0], s[1], s[2], s[3]};
            *reinterpret_cast<int4 *>(pos + i0) = int4{p[0], p[1], p[2], p[3]};
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (i0 + q < max_tokens) slot[i0 + q] = s[q], pos[i0 + q] = p[q];
        }
    }
}

// ───────────────────────── rows into their slots ─────────────────────────
// A thread takes eight elements of a head's lower half and the eight that
// they rotate with, or sixteen of a value head. Bound by HBM for many rows, by
// the launch for a decode step's.
constexpr int STORE_THREADS = 256;

template <typename A, typename C>
__global__ __launch_bounds__(STORE_THREADS) void k_store_pages(pk_kv_rows a, int rows_per_wg) {
    const int hd = a.pages.head_dim, half = hd >> 1, u = half >> 3, KVH = a.pages.n_kv_heads, H = a.n_heads;
    const int items = (H + 2 * KVH) * u, ps = a.pages.page_size;
    const int64_t n_slots = (int64_t)a.pages.n_pages * ps, r0 = (int64_t)blockIdx.x * rows_per_wg;
    const int rows = (int)min((int64_t)rows_per_wg, a.n_tokens - r0);
    for (int i = threadIdx.x; i < rows * items; i += STORE_THREADS) {
        const int row = i / items, it = i - row * items, head = it / u, j = (it - head * u) * 8;
        const int64_t t = r0 + row;
        const int slot = a.slot_dev[t], pos = a.pos_dev[t];
        if (slot < 0 || slot >= n_slots || (a.rope_dev && (pos < 0 || pos >= a.rope_len))) continue;
        const int kvh = head < H ? 0 : head < H + KVH ? head - H : head - H - KVH;
        const A *src = head < H ? (const A *)a.q_dev + t * a.q_stride + head * hd
                                : (head < H + KVH ? (const A *)a.k_dev + t * a.k_stride : (const A *)a.v_dev + t * a.v_stride) +
                                      kvh * hd;
        float x[8], y[8];
        pk_load8(src + j, x);
        pk_load8(src + half + j, y);
        if (a.rope_dev && head < H + KVH) {
            const float *cs = a.rope_dev + ((int64_t)pos * half + j) * 2;
            float c0[8], c1[8];
            pk_load8(cs, c0);
            pk_load8(cs + 8, c1);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float c = k < 4 ? c0[2 * k] : c1[2 * k - 8], s = k < 4 ? c0[2 * k + 1] : c1[2 * k - 7];
                const float r = __builtin_fmaf(x[k], c, -(y[k] * s));
                y[k] = __builtin_fmaf(x[k], s, y[k] * c);
                x[k] = r;
            }
        }
        if (head < H) {
            A *dst = (A *)a.q_out_dev + t * a.q_out_stride + head * hd;
            pk_store8(dst + j, x);
            pk_store8(dst + half + j, y);
        } else {
            C *dst = (C *)(head < H + KVH ? a.pages.k_dev : a.pages.v_dev) +
                     (((int64_t)(slot / ps) * KVH + kvh) * ps + (slot & (ps - 1))) * hd;
            pk_store8(dst + j, x);
            pk_store8(dst + half + j, y);
        }
    }
}

}  // namespace

extern "C" int pk_plan_pages(pk_engine *e, const pk_page_plan *p) {
    PK_CHECK(e && p, PK_ERR_ARG, "null argument");
    PK_CHECK(p->n_req >= 0 && p->max_tokens >= 0 && p->max_blocks > 0 && p->n_pages > 0, PK_ERR_ARG,
             "plan_pages: n_req %d, max_tokens %d, max_blocks %d, n_pages %d", p->n_req, p->max_tokens, p->max_blocks,
             p->n_pages);
    PK_CHECK(p->n_req <= PLAN_REQ, PK_ERR_UNSUPPORTED, "plan_pages: n_req %d (supported: up to %d)", p->n_req, PLAN_REQ);
    PK_CHECK(p->page_size >= 8 && p->page_size <= 256 && (p->page_size & (p->page_size - 1)) == 0, PK_ERR_UNSUPPORTED,
             "page_size %d (supported: powers of two from 8 to 256)", p->page_size);
    PK_CHECK((int64_t)p->n_pages * p->page_size <= INT32_MAX && (int64_t)p->max_blocks * p->page_size <= INT32_MAX,
             PK_ERR_ARG, "plan_pages: %d pages, tables of %d, of %d positions", p->n_pages, p->max_blocks, p->page_size);
    PK_CHECK(p->ring_dev && p->ring_state_dev && p->cu_q_dev, PK_ERR_ARG, "plan_pages: null argument");
    PK_CHECK(p->n_req == 0 || (p->old_len_dev && p->new_len_dev && p->table_dev && p->len_dev), PK_ERR_ARG,
             "plan_pages: null argument");
    PK_CHECK(p->max_tokens == 0 || (p->slot_dev && p->pos_dev), PK_ERR_ARG, "plan_pages: null argument");
    PK_CHECK(p->len_dev + p->n_req <= p->old_len_dev || p->old_len_dev + p->n_req <= p->len_dev || p->n_req == 0,
             PK_ERR_ARG, "plan_pages: len_dev overlaps old_len_dev");
    PK_CHECK(p->len_dev + p->n_req <= p->new_len_dev || p->new_len_dev + p->n_req <= p->len_dev || p->n_req == 0,
             PK_ERR_ARG, "plan_pages: len_dev overlaps new_len_dev");
    pk_device_scope dev(e->device);
    PK_TRY(dev.rc);
    // (three workgroups per CU at most: 256 to 1024 of them measured alike)
    const int64_t wgs = std::max<int64_t>(((int64_t)p->max_tokens + PLAN_ROWS - 1) / PLAN_ROWS, (p->n_req + 31) / 32);
    k_plan_pages<<<(unsigned)std::min<int64_t>(std::max<int64_t>(wgs, 1), 768), PLAN_THREADS, 0, e->stream>>>(
        p->n_req, p->max_blocks, p->n_pages, __builtin_ctz((unsigned)p->page_size), p->max_tokens, p->old_len_dev,
        p->new_len_dev, p->table_dev, p->ring_dev, p->ring_state_dev, p->len_dev, p->cu_q_dev, p->slot_dev, p->pos_dev,
        e->counters + PK_CTR_PLAN);
    PK_HIP(hipGetLastError());
    return PK_OK;
}

extern "C" int pk_store_pages(pk_engine *e, const pk_kv_rows *r) {
    PK_CHECK(e && r, PK_ERR_ARG, "null argument");
    PK_TRY(pk_check_pages(r->pages, r->type));
    const int hd = r->pages.head_dim, KVH = r->pages.n_kv_heads;
    PK_CHECK(r->n_tokens >= 0 && r->n_heads >= 0 && (int64_t)(r->n_heads + 2ll * KVH) * hd <= 1 << 20, PK_ERR_ARG,
             "store_pages: n_tokens %d, n_heads %d, n_kv_heads %d", r->n_tokens, r->n_heads, KVH);
    if (r->n_tokens == 0) return PK_OK;
    PK_CHECK(r->pos_dev && r->slot_dev, PK_ERR_ARG, "store_pages: null argument");
    if (r->n_heads) {
        PK_TRY(pk_check_rows(r->q_dev, r->q_stride, r->n_heads, hd, "q"));
        PK_TRY(pk_check_rows(r->q_out_dev, r->q_out_stride, r->n_heads, hd, "q_out"));
    }
    PK_TRY(pk_check_rows(r->k_dev, r->k_stride, KVH, hd, "k"));
    PK_TRY(pk_check_rows(r->v_dev, r->v_stride, KVH, hd, "v"));
    PK_CHECK(!r->rope_dev || (r->rope_len > 0 && ((uintptr_t)r->rope_dev & 15) == 0), PK_ERR_ARG,
             "store_pages: rope_len %d, or table not 16-byte aligned", r->rope_len);
    pk_device_scope dev(e->device);
    PK_TRY(dev.rc);
    // rows per workgroup: one pass of its threads over their items
    const int items = (r->n_heads + 2 * KVH) * (hd / 16), per = std::max(1, STORE_THREADS / items);
    const unsigned grid = (unsigned)(((int64_t)r->n_tokens + per - 1) / per);
#define PK_STORE(A, C) k_store_pages<A, C><<<grid, STORE_THREADS, 0, e->stream>>>(*r, per)
    PK_BY_TYPES(r->type, r->pages.type, PK_STORE);
#undef PK_STORE
    PK_HIP(hipGetLastError());
    return PK_OK;
}

extern "C" const float *pk_engine_rope(pk_engine *e, int *n_pos) {
    if (!e) {
        pk_set_error("engine is null");
        return nullptr;
    }
    if (n_pos) *n_pos = e->c.ctx_len;
    return e->rope;
}
