// pk_attn_few.hip — paged attention of requests with few rows: a decode step,
// or a few drafted tokens. Bound by the reads of K and V.
//
// The rows of a request times the query heads of one KV head are the columns
// of a product (at most 16 NQ of them); keys are its rows: S^T = K Q^T, O^T =
// V^T P^T. A lane of a 16 x 16 product holds one query's scores of 4 keys out of
// 16, which is how the second product takes its operand, so that probabilities
// never leave the registers; and the order of the head's elements in the first
// product, and of the keys in the second, is free, so that both operands are
// loaded straight from the pages, 8 or 16 bytes per lane, with no LDS between.
//
// The tiles of KT positions of all requests, U of them, are cut into chunks of
// about U / W: a request of up to a chunk is one item, a longer one several of
// equal length. A workgroup (per KV head) is one item, whatever the requests'
// lengths, and its waves take every fourth tile of it. Of a request of several
// items each leaves its part, and the workgroup that arrives last joins them in
// order. (Equal shares of one line of tiles instead, across requests, left a
// workgroup with the parts of several, one after the other: 32 requests with
// 128-position windows 23 us, as items 12.)
//
// Measured, 64 query heads over 8 of 64, the bytes of K and V per second: 32 requests of
// up to 8192 positions, bf16, 50 us, 3.8 TB/s; one of 100,001, fp32 over fp16, 51 us,
// 4.0 TB/s; 32 of 128-element heads 72 us, 4.3 TB/s; what is missing to a copy's 5.2 is the
// start (a workgroup's request, its pages, the first keys: four loads that wait for
// each other) and the join.
#include "pk_attention.h"

namespace {

constexpr int FEW_THREADS = 256, FEW_WAVES = FEW_THREADS / 64;

typedef float f32x4 __attribute__((ext_vector_type(4)));

// N elements of T as loaded: 4, 8 or 16 bytes at a time.
template <typename T, int N>
struct regs {
    typedef T type __attribute__((ext_vector_type(N)));
};

__device__ __forceinline__ f32x4 mfma(pk_f16x8 a, pk_f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma(pk_bf16x8 a, pk_bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// A value's planes: itself in T, or N values of T that add up to it (cut to 8 bits each
// for bf16; for fp16 rounded, the second the rest).
template <typename T, int N, typename V8>
__device__ __forceinline__ void planes(const V8 &x, typename regs<T, 8>::type (&p)[N]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (N == 1) {
            p[0][i] = (T)x[i];
        } else if constexpr (N == 2) {
            p[0][i] = (T)(float)x[i];
            p[1][i] = (T)((float)x[i] - (float)p[0][i]);
        } else {
            float v = (float)x[i];
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const uint32_t hi = __float_as_uint(v) & 0xffff0000u;
                p[n][i] = __builtin_bit_cast(T, (uint16_t)(hi >> 16));
                v = v - __uint_as_float(hi);
            }
        }
    }
}

// Positions per tile: a wave has a tile's keys (also the next one's) and values in
// registers, 256 of them per lane with two columns' worth of everything else.
// (32 positions where 64 fit: one row over 100,001 positions, fp32 over fp16, 63 us for 52; with
// three workgroups on a CU 59.)
constexpr int few_tile(int row_bytes, int nq) { return row_bytes <= 128 ? 64 / nq : row_bytes <= 256 ? 32 : 16; }
constexpr int FEW_PER_CU = 2;

// Not 0 where one of N values is an infinity or NaN (exponent all ones).
template <typename T, int N>
__device__ __forceinline__ uint32_t odd_row(const typename regs<T, N>::type &v) {
    constexpr uint32_t E = sizeof(T) == 4 ? 0x7f800000u : __is_same(T, pk_f16) ? 0x7c007c00u : 0x7f807f80u;
    constexpr uint32_t ONE = sizeof(T) == 4 ? 0x00800000u : __is_same(T, pk_f16) ? 0x04000400u : 0x00800080u;
    constexpr uint32_t TOP = sizeof(T) == 4 ? 0x80000000u : 0x80008000u;
    const auto w = __builtin_bit_cast(typename regs<uint32_t, N * (int)sizeof(T) / 4>::type, v);
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < N * (int)sizeof(T) / 4; ++i) any |= (w[i] & E) + ONE;
    return any & TOP;
}

// A request's tiles.
struct seg {
    pk_span s;
    int first, end, tiles;     // first position (a multiple of KT), the one behind the last, tiles (0: no rows; at least 1 otherwise)
};
template <int KT>
__device__ __forceinline__ seg few_seg(const pk_attn_args &a, int r) {
    seg g;
    g.s = pk_request(a, r);
    const int p0 = max(g.s.kv - g.s.rows, 0);                  // the first row's position
    g.first = a.window > 0 ? max(p0 - a.window + 1, 0) & ~(KT - 1) : 0;
    g.end = max(g.s.kv - max(g.s.rows - a.max_q, 0), 0);       // (rows beyond max_q are not computed: nor their positions read)
    g.tiles = g.s.rows && !(a.few_only && g.s.rows > a.max_q) ? max((g.end - g.first + KT - 1) / KT, 1) : 0;
    return g;
}

constexpr int FEW_TRIES = 8, FEW_KEPT = 4;
__device__ __forceinline__ int try_chunk(int64_t share, int k) {
    return (int)min(share + share * (k < 5 ? k : 2 * k - 4) / 8, (int64_t)INT32_MAX / 2);     // 1, 9/8 .. 12/8, 14/8, 2, 18/8
}

// Sums over the lanes up to this one.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, true);
}
__device__ __forceinline__ int wave_scan(int v) {
    v = dpp_add<0x111, 0xf>(v);                                // row_shr 1, 2, 4, 8
    v = dpp_add<0x112, 0xf>(v);
    v = dpp_add<0x114, 0xf>(v);
    v = dpp_add<0x118, 0xf>(v);
    v = dpp_add<0x142, 0xa>(v);                                // lane 15 of a row to the next row, 31 to the upper half
    return dpp_add<0x143, 0xc>(v);
}

// A workgroup's item: request r (< 0: none), part `it` of n_it, the first of them part0 among the
// parts of split requests.
struct piece {
    int r, it, n_it, part0;
};
struct find_lds {
    double tiles[FEW_WAVES];
    int items[FEW_WAVES][2], found[4];
};
template <int KT>
__device__ __forceinline__ piece few_find(const pk_attn_args &a, int W, find_lds &lds) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // equal chunks of the one request: nothing to search (37 positions 8.7 us with the
    // search, 7.6 without)
    if (a.n_req == 1) {
        const int t = few_seg<KT>(a, 0).tiles, chunk = max((t + W - 1) / W, FEW_WAVES), n = (t + chunk - 1) / chunk;
        return {(int)blockIdx.x < n ? 0 : -1, (int)blockIdx.x, max(n, 1), 0};
    }
    // Up to 64 FEW_KEPT requests: each wave finds it for itself, a lane for every 64th of the
    // requests, with no barriers (~1 us). More: a thread for every 256th.
    const bool wide = a.n_req > 64 * FEW_KEPT;
    const int id = wide ? tid : lane, per = wide ? (a.n_req + FEW_THREADS - 1) / FEW_THREADS : (a.n_req + 63) >> 6;
    const auto tiles_of = [&](int i) { return i < per && id * per + i < a.n_req ? few_seg<KT>(a, id * per + i).tiles : 0; };
    int tiles[FEW_KEPT];                                        // (the first FEW_KEPT of a lane: read once)
#pragma unroll
    for (int i = 0; i < FEW_KEPT; ++i) tiles[i] = tiles_of(i);
    const auto each = [&](auto f) {                             // f(i, tiles) in order, until it is true
#pragma unroll
        for (int i = 0; i < FEW_KEPT; ++i)
            if (i < per && f(i, tiles[i])) return;
        for (int i = FEW_KEPT; i < per; ++i)
            if (f(i, tiles_of(i))) return;
    };
    double all = 0.0;
    each([&](int, int n) { all += n; return false; });
    all = pk_wave_sum_d(all);                                   // (exact)
    if (wide) {
        if (lane == 0) lds.tiles[wave] = all;
        __syncthreads();
        all = lds.tiles[0] + lds.tiles[1] + lds.tiles[2] + lds.tiles[3];
    }
    // The shortest chunk, from an equal share of the tiles for each of W workgroups on, with which
    // the items are at most W (give or take one for the division): all run at once, the
    // longest of them for as little as such chunks allow. More requests than W (or than
    // are worth the search): several rounds, of twice the share.
    const int64_t share = max(((int64_t)all + W - 1) / W, (int64_t)FEW_WAVES);
    int chunk = try_chunk(share, 6);
    if (a.n_req <= W && !wide) {
        float n[FEW_TRIES] = {};
        each([&](int, int t) {
#pragma unroll
            for (int k = 0; k < FEW_TRIES; ++k) n[k] += __builtin_ceilf((float)t * __builtin_amdgcn_rcpf((float)try_chunk(share, k)) * 0.999999f);
            return false;
        });
        int k = 0;
#pragma unroll
        for (int y = 0; y < FEW_TRIES - 1; ++y) k += k == y && pk_wave_sum_f(n[y]) > (float)W;
        chunk = try_chunk(share, k);
    }
    const auto items_of = [&](int t) { return (int)(((uint32_t)t + (uint32_t)chunk - 1) / (uint32_t)chunk); };
    int items = 0, parts = 0;                                   // of this lane's requests; parts: of the split ones
    each([&](int, int t) {
        const int n = items_of(t);
        items += n;
        parts += n > 1 ? n : 0;
        return false;
    });
    int at = wave_scan(items), part_at = wave_scan(parts);
    if (wide) {
        if (lane == 63) lds.items[wave][0] = at, lds.items[wave][1] = part_at;
        if (tid == 0) lds.found[0] = -1;
        __syncthreads();
        for (int i = 0; i < wave; ++i) at += lds.items[i][0], part_at += lds.items[i][1];
    }
    at -= items;
    part_at -= parts;
    const uint64_t whose = __ballot((int)blockIdx.x >= at && (int)blockIdx.x < at + items);
    int my_r = 0, my_n = 0;
    if (whose >> lane & 1)
        each([&](int i, int t) {
            my_n = items_of(t);
            my_r = id * per + i;
            if ((int)blockIdx.x < at + my_n) return true;
            at += my_n;
            part_at += my_n > 1 ? my_n : 0;
            return false;
        });
    const int src = whose ? __ffsll((unsigned long long)whose) - 1 : 0;
    int r = whose ? __builtin_amdgcn_readlane(my_r, src) : -1, n_it = __builtin_amdgcn_readlane(my_n, src);
    int it = (int)blockIdx.x - __builtin_amdgcn_readlane(at, src), part0 = __builtin_amdgcn_readlane(part_at, src);
    if (wide) {
        if (whose && lane == 0) lds.found[0] = r, lds.found[1] = n_it, lds.found[2] = it, lds.found[3] = part0;
        __syncthreads();
        r = __builtin_amdgcn_readfirstlane(lds.found[0]), n_it = __builtin_amdgcn_readfirstlane(lds.found[1]);
        it = __builtin_amdgcn_readfirstlane(lds.found[2]), part0 = __builtin_amdgcn_readfirstlane(lds.found[3]);
    }
    return {r, it, n_it, part0};
}

template <typename A, typename C, int HDP, int NQ>
__global__ __launch_bounds__(FEW_THREADS, FEW_PER_CU) void k_attn_few(pk_attn_args a, int W, int max_parts, float *part, uint32_t *count) {
    constexpr bool F32 = sizeof(C) == 4;                        // fp32 cache: fp32 products
    // fp32 queries and probabilities over a 16-bit cache: as planes of the cache's type, whose
    // products are exact. bf16: three, 8 bits each. fp16: two, 11 bits each, of values
    // scaled to at most 2^14, so that the low plane's last bit is at 2^-38 of that. With 16-bit
    // queries a probability is rounded once, to the type that the product takes and the result
    // has; the sum of them takes it unrounded.
    constexpr int QP = F32 || sizeof(A) == 2 ? 1 : __is_same(C, pk_f16) ? 2 : 3;
    constexpr float SHIFT = __is_same(C, pk_f16) ? 14.0f : 0.0f;    // probabilities are at most 2^SHIFT
    typedef typename regs<C, 8>::type c8;
    constexpr int KT = few_tile(HDP * (int)sizeof(C), NQ), NB = KT / 16;
    constexpr int KE = HDP / 4, KV8 = KE / 8;                   // elements of a key per lane, in vectors of 8
    constexpr int VE = HDP / 16;                                // elements of a value per lane
    constexpr int COLS = 16 * NQ, LD = HDP + 4;
    typedef typename regs<C, 8>::type k8;
    typedef typename regs<C, VE>::type vrow;

    __shared__ __attribute__((aligned(16))) float so[FEW_WAVES][COLS][LD];
    __shared__ float sm[FEW_WAVES][COLS], sl[FEW_WAVES][COLS];
    __shared__ find_lds lds;
    __shared__ int last_in;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, m16 = lane & 15;
    const int kvh = blockIdx.y, G = a.H / a.KVH, hd = a.hd;
    const int ps = 1 << a.page_shift;

    const auto [r, it, n_it, part0] = few_find<KT>(a, W, lds);
    if (r < 0) return;
    const seg sg = few_seg<KT>(a, r);
    const int t0 = (int)((int64_t)sg.tiles * it / n_it), t1 = (int)((int64_t)sg.tiles * (it + 1) / n_it);
    {
        const int rows = min(sg.s.rows, min(a.max_q, COLS / G)), cols = rows * G;
        const int p_first = sg.s.kv - sg.s.rows, p_last = p_first + rows - 1;
        const int32_t *tab = a.table + (int64_t)r * a.max_blocks;

        // ── the queries: lane (m16, g) holds elements g KE .. of column m16 ──
        typedef typename regs<A, 8>::type q8;
        c8 q[NQ][QP][KV8];
        int pos[NQ];
        float scale2[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const int c = n * 16 + m16, i = c / G;
            pos[n] = c < cols ? p_first + i : p_last;
            const A *src = (const A *)a.q + (int64_t)(sg.s.row0 + i) * a.q_stride + ((int64_t)kvh * G + (c - i * G)) * hd;
            q8 v[KV8];
#pragma unroll
            for (int s = 0; s < KV8; ++s) {
                const int e = g * KE + 8 * s;
                v[s] = q8{};
                if (c < cols && e < hd) v[s] = *reinterpret_cast<const q8 *>(src + e);
            }
            scale2[n] = a.scale2;
            if constexpr (QP == 2) {                            // to a largest magnitude in [2^13, 2^14)
                float top = 0.0f;
#pragma unroll
                for (int s = 0; s < KV8; ++s)
#pragma unroll
                    for (int i = 0; i < 8; ++i) top = fmaxf(top, __builtin_fabsf((float)v[s][i]));
                top = pk_max_rows4(top);
                const int k = min(max(14 - __builtin_amdgcn_frexp_expf(top), -114), 110);
                const float up = __builtin_ldexpf(1.0f, k);
#pragma unroll
                for (int s = 0; s < KV8; ++s) v[s] *= up;
                scale2[n] = a.scale2 * __builtin_ldexpf(1.0f, -k);
            }
#pragma unroll
            for (int s = 0; s < KV8; ++s) {
                c8 p[QP];
                planes<C, QP>(v[s], p);
#pragma unroll
                for (int x = 0; x < QP; ++x) q[n][x][s] = p[x];
            }
        }

        f32x4 o[NQ][VE];
        float mx[NQ], ls[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            mx[n] = -INFINITY;
            ls[n] = 0.0f;
#pragma unroll
            for (int c = 0; c < VE; ++c) o[n][c] = f32x4{0, 0, 0, 0};
        }

        // Page of position j (a position past the end or a page that is none: page 0, and the bit of j not set)
        const auto look = [&](int t, uint64_t &ok) {
            const int j = sg.first + t * KT + (lane & (KT - 1));
            const int pg = tab[min(j, max(sg.end - 1, 0)) >> a.page_shift];
            const bool good = j < sg.end && pg >= 0 && pg < a.n_pages;
            ok = __ballot(good);
            return good ? pg : 0;
        };
        const auto row_at = [&](int pg, int j) {                // element offset of position j's row on page pg
            return ((((int64_t)pg * a.KVH + kvh) << a.page_shift) + (j & (ps - 1))) * hd;
        };
        k8 k[NB][KV8];
        const auto load_k = [&](int t, int pgs) {
            const int base = sg.first + t * KT;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int pg = __shfl(pgs, b * 16 + m16);
                const C *src = (const C *)a.k + row_at(pg, base + b * 16 + m16);
#pragma unroll
                for (int s = 0; s < KV8; ++s) {
                    const int e = g * KE + 8 * s;
                    k[b][s] = *reinterpret_cast<const k8 *>(src + (e < hd ? e : 0));
                }
            }
        };

        int t = t0 + wave;
        uint64_t ok = 0, ok_next = 0;
        int pgs = 0, pgs_next = 0;
        if (t < t1) {
            pgs = look(t, ok);
            load_k(t, pgs);
            if (t + FEW_WAVES < t1) pgs_next = look(t + FEW_WAVES, ok_next);
        }
        for (; t < t1; t += FEW_WAVES) {
            const int base = sg.first + t * KT;
            // V: lane (m16, g) elements VE m16 .. of the keys 16 b + 4 g + i
            vrow v[NB][4];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int j = base + b * 16 + 4 * g, pg = __shfl(pgs, b * 16 + 4 * g);
                const C *src = (const C *)a.v + row_at(pg, j) + (VE * m16 < hd ? VE * m16 : 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[b][i] = *reinterpret_cast<const vrow *>(src + i * hd);
            }
            // S^T
            f32x4 s[NQ][NB];
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int b = 0; b < NB; ++b) s[n][b] = f32x4{0, 0, 0, 0};
            if (hd < HDP) {                                     // elements past the head count nothing
#pragma unroll
                for (int x = 0; x < KV8; ++x)
                    if (g * KE + 8 * x >= hd)
#pragma unroll
                        for (int b = 0; b < NB; ++b) k[b][x] = k8{};
            }
#pragma unroll
            for (int x = 0; x < KV8; ++x)
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
                        if constexpr (F32) {
#pragma unroll
                            for (int e = 0; e < 8; ++e) s[n][b] = mfma(k[b][x][e], q[n][0][x][e], s[n][b]);
                        } else {
#pragma unroll
                            for (int y = 0; y < QP; ++y) s[n][b] = mfma(k[b][x], q[n][y][x], s[n][b]);
                        }
                    }
            const uint64_t ok_now = ok;
            if (t + FEW_WAVES < t1) {
                load_k(t + FEW_WAVES, pgs_next);
                pgs = pgs_next;
                ok = ok_next;
                if (t + 2 * FEW_WAVES < t1) pgs_next = look(t + 2 * FEW_WAVES, ok_next);
            }
            // tiles that some row does not see whole
            const uint64_t all = KT == 64 ? ~0ull : (1ull << KT) - 1;
            const bool masked = (ok_now & all) != all || base + KT - 1 > p_first || (a.window > 0 && base <= p_last - a.window);
            uint64_t odd = 0;                                   // keys with values that are added one by one
            if (masked) {
                // (the empty asm keeps these branches: as selects they would be work of every tile)
                if (base + KT - 1 > p_first)
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
                        int upto = pos[n] - base - 4 * g;
                        asm volatile("" : "+v"(upto));
#pragma unroll
                        for (int b = 0; b < NB; ++b)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (b * 16 + i > upto) s[n][b][i] = -INFINITY;
                    }
                if (a.window > 0 && base <= p_last - a.window)
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
                        int from = pos[n] - a.window - base - 4 * g;
                        asm volatile("" : "+v"(from));
#pragma unroll
                        for (int b = 0; b < NB; ++b)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (b * 16 + i <= from) s[n][b][i] = -INFINITY;
                    }
                if ((ok_now & all) != all) {
                    uint64_t mine = ok_now >> (4 * g);
                    asm volatile("" : "+v"(mine));
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const bool there = mine >> (b * 16 + i) & 1;
#pragma unroll
                            for (int n = 0; n < NQ; ++n)
                                if (!there) s[n][b][i] = -INFINITY;
                        }
                }
            }
            // Values that are not finite: with planes they meet zeros, and where some rows do not
            // see them (or the place holds no position), zero probabilities.
            if (masked || QP > 1) {
                uint32_t any = 0;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) any |= odd_row<C, VE>(v[b][i]);
                if (__any(any != 0 && VE * m16 < hd)) {
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int j = base + b * 16 + 4 * g + i;
                            const bool every = (ok_now >> (j - base) & 1) && j <= p_first && (a.window <= 0 || j > p_last - a.window);
                            const uint64_t who = __ballot(odd_row<C, VE>(v[b][i]) != 0 && VE * m16 < hd && (QP > 1 || !every));
#pragma unroll
                            for (int gg = 0; gg < 4; ++gg)
                                if (who >> (16 * gg) & 0xffff) odd |= 1ull << (b * 16 + 4 * gg + i);
                            if (odd >> (b * 16 + 4 * g + i) & 1) v[b][i] = vrow{};
                        }
                }
            }
            // the running maximum, and probabilities in place of the scores
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                float top = s[n][0][0];
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) top = fmaxf(top, s[n][b][i]);
                top = pk_max_rows4(top) * scale2[n] - SHIFT;
                const float mn = fmaxf(mx[n], top);
                // (nothing seen yet: any finite value keeps exp2 at 0)
                const float ref = mn == -INFINITY ? 0.0f : mn, f = __builtin_amdgcn_exp2f(mx[n] - ref);
                mx[n] = mn;
                float sum = 0.0f;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][b][i], scale2[n], -ref));
                        s[n][b][i] = p;
                        sum += p;
                    }
                ls[n] = __builtin_fmaf(ls[n], f, sum);
#pragma unroll
                for (int c = 0; c < VE; ++c) o[n][c] *= f;
            }
            // O^T
            if constexpr (F32) {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int c = 0; c < VE; ++c)
#pragma unroll
                            for (int n = 0; n < NQ; ++n) o[n][c] = mfma(v[b][i][c], s[n][b][i], o[n][c]);
            } else {
#pragma unroll
                for (int b = 0; b < NB; b += 2) {
                    c8 p[NQ][QP];
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
                        typename regs<float, 8>::type x;
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[i] = s[n][b][i], x[4 + i] = s[n][b + 1][i];
                        planes<C, QP>(x, p[n]);
                    }
#pragma unroll
                    for (int c = 0; c < VE; ++c) {
                        c8 vt;
#pragma unroll
                        for (int i = 0; i < 4; ++i) vt[i] = v[b][i][c], vt[4 + i] = v[b + 1][i][c];
#pragma unroll
                        for (int n = 0; n < NQ; ++n)
#pragma unroll
                            for (int x = 0; x < QP; ++x) o[n][c] = mfma(vt, p[n][x], o[n][c]);
                    }
                }
            }
            // values that are not finite, on the rows that see them
            while (odd) {
                const int jj = __ffsll((unsigned long long)odd) - 1, j = base + jj;
                odd &= odd - 1;
                if (!(ok_now >> jj & 1)) continue;
                const int pg = tab[j >> a.page_shift];          // (a page: `there`)
                const C *src = (const C *)a.v + row_at(pg, j);
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    float p = 0.0f;
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (b == jj >> 4 && i == (jj & 3)) p = s[n][b][i];
                    p = __shfl(p, (jj & 12) * 4 + m16);
                    if (j <= pos[n] && (a.window <= 0 || j > pos[n] - a.window))
#pragma unroll
                        for (int c = 0; c < VE; ++c)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int e = VE * (4 * g + i) + c;
                                if (e < hd) o[n][c][i] = __builtin_fmaf(p, (float)src[e], o[n][c][i]);
                            }
                }
            }
        }

        // a column's four elements from e on, and its lse
        const auto finish = [&](const seg &sg, int kvh, int G, int c, int e, const f32x4 &acc, float l, float ref) {
            const int i = c / G, h = kvh * G + (c - i * G);
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const int64_t row = sg.s.row0 + i;
            typename regs<A, 4>::type v;
#pragma unroll
            for (int z = 0; z < 4; ++z) v[z] = (A)(acc[z] * inv);
            *reinterpret_cast<typename regs<A, 4>::type *>((A *)a.out + row * a.out_stride + (int64_t)h * hd + e) = v;
            if (a.lse && e == 0) a.lse[row * a.H + h] = l == 0.0f ? -INFINITY : (ref + __builtin_amdgcn_logf(l)) * PK_LN2;
        };
        // ── the waves' parts, joined ──
        __syncthreads();                                        // (so: the previous request's reads)
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const float l = pk_sum_rows4(ls[n]);
            const int c = n * 16 + m16;
            if (g == 0) sm[wave][c] = mx[n], sl[wave][c] = l;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < VE; ++e) so[wave][c][VE * (4 * g + i) + e] = o[n][e][i];
        }
        __syncthreads();
        const bool whole = n_it == 1;
        const int quads = hd >> 2;
        // a part: m and l of each column, then its sums
        constexpr int PART = COLS * (HDP + 2);
        float *first = part + ((int64_t)kvh * max_parts + part0) * PART, *slot = first + it * PART;
        for (int x = tid; x < cols * quads; x += FEW_THREADS) {
            const int c = x / quads, e = (x - c * quads) * 4;
            float mm = -INFINITY;
#pragma unroll
            for (int i = 0; i < FEW_WAVES; ++i) mm = fmaxf(mm, sm[i][c]);
            const int i = c / G, h = kvh * G + (c - i * G);
            float ref = mm == -INFINITY ? 0.0f : mm, l = 0.0f;
            const float sk = whole && a.sinks ? a.sinks[h] * PK_LOG2E : -INFINITY;
            if (sk > ref || (mm == -INFINITY && sk > -INFINITY)) ref = sk;
            f32x4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int y = 0; y < FEW_WAVES; ++y) {
                const float f = __builtin_amdgcn_exp2f(sm[y][c] - ref);
                l = __builtin_fmaf(sl[y][c], f, l);
                const f32x4 ov = *reinterpret_cast<const f32x4 *>(&so[y][c][e]);
#pragma unroll
                for (int z = 0; z < 4; ++z) acc[z] = __builtin_fmaf(ov[z], f, acc[z]);
            }
            if (whole) {
                finish(sg, kvh, G, c, e, acc, l + __builtin_amdgcn_exp2f(sk - ref), ref);
            } else {
                const uint64_t *b = reinterpret_cast<const uint64_t *>(&acc);
                uint64_t *p = (uint64_t *)(slot + 2 * COLS + c * HDP + e);
                // past the L2: another XCD's workgroup may join
                __hip_atomic_store(p, b[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __hip_atomic_store(p + 1, b[1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                if (e == 0)
                    __hip_atomic_store((uint64_t *)slot + c, (uint64_t)__float_as_uint(l) << 32 | __float_as_uint(mm), __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
            }
        }
        if (!whole) {
            uint32_t *cnt = count + (int64_t)kvh * max_parts + part0;
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            if (tid == 0) {
                const uint32_t was = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                last_in = was == (uint32_t)(n_it - 1);
                if (last_in) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            __syncthreads();
            if (last_in) {
                // (all loads past the L2)
                const auto at = [&](int y) { return (const uint64_t *)(first + y * PART); };
                const auto ld = [](const uint64_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
                const int np = n_it;
                // four elements of a column per thread, the parts over as many groups of threads as
                // there are, 8 of a group's parts in flight: a running reference, the sum and the
                // sums of values, in the order of the parts. (References and sums first, in
                // a pass of their own: a round trip more, 1 us.)
                const int items = cols * quads, groups = max(1, FEW_THREADS / items), grp = tid / items;
                f32x4 *sums = reinterpret_cast<f32x4 *>(&so[0][0][0]);
                float *ms = reinterpret_cast<float *>(sums + FEW_THREADS), *ls = ms + FEW_THREADS;
                static_assert(sizeof(so) >= FEW_THREADS * 24);
                const auto add = [](float &top, float &l, f32x4 &acc, float m, float lp, const f32x4 &v) {
                    // (a factor of 0 stays one beside an infinity)
                    const float mn = fmaxf(top, m), ref = mn == -INFINITY ? 0.0f : mn;
                    const float f0 = __builtin_amdgcn_exp2f(top - ref), f1 = __builtin_amdgcn_exp2f(m - ref);
                    top = mn;
                    l = __builtin_fmaf(lp, f1, l * f0);
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        if (f0 != 1.0f) acc[z] = f0 == 0.0f ? 0.0f : acc[z] * f0;
                        if (f1 != 0.0f) acc[z] = __builtin_fmaf(v[z], f1, acc[z]);
                    }
                };
                const auto end = [&](int c, int e, float top, float l, f32x4 acc) {
                    const float sk = a.sinks ? a.sinks[kvh * G + c % G] * PK_LOG2E : -INFINITY;
                    add(top, l, acc, sk, sk > -INFINITY ? 1.0f : 0.0f, f32x4{0, 0, 0, 0});
                    finish(sg, kvh, G, c, e, acc, l, top == -INFINITY ? 0.0f : top);
                };
                for (int x = groups > 1 ? tid - grp * items : tid; x < items && grp < groups; x += FEW_THREADS) {
                    const int c = x / quads, e = (x - c * quads) * 4;
                    float top = -INFINITY, l = 0.0f;
                    f32x4 acc = {0, 0, 0, 0};
                    for (int y0 = grp; y0 < np; y0 += 8 * groups) {
                        uint64_t ml[8], v[8][2];
#pragma unroll
                        for (int y = 0; y < 8; ++y) {
                            const uint64_t *p = at(min(y0 + y * groups, np - 1));
                            ml[y] = ld(p + c);
                            v[y][0] = ld(p + (2 * COLS + c * HDP + e) / 2);
                            v[y][1] = ld(p + (2 * COLS + c * HDP + e) / 2 + 1);
                        }
#pragma unroll
                        for (int y = 0; y < 8; ++y)
                            if (y0 + y * groups < np)
                                add(top, l, acc, __uint_as_float((uint32_t)ml[y]), __uint_as_float((uint32_t)(ml[y] >> 32)),
                                    *reinterpret_cast<const f32x4 *>(v[y]));
                    }
                    if (groups > 1) sums[tid] = acc, ms[tid] = top, ls[tid] = l;
                    else end(c, e, top, l, acc);
                }
                if (groups > 1) {
                    __syncthreads();
                    if (tid < items) {
                        f32x4 acc = sums[tid];
                        float top = ms[tid], l = ls[tid];
                        for (int y = 1; y < groups; ++y) add(top, l, acc, ms[y * items + tid], ls[y * items + tid], sums[y * items + tid]);
                        const int c = tid / quads;
                        end(c, (tid - c * quads) * 4, top, l, acc);
                    }
                }
            }
        }
    }
}

template <typename A, typename C, int HDP, int NQ>
int launch(pk_engine *e, const pk_attn_args &a, int64_t tiles) {
    // W: two workgroups on every CU. The items are at most W chunks and one for each request,
    // and never more than the tiles; the split requests' parts at most 2 W, since each of them is
    // longer than a chunk
    const int64_t slots = (FEW_PER_CU * (int64_t)e->n_cu + a.KVH - 1) / a.KVH;
    // (Requests up to twice as many: two rounds of half as long chunks. 48 requests of up to 4000
    // positions, 16 KV heads of 128, 134 us, 177 with one round's chunks; 70 of up to 8000, 8 of 64,
    // 88 / 94; but 200 of up to 2000 92 / 89.)
    const int W = (int)std::max<int64_t>(slots, 1) * (a.n_req > slots && a.n_req <= 2 * slots ? 2 : 1);
    const int64_t grid = std::min<int64_t>(W + (int64_t)a.n_req, std::max<int64_t>(tiles, 1));
    PK_TRY(pk_attn_workspace(e, (int64_t)a.KVH * 2 * W * 16 * NQ * (HDP + 2), (int64_t)a.KVH * 2 * W));
    k_attn_few<A, C, HDP, NQ><<<dim3((unsigned)grid, (unsigned)a.KVH), FEW_THREADS, 0, e->stream>>>(a, W, 2 * W, e->att_ws, e->att_cnt);
    PK_HIP(hipGetLastError());
    return PK_OK;
}

template <typename A, typename C>
int by_shape(pk_engine *e, const pk_attn_args &a, int64_t positions) {
    const int rows = a.max_q * (a.H / a.KVH);
    const int kt = few_tile((a.hd <= 64 ? 64 : 128) * (int)sizeof(C), rows <= 16 ? 1 : 2);
    const int64_t tiles = (int64_t)a.n_req * ((positions + kt - 1) / kt + 1);
    if (a.hd <= 64) return rows <= 16 ? launch<A, C, 64, 1>(e, a, tiles) : launch<A, C, 64, 2>(e, a, tiles);
    return rows <= 16 ? launch<A, C, 128, 1>(e, a, tiles) : launch<A, C, 128, 2>(e, a, tiles);
}

}  // namespace

int pk_launch_attn_few(pk_engine *e, const pk_attn_args &a) {
    // positions that a request's rows may read: its table's, or a window and a tile's rest
    const int64_t cap = (int64_t)a.max_blocks << a.page_shift;
    const int64_t positions = a.window > 0 ? std::min<int64_t>(cap, (int64_t)a.window + a.max_q + 64) : cap;
#define PK_FEW(A, C) return by_shape<A, C>(e, a, positions)
    PK_BY_TYPES(a.type, a.cache_type, PK_FEW);
#undef PK_FEW
}
