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
// The positions of all requests, in tiles of KT, lie behind each other on one
// line, of which each workgroup takes an equal share (per KV head), whatever
// the requests' lengths; its waves take every fourth tile. A request that ends
// inside one share is written out there; of one that spans several, each
// workgroup leaves its part, and the one that arrives last joins them in the
// line's order.
#include "pk_attention.h"

namespace {

constexpr int FEW_THREADS = 256, FEW_WAVES = FEW_THREADS / 64;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

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

// Positions per tile: a wave has a tile's keys (also the next one's) and values in
// registers, 256 of them per lane with two columns' worth of everything else.
constexpr int few_tile(int row_bytes, int nq) { return row_bytes <= 128 ? 64 / nq : row_bytes <= 256 ? 32 : 16; }

template <typename T>
__device__ __forceinline__ bool not_finite(T v) {
    return !(__builtin_fabsf((float)v) <= 3.4028234e38f);
}

// The tiles of a request, and of those before it, on the line.
struct seg {
    pk_span s;
    int first, tiles;          // first position (a multiple of KT), tiles (0: no rows; at least 1 otherwise)
};
template <int KT>
__device__ __forceinline__ seg few_seg(const pk_attn_args &a, int r) {
    seg g;
    g.s = pk_request(a, r);
    const int p0 = max(g.s.kv - g.s.rows, 0);                  // the first row's position
    g.first = a.window > 0 ? max(p0 - a.window + 1, 0) & ~(KT - 1) : 0;
    g.tiles = g.s.rows && !(a.few_only && g.s.rows > a.max_q) ? max((g.s.kv - g.first + KT - 1) / KT, 1) : 0;
    return g;
}

// Share of the line: worker w of W takes tiles [w U / W, (w + 1) U / W).
__device__ __forceinline__ int64_t share(int64_t U, int w, int W) { return U * w / W; }
// The worker that has tile u.
__device__ __forceinline__ int owner(int64_t u, int64_t U, int W) {
    int w = (int)(((u + 1) * W - 1) / U);                       // share(w) <= u < share(w + 1)
    return w;
}

template <typename A, typename C, int HDP, int NQ>
__global__ __launch_bounds__(FEW_THREADS, 2) void k_attn_few(pk_attn_args a, float *part, uint32_t *count) {
    constexpr bool F32 = sizeof(A) == 4;                        // fp32 products, the cache widened
    constexpr int KT = few_tile(HDP * (int)sizeof(C), NQ), NB = KT / 16;
    constexpr int KE = HDP / 4, KV8 = KE / 8;                   // elements of a key per lane, in vectors of 8
    constexpr int VE = HDP / 16;                                // elements of a value per lane
    constexpr int COLS = 16 * NQ, LD = HDP + 4;
    typedef typename regs<C, 8>::type k8;
    typedef typename regs<C, VE>::type vrow;

    __shared__ __attribute__((aligned(16))) float so[FEW_WAVES][COLS][LD];
    __shared__ float sm[FEW_WAVES][COLS], sl[FEW_WAVES][COLS];
    __shared__ int64_t line[FEW_THREADS / 64 + 1];
    __shared__ int64_t start_at;
    __shared__ int start_r, last_in;

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, m16 = lane & 15;
    const int W = gridDim.x, kvh = blockIdx.y, G = a.H / a.KVH, hd = a.hd;
    const int ps = 1 << a.page_shift;

    // ── this workgroup's share of the line ──
    const int per = (a.n_req + FEW_THREADS - 1) / FEW_THREADS;
    int64_t mine = 0;
    for (int i = 0; i < per; ++i)
        if (tid * per + i < a.n_req) mine += few_seg<KT>(a, tid * per + i).tiles;
    int64_t upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t u = __shfl_up(upto, d);
        if (lane >= d) upto += u;
    }
    if (lane == 63) line[wave] = upto;
    __syncthreads();
    int64_t U = 0;
    for (int w = 0; w < FEW_WAVES; ++w) {
        if (w < wave) upto += line[w];
        U += line[w];
    }
    if (U == 0) return;
    // fewer workers than workgroups where the line is short: a tile for every wave
    const int We = (int)min((int64_t)W, (U + FEW_WAVES - 1) / FEW_WAVES), w = blockIdx.x;
    if (w >= We) return;
    int64_t u0 = share(U, w, We);
    const int64_t u1 = share(U, w + 1, We);
    if (u0 >= upto - mine && u0 < upto) {
        int64_t at = upto - mine;
        int r = tid * per;
        for (;; ++r) {
            const int n = few_seg<KT>(a, r).tiles;
            if (u0 < at + n) break;
            at += n;
        }
        start_r = r;
        start_at = at;
    }
    __syncthreads();
    int r = start_r;
    int64_t r_at = start_at;                                    // the request's first tile on the line

    while (u0 < u1) {
        const seg sg = few_seg<KT>(a, r);
        if (sg.tiles == 0) { ++r; continue; }
        const int t0 = (int)(u0 - r_at), t1 = (int)min(u1 - r_at, (int64_t)sg.tiles);
        const int rows = min(sg.s.rows, min(a.max_q, COLS / G)), cols = rows * G;
        const int p_first = sg.s.kv - sg.s.rows, p_last = p_first + rows - 1;
        const int32_t *tab = a.table + (int64_t)r * a.max_blocks;

        // ── the queries: lane (m16, g) holds elements g KE .. of column m16 ──
        typedef typename regs<A, 8>::type q8;
        q8 q[NQ][KV8];
        int pos[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const int c = n * 16 + m16, i = c / G;
            pos[n] = c < cols ? p_first + i : p_last;
            const A *src = (const A *)a.q + (int64_t)(sg.s.row0 + i) * a.q_stride + ((int64_t)kvh * G + (c - i * G)) * hd;
#pragma unroll
            for (int s = 0; s < KV8; ++s) {
                const int e = g * KE + 8 * s;
                q[n][s] = q8{};
                if (c < cols && e < hd) q[n][s] = *reinterpret_cast<const q8 *>(src + e);
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
            const int pg = tab[min(j, max(sg.s.kv - 1, 0)) >> a.page_shift];
            const bool good = j < sg.s.kv && pg >= 0 && pg < a.n_pages;
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
                            for (int e = 0; e < 8; ++e) s[n][b] = mfma((float)k[b][x][e], q[n][x][e], s[n][b]);
                        } else {
                            s[n][b] = mfma(k[b][x], q[n][x], s[n][b]);
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
            uint64_t odd = 0;                                   // keys with values that are not finite, seen by some rows only
            if (masked) {
                // (the empty asm keeps this a branch: as selects it would be work of every tile)
                uint64_t mine = ok_now >> (4 * g);
                asm volatile("" : "+v"(mine));
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int jj = b * 16 + 4 * g + i, j = base + jj;
                        const bool there = mine >> (b * 16 + i) & 1;
#pragma unroll
                        for (int n = 0; n < NQ; ++n) {
                            const bool see = there && j <= pos[n] && (a.window <= 0 || j > pos[n] - a.window);
                            if (!see) s[n][b][i] = -INFINITY;
                        }
                        const bool none = !there || j > p_last || (a.window > 0 && j <= p_first - a.window);
                        const bool every = there && j <= p_first && (a.window <= 0 || j > p_last - a.window);
                        if (none) v[b][i] = vrow{};             // 0 x NaN
                        bool bad = false;
#pragma unroll
                        for (int c = 0; c < VE; ++c) bad |= not_finite(v[b][i][c]);
                        bad = bad && !every && VE * m16 < hd;
                        const uint64_t who = __ballot(bad);     // (lanes of one g: one key)
#pragma unroll
                        for (int gg = 0; gg < 4; ++gg)
                            if (who >> (16 * gg) & 0xffff) odd |= 1ull << (b * 16 + 4 * gg + i);
                        if (odd >> jj & 1) v[b][i] = vrow{};
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
                top = pk_max_rows4(top) * a.scale2;
                const float mn = fmaxf(mx[n], top);
                // (nothing seen yet: any finite value keeps exp2 at 0)
                const float ref = mn == -INFINITY ? 0.0f : mn, f = __builtin_amdgcn_exp2f(mx[n] - ref);
                mx[n] = mn;
                float sum = 0.0f;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][b][i], a.scale2, -ref));
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
                            for (int n = 0; n < NQ; ++n) o[n][c] = mfma((float)v[b][i][c], s[n][b][i], o[n][c]);
            } else {
                typedef typename regs<A, 8>::type op8;
#pragma unroll
                for (int b = 0; b < NB; b += 2) {
                    op8 p[NQ];
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) p[n][i] = (A)s[n][b][i], p[n][4 + i] = (A)s[n][b + 1][i];
#pragma unroll
                    for (int c = 0; c < VE; ++c) {
                        op8 vt;
#pragma unroll
                        for (int i = 0; i < 4; ++i) vt[i] = v[b][i][c], vt[4 + i] = v[b + 1][i][c];
#pragma unroll
                        for (int n = 0; n < NQ; ++n) o[n][c] = mfma(vt, p[n], o[n][c]);
                    }
                }
            }
            // values that are not finite, on the rows that see them
            while (odd) {
                const int jj = __ffsll((unsigned long long)odd) - 1, j = base + jj;
                odd &= odd - 1;
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
        const bool whole = t0 == 0 && t1 == sg.tiles;
        const int quads = hd >> 2;
        float *slot = part + (((int64_t)kvh * W + w) * 2 + (t0 == 0)) * (COLS * (HDP + 4));
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
                l += __builtin_amdgcn_exp2f(sk - ref);
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                const int64_t row = sg.s.row0 + i;
                A *dst = (A *)a.out + row * a.out_stride + (int64_t)h * hd + e;
                typename regs<A, 4>::type ov;
#pragma unroll
                for (int z = 0; z < 4; ++z) ov[z] = (A)(acc[z] * inv);
                *reinterpret_cast<typename regs<A, 4>::type *>(dst) = ov;
                if (a.lse && e == 0) a.lse[row * a.H + h] = l == 0.0f ? -INFINITY : (ref + __builtin_amdgcn_logf(l)) * PK_LN2;
            } else {
                float *p = slot + c * (HDP + 4);
                const uint64_t *b = reinterpret_cast<const uint64_t *>(&acc);
                // past the L2: another XCD's workgroup may join
                __hip_atomic_store((uint64_t *)(p + 4 + e), b[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __hip_atomic_store((uint64_t *)(p + 4 + e) + 1, b[1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                if (e == 0) {
                    __hip_atomic_store(p, mm, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    __hip_atomic_store(p + 1, l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
            }
        }
        if (!whole) {
            // the request's parts: workers wa .. wb
            const int wa = owner(r_at, U, We), wb = owner(r_at + sg.tiles - 1, U, We);
            uint32_t *cnt = count + (int64_t)kvh * W + wa;
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            if (tid == 0) {
                const uint32_t was = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                last_in = was == (uint32_t)(wb - wa);
                if (last_in) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            __syncthreads();
            if (last_in) {
                const auto at = [&](int i, int c) {             // worker wa holds the request's start, the others its middle
                    return part + (((int64_t)kvh * W + i) * 2 + (i == wa)) * (COLS * (HDP + 4)) + c * (HDP + 4);
                };
                const auto ld = [](const float *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
                for (int x = tid; x < cols * quads; x += FEW_THREADS) {
                    const int c = x / quads, e = (x - c * quads) * 4;
                    const int i = c / G, h = kvh * G + (c - i * G);
                    const float sk = a.sinks ? a.sinks[h] * PK_LOG2E : -INFINITY;
                    float mm = sk;
                    for (int y = wa; y <= wb; ++y) mm = fmaxf(mm, ld(at(y, c)));
                    const float ref = mm == -INFINITY ? 0.0f : mm;
                    float l = __builtin_amdgcn_exp2f(sk - ref);
                    f32x4 acc = {0, 0, 0, 0};
                    for (int y = wa; y <= wb; ++y) {
                        const float *p = at(y, c);
                        const float f = __builtin_amdgcn_exp2f(ld(p) - ref);
                        l = __builtin_fmaf(ld(p + 1), f, l);
                        uint64_t b[2];
                        b[0] = __hip_atomic_load((const uint64_t *)(p + 4 + e), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                        b[1] = __hip_atomic_load((const uint64_t *)(p + 4 + e) + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                        const float *ov = reinterpret_cast<const float *>(b);
#pragma unroll
                        for (int z = 0; z < 4; ++z) acc[z] = __builtin_fmaf(ov[z], f, acc[z]);
                    }
                    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                    const int64_t row = sg.s.row0 + i;
                    typename regs<A, 4>::type ov;
#pragma unroll
                    for (int z = 0; z < 4; ++z) ov[z] = (A)(acc[z] * inv);
                    *reinterpret_cast<typename regs<A, 4>::type *>((A *)a.out + row * a.out_stride + (int64_t)h * hd + e) = ov;
                    if (a.lse && e == 0)
                        a.lse[row * a.H + h] = l == 0.0f ? -INFINITY : (ref + __builtin_amdgcn_logf(l)) * PK_LN2;
                }
            }
        }
        u0 = r_at + t1;
        r_at += sg.tiles;
        ++r;
    }
}

template <typename A, typename C, int HDP, int NQ>
int launch(pk_engine *e, const pk_attn_args &a, int64_t tiles) {
    // workers per KV head: two workgroups per CU in all, no more than the line may have tiles for its waves
    const int64_t most = (tiles + FEW_WAVES - 1) / FEW_WAVES;
    const int W = (int)std::max<int64_t>(1, std::min<int64_t>(most, (2 * e->n_cu + a.KVH - 1) / a.KVH));
    PK_TRY(pk_attn_workspace(e, (int64_t)a.KVH * W * 2 * 16 * NQ * (HDP + 4), (int64_t)a.KVH * W));
    k_attn_few<A, C, HDP, NQ><<<dim3((unsigned)W, (unsigned)a.KVH), FEW_THREADS, 0, e->stream>>>(a, e->att_ws, e->att_cnt);
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

int pk_launch_attn_few(pk_engine *e, const pk_attn_args &a, int max_kv) {
    // (with a window, a row reads no more than it and a tile's rest)
    const int64_t positions = a.window > 0 ? std::min<int64_t>(max_kv, (int64_t)a.window + a.max_q + 64) : max_kv;
#define PK_FEW(A, C) return by_shape<A, C>(e, a, positions)
    PK_BY_TYPES(a.type, a.cache_type, PK_FEW);
#undef PK_FEW
}
