// pk_attn_tile.hip — attention of many rows: packed prompts, and chunks of new
// rows over paged caches.
//
// A workgroup takes BM columns: rows of one request times the query heads of
// one KV head, rows first, so that BM / G neighbouring rows share every key
// and value it reads and a window or the causal edge costs few tiles. Its waves
// hold 32 columns each and go over the keys in tiles of KT, staged through LDS:
// S^T = K Q^T, then O^T = V^T P^T. A lane of a 32 x 32 product holds one query's
// scores of 4 keys out of 8, in the order in which the second product may take
// them, so that probabilities stay in registers; V comes out of LDS transposed
// (ds_read_b64_tr_b16). Rows of LDS are XOR-swizzled in 16-byte pieces against
// bank conflicts.
//
// fp32 activations run on the bf16 products as well: a value is three bf16 (its 24
// bits, 8 at a time, exactly), and of the nine partial products the six above
// 2^-24 of the result are taken, each exact, summed in fp32: 6 x 16 cycles where
// the fp32 instructions take 256. A bf16 cache is one plane (three products), an
// fp16 cache two (five). Not finite values meet zeros among the partial products:
// a key with one makes the rows that see it NaN, and values of V are looked
// at as they are staged (slow_column).
//
// Where the columns are too few for the device, the keys are split too: each
// part leaves m, l and o, and k_attn_join adds them up in order.
//
// Bound by the SIMD's issue of everything beside the products: of a tile's 2100 cycles
// per wave half are the matrix unit's, the rest exponentials (8 cycles each), sums,
// conversions and LDS reads that four waves overlap only in part. 64 query heads over 8
// of 64, bf16: 12 prompts of up to 4096 rows 465 us, 820 TFLOP/s; 512 rows after 23,488
// positions 262 us, 760. fp32, heads of 128, prompts of up to 1500 rows: 235 us, 132 TFLOP/s.
#include "pk_attention.h"

#include <type_traits>

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <typename T, int N>
struct regs {
    typedef T type __attribute__((ext_vector_type(N)));
};

__device__ __forceinline__ f32x16 mfma(pk_f16x8 a, pk_f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma(pk_bf16x8 a, pk_bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// A value's planes: itself in T, or N bf16 that add up to it.
template <typename T, int N, typename V8>
__device__ __forceinline__ void planes(const V8 &x, typename regs<T, 8>::type (&p)[N]) {
    if constexpr (N == 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[0][i] = (T)x[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
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

// Which columns a workgroup has.
struct place {
    pk_span s;
    int r, tile, tiles;      // request, its tile and number of tiles; r < 0: none
    int idx0, n_idx;         // first column, number of columns of the request
    int p_lo, p_hi;          // positions of the first and last row
    int first, n_t;          // first key, tiles of keys
};
// Request r's tiles are numbered from floor(row0 G / BM) + r on: at least as many
// numbers as it has tiles, known without the other requests' lengths.
template <int BM, int KT>
__device__ __forceinline__ place find(const pk_attn_args &a, int64_t b, int cut, int *found) {
    const int G = a.H / a.KVH;
    if (threadIdx.x == 0) *found = -1;
    __syncthreads();
    for (int r = threadIdx.x; r < a.n_req; r += blockDim.x) {
        const int64_t x = min(max(a.cu[r], 0), a.n_tokens), y = min(max(a.cu[r + 1], 0), a.n_tokens);
        if (x * G / BM + r <= b && b < y * G / BM + r + 1) *found = r;
    }
    __syncthreads();
    place p;
    p.r = __builtin_amdgcn_readfirstlane(*found);
    if (p.r < 0) return p;
    p.s = pk_request(a, p.r);
    p.n_idx = min(p.s.rows, a.max_q) * G;
    p.tiles = (p.n_idx + BM - 1) / BM;
    const int64_t j = b - ((int64_t)p.s.row0 * G / BM + p.r);
    if (j < 0 || j >= p.tiles || p.n_idx <= cut) {
        p.r = -1;
        return p;
    }
    p.tile = p.tiles - 1 - (int)j;                       // the ones with the most keys first
    p.idx0 = p.tile * BM;
    const int before = p.s.kv - p.s.rows;
    p.p_lo = before + p.idx0 / G;
    p.p_hi = before + (min(p.idx0 + BM, p.n_idx) - 1) / G;
    p.first = a.window > 0 ? max(p.p_lo - a.window + 1, 0) & ~(KT - 1) : 0;
    p.n_t = max(p.p_hi + 1 - p.first + KT - 1, 0) / KT;
    return p;
}

template <typename A>
__device__ __forceinline__ void store4(A *dst, float x, float y, float z, float w) {
    typename regs<A, 4>::type v;
    v[0] = (A)x, v[1] = (A)y, v[2] = (A)z, v[3] = (A)w;
    *reinterpret_cast<typename regs<A, 4>::type *>(dst) = v;
}

// Keys of a tile, waves of a SIMD, and buffers of a tile's place in LDS. With 16-bit
// products and heads up to 64 a wave fits 128 registers: four waves of a SIMD hide
// each other's exponentials, LDS reads and barriers (two waves of 64 columns each, with
// half the LDS reads: 480 us for 12 prompts of up to 4096 rows; four of 32: 471, and
// 48 against 54 for 128-position windows). Tiles that come straight into LDS
// need the next one's place too; planes are split from registers, into the other
// buffer where one workgroup fills a CU (one barrier a tile).
constexpr int tile_keys(int hdp, int qp) { return hdp <= 64 || qp == 1 ? 64 : 32; }
constexpr int tile_simd(int hdp, int qp) { return hdp <= 64 && qp == 1 ? 4 : 2; }
constexpr int tile_bufs(int wv, int qp) { return qp == 1 || wv == 8 ? 2 : 1; }

// 16 bytes per lane from base + off straight to LDS (lane i's at lds + 16 i). In
// assembly: the compiler does not pair these loads with the kernel's LDS reads
// (it would wait for every outstanding one before each read); the kernel's own wait
// and barrier order them. M0 carries the LDS address.
typedef __attribute__((address_space(3))) void lds_void;
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma16(const void *base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
}
#pragma clang diagnostic pop

// Whether one of eight 16-bit values is an infinity or NaN (exponent all ones).
template <typename T>
__device__ __forceinline__ uint32_t odd8(const uint4 &v) {
    constexpr uint32_t E = __is_same(T, pk_f16) ? 0x7c007c00u : 0x7f807f80u, ONE = __is_same(T, pk_f16) ? 0x04000400u : 0x00800080u;
    return (((v.x & E) + ONE) | ((v.y & E) + ONE) | ((v.z & E) + ONE) | ((v.w & E) + ONE)) & 0x80008000u;
}

// Element offset of position j's row of keys or values.
template <bool PAGED>
__device__ __forceinline__ int64_t row_at(const pk_attn_args &a, const place &pl, int64_t stride, int kvh, int j, bool &there) {
    if constexpr (PAGED) {
        const int pg = a.table[(int64_t)pl.r * a.max_blocks + (j >> a.page_shift)];
        there = pg >= 0 && pg < a.n_pages;
        return ((((int64_t)(there ? pg : 0) * a.KVH + kvh) << a.page_shift) + (j & ((1 << a.page_shift) - 1))) * a.hd;
    }
    there = true;
    return (pl.s.row0 + (int64_t)j) * stride + kvh * a.hd;
}

// One column over the keys from..to, a wave at a time, position by position: for
// workgroups that met values of V that are not finite where some row does not
// see them (0 x infinity in a product), which then do all their columns so.
template <typename A, typename C, int BM, bool PAGED>
__device__ __attribute__((noinline)) void slow_column(pk_attn_args a, place pl, int kvh, int idx, int from, int to, bool whole,
                                                      float *part_m, float *part_o) {
    const int lane = threadIdx.x & 63, G = a.H / a.KVH, hd = a.hd, i = idx / G, h = kvh * G + (idx - i * G);
    const int p = pl.s.kv - pl.s.rows + i;
    const int64_t row = pl.s.row0 + i;
    const A *q = (const A *)a.q + row * a.q_stride + (int64_t)h * hd;
    const float sk = whole && a.sinks ? a.sinks[h] * PK_LOG2E : -INFINITY;
    float m = sk, l = whole && a.sinks && sk > -INFINITY ? 1.0f : 0.0f, o0 = 0.0f, o1 = 0.0f;
    const int lo = a.window > 0 ? max(from, p - a.window + 1) : from, hi = min(to, p + 1);
    for (int j = lo; j < hi; ++j) {
        bool there;
        const C *k = (const C *)a.k + row_at<PAGED>(a, pl, a.k_stride, kvh, j, there);
        const C *v = (const C *)a.v + row_at<PAGED>(a, pl, a.v_stride, kvh, j, there);
        if (!there) continue;
        float s = 0.0f;
        if (lane < hd) s = (float)q[lane] * (float)k[lane];
        if (lane + 64 < hd) s = __builtin_fmaf((float)q[lane + 64], (float)k[lane + 64], s);
        s = pk_wave_sum_f(s) * a.scale2;
        const float mn = fmaxf(m, s), ref = mn == -INFINITY ? 0.0f : mn;
        const float f = __builtin_amdgcn_exp2f(m - ref), e = __builtin_amdgcn_exp2f(s - ref);
        m = mn;
        l = __builtin_fmaf(l, f, e);
        o0 = __builtin_fmaf(e, lane < hd ? (float)v[lane] : 0.0f, o0 * f);
        o1 = __builtin_fmaf(e, lane + 64 < hd ? (float)v[lane + 64] : 0.0f, o1 * f);
    }
    if (whole) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        A *dst = (A *)a.out + row * a.out_stride + (int64_t)h * hd;
        if (lane < hd) dst[lane] = (A)(o0 * inv);
        if (lane + 64 < hd) dst[lane + 64] = (A)(o1 * inv);
        if (a.lse && lane == 0) a.lse[row * a.H + h] = l == 0.0f ? -INFINITY : ((m == -INFINITY ? 0.0f : m) + __builtin_amdgcn_logf(l)) * PK_LN2;
    } else {
        if (lane == 0) part_m[0] = m, part_m[BM] = l;
        if (lane < hd) part_o[lane] = o0;
        if (lane + 64 < hd) part_o[lane + 64] = o1;
    }
}

template <typename T, typename A, typename C, int HDP, int WV, int QP, int KP, bool PAGED, bool FULL>
__global__ __launch_bounds__(64 * WV, tile_simd(HDP, QP)) void k_attn_tile(pk_attn_args a, int cut, int splits, float *part) {
    constexpr int BM = 32 * WV, KT = tile_keys(HDP, QP);
    constexpr int NB = KT / 32, QS = HDP / 16, HT = HDP / 32;
    // a tile's 16-byte pieces: CPR to a row, KPW rows to a wave, RPP to a pass of the
    // workgroup (the first PW waves where a pass would be more than the tile)
    constexpr int CPR = HDP / 8, KPW = 64 / CPR, PW = WV * KPW > KT ? KT / KPW : WV, RPP = PW * KPW, NP = KT / RPP, ROWB = HDP * 2;
    constexpr bool PLANES = QP > 1;
    constexpr int BUFS = tile_bufs(WV, QP);
    // fp16 probabilities are scaled by 2^7 (at most 2^15 with what the reference lags), so that
    // those down to 2^-21 of the largest are no subnormals
    constexpr float SHIFT = __is_same(T, pk_f16) ? 7.0f : 0.0f;
    constexpr uint64_t ALL = KT == 64 ? ~0ull : (1ull << KT) - 1;
    typedef typename regs<T, 8>::type t8;
    typedef typename regs<C, 8>::type c8;
    typedef typename regs<A, 8>::type a8;

    __shared__ __attribute__((aligned(16))) uint8_t sK[BUFS][KP][KT * ROWB], sV[BUFS][KP][KT * ROWB];
    __shared__ int found;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, c32 = lane & 31;
    const int kvh = blockIdx.x % a.KVH, G = a.H / a.KVH, hd = FULL ? HDP : a.hd;
    const int64_t slot = blockIdx.x / a.KVH;
    const place pl = find<BM, KT>(a, slot, cut, &found);
    if (pl.r < 0) return;
    const int t_first = (int)((int64_t)pl.n_t * blockIdx.y / splits), t_end = (int)((int64_t)pl.n_t * (blockIdx.y + 1) / splits);
    const int before = pl.s.kv - pl.s.rows, end = pl.p_hi + 1;

    // ── queries ──
    const int w0 = pl.idx0 + wave * 32;                         // the wave's first column
    const bool active = w0 < pl.n_idx;
    const int w_lo = before + w0 / G, w_hi = before + (min(w0 + 32, pl.n_idx) - 1) / G;
    // keys at or below p_old (w_old) lie outside the window of some row of the workgroup
    // (the wave), at or below w_none of every row of the wave
    const int p_old = a.window > 0 ? pl.p_hi - a.window : -1;
    const int w_old = a.window > 0 ? w_hi - a.window : -1, w_none = a.window > 0 ? w_lo - a.window : -1;
    const int idx = w0 + c32, i_row = idx / G;
    const int pos = idx < pl.n_idx ? before + i_row : w_hi;
    t8 q[QP][QS];
    {
        const A *src = (const A *)a.q + (int64_t)(pl.s.row0 + i_row) * a.q_stride + ((int64_t)kvh * G + (idx - i_row * G)) * hd;
#pragma unroll
        for (int x = 0; x < QS; ++x) {
            const int e = 16 * x + 8 * h;
            a8 v = {};
            if (idx < pl.n_idx && e < hd) v = *reinterpret_cast<const a8 *>(src + e);
            t8 p[QP];
            planes<T, QP>(v, p);
#pragma unroll
            for (int n = 0; n < QP; ++n) q[n][x] = p[n];
        }
    }
    float scale2 = a.scale2;
    asm volatile("" : "+v"(scale2));                            // (a register: or it is loaded anew for every tile)

    f32x16 o[HT];
    float mx = -INFINITY, ls = 0.0f;
#pragma unroll
    for (int x = 0; x < HT; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[x][i] = 0.0f;

    // ── staging ──
    // A wave's share of a pass is KPW neighbouring rows, which lie on one page: their
    // address is a scalar, a lane's offset from it the same for every tile. Piece c
    // of row r is kept at place c ^ f(r): f(r) = r % 8 for K (32 lanes read a piece of 32
    // rows), 2 (r % 4) for V (16 lanes read two pieces of four rows).
    const bool stages = PW == WV || wave < PW;
    const int my_row = lane / CPR, my_c = lane % CPR, my_key = wave * KPW + my_row;
    const int ck = PLANES ? my_c : my_c ^ (my_key & 7), cv = PLANES ? my_c : my_c ^ ((my_key & 3) << 1);
    const int64_t rowk = PAGED ? hd : a.k_stride, rowv = PAGED ? hd : a.v_stride;
    const uint32_t offk = (uint32_t)(my_row * rowk + (ck * 8 < hd ? ck * 8 : 0)) * (uint32_t)sizeof(C);
    const uint32_t offv = (uint32_t)(my_row * rowv + (cv * 8 < hd ? cv * 8 : 0)) * (uint32_t)sizeof(C);
    // Page of position base + lane of tile t, and the bits of the positions that there are.
    const auto look = [&](int t, uint64_t &ok) {
        const int base = pl.first + t * KT;
        if constexpr (PAGED) {
            const int j = base + (lane & (KT - 1));
            const int pg = a.table[(int64_t)pl.r * a.max_blocks + (min(j, max(end - 1, 0)) >> a.page_shift)];
            const bool good = j < end && pg >= 0 && pg < a.n_pages;
            ok = __ballot(good) & ALL;
            return good ? pg : 0;
        } else {
            ok = end - base >= KT ? ALL : (1ull << max(end - base, 0)) - 1;
            return 0;
        }
    };
    const uint32_t at_k = (uint32_t)(uintptr_t)(lds_void *)&sK, at_v = (uint32_t)(uintptr_t)(lds_void *)&sV;
    c8 rk[PLANES ? NP : 1], rv[PLANES ? NP : 1];
    // Rows without pages: the wave's first row of the next tile; pages: the KV head's first page.
    const char *nk = (const char *)((const C *)a.k + (PAGED ? ((int64_t)kvh << a.page_shift) * hd
                                                            : (pl.s.row0 + (int64_t)pl.first + t_first * KT + wave * KPW) * rowk + kvh * hd));
    const char *nv = (const char *)((const C *)a.v + (PAGED ? ((int64_t)kvh << a.page_shift) * hd
                                                            : (pl.s.row0 + (int64_t)pl.first + t_first * KT + wave * KPW) * rowv + kvh * hd));
    const uint32_t page_bytes = ((uint32_t)a.KVH << a.page_shift) * (uint32_t)hd * (uint32_t)sizeof(C);
    const int64_t passk = RPP * rowk * (int64_t)sizeof(C), passv = RPP * rowv * (int64_t)sizeof(C);
    const auto load = [&](int t, int pgs, uint64_t ok) {
        if (!stages) return;
        const int base = pl.first + t * KT, buf = t & (BUFS - 1);
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const int k0 = n * RPP + wave * KPW, j0 = base + k0;
            const char *pk, *pv;
            uint32_t ok_ = offk, ov_ = offv;
            if constexpr (PAGED) {
                const uint64_t at = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(pgs, k0) * page_bytes +
                                    (uint32_t)(j0 & ((1 << a.page_shift) - 1)) * (uint32_t)hd * (uint32_t)sizeof(C);
                pk = nk + at;
                pv = nv + at;
            } else {
                pk = nk;
                pv = nv;
                nk += passk;
                nv += passv;
                if (ok != ALL && j0 + KPW > end) {              // no row behind the prompt's last one: that one again
                    const int past = max(j0 - (end - 1), 0);
                    int back = max(j0 + my_row - (end - 1), 0) - past;
                    asm volatile("" : "+v"(back));
                    pk -= past * rowk * (int64_t)sizeof(C);
                    pv -= past * rowv * (int64_t)sizeof(C);
                    ok_ -= (uint32_t)(back * rowk) * (uint32_t)sizeof(C);
                    ov_ -= (uint32_t)(back * rowv) * (uint32_t)sizeof(C);
                }
            }
            if constexpr (PLANES) {
                rk[n] = *reinterpret_cast<const c8 *>(pk + ok_);
                rv[n] = *reinterpret_cast<const c8 *>(pv + ov_);
            } else {
                dma16(pk, ok_, at_k + (uint32_t)(buf * (KT * ROWB) + k0 * ROWB));
                dma16(pv, ov_, at_v + (uint32_t)(buf * (KT * ROWB) + k0 * ROWB));
            }
        }
    };
    uint32_t odd = 0;                                           // this thread met a value that calls for slow_column
    // planes: the loaded tile into its buffer
    const auto place_tile = [&](int t, uint64_t ok) {
        if (!stages) return;
        const int buf = t & (BUFS - 1);
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const int kk = n * RPP + my_key;
            if (ok != ALL) {
                uint64_t mine = ok;
                asm volatile("" : "+v"(mine));
                if (!(mine >> kk & 1)) rk[n] = c8{}, rv[n] = c8{};
            }
            float sum = 0.0f;                                   // (finite values: 0)
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = __builtin_fmaf((float)rv[n][i], 0.0f, sum);
            odd |= sum != 0.0f;
            t8 pk[KP], pv[KP];
            planes<T, KP>(rk[n], pk);
            planes<T, KP>(rv[n], pv);
#pragma unroll
            for (int x = 0; x < KP; ++x) {
                *reinterpret_cast<t8 *>(&sK[buf][x][kk * ROWB + ((my_c ^ (kk & 7)) << 4)]) = pk[x];
                *reinterpret_cast<t8 *>(&sV[buf][x][kk * ROWB + ((my_c ^ ((kk & 3) << 1)) << 4)]) = pv[x];
            }
        }
    };

    // Positions that there are of this tile, the next, the one after; the pages of the next to load.
    // (Planes with two buffers: a tile is loaded two tiles, split one tile ahead.)
    constexpr int AHEAD = PLANES && BUFS == 2 ? 2 : 1;
    uint64_t ok_now = 0, ok_1 = 0, ok_2 = 0;
    int pgs = 0;
    if (t_first < t_end) {
        pgs = look(t_first, ok_now);
        load(t_first, pgs, ok_now);
        if (t_first + 1 < t_end) pgs = look(t_first + 1, ok_1);
        if constexpr (AHEAD == 2) {
            place_tile(t_first, ok_now);
            if (t_first + 1 < t_end) load(t_first + 1, pgs, ok_1);
            if (t_first + 2 < t_end) pgs = look(t_first + 2, ok_2);
        }
    }

    for (int t = t_first; t < t_end; ++t) {
        const int base = pl.first + t * KT, buf = t & (BUFS - 1);
        if constexpr (!PLANES) {
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(0x0f70);                 // vmcnt(0): the wave's part of this tile is in LDS
            __syncthreads();
        } else if constexpr (BUFS == 1) {
            __syncthreads();                                    // the previous tile has been read
            place_tile(t, ok_now);
            __syncthreads();
        } else {
            __syncthreads();
            if (t + 1 < t_end) place_tile(t + 1, ok_1);
        }
        if constexpr (AHEAD == 2) {
            if (t + 2 < t_end) load(t + 2, pgs, ok_2);
        } else {
            if (t + 1 < t_end) load(t + 1, pgs, ok_1);
        }
        const uint64_t ok = ok_now;
        ok_now = ok_1;
        if constexpr (AHEAD == 2) {
            ok_1 = ok_2;
            if (t + 3 < t_end) pgs = look(t + 3, ok_2);
        } else {
            if (t + 2 < t_end) pgs = look(t + 2, ok_1);
        }
        if (!PLANES && (ok != ALL || base + KT - 1 > pl.p_lo || base <= p_old)) {
            // a tile that some row of the workgroup does not see whole. Rows that are not
            // there: zero (0 x NaN); values that are not finite, on rows that not all see: noted
            if (stages) {
                uint64_t mine = ok >> my_key;
                asm volatile("" : "+v"(mine));
#pragma unroll
                for (int n = 0; n < NP; ++n) {
                    uint4 *pv = reinterpret_cast<uint4 *>(&sV[buf][0][(n * RPP + wave * KPW) * ROWB + lane * 16]);
                    const int j = base + n * RPP + my_key;
                    if (!(mine >> (n * RPP) & 1)) *pv = uint4{0, 0, 0, 0};
                    else if (j > pl.p_lo || j <= p_old) odd |= odd8<T>(*pv);
                }
            }
            if (ok != ALL) __syncthreads();
        }
        // a tile that the wave's rows do not see at all
        if (!active || base > w_hi || base + KT - 1 <= w_none) continue;

        // Planes: the key blocks one after the other, the products of one beside the
        // exponentials of its neighbour (the 16-bit kernels have other waves for that).
        constexpr int UNITS = PLANES ? NB : 1, UB = NB / UNITS;
        f32x16 s[UNITS][UB];                                    // scores
        t8 p[UNITS][QP][UB * 2];                                // probabilities
        // S^T = K Q^T
        const auto scores = [&](auto uc) {
            constexpr int u = uc.value;
#pragma unroll
            for (int b = 0; b < UB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[u][b][i] = 0.0f;
#pragma unroll
            for (int x = 0; x < QS; ++x) {
                if (!FULL && 16 * x >= hd) break;
#pragma unroll
                for (int b = 0; b < UB; ++b)
#pragma unroll
                    for (int kp = 0; kp < KP; ++kp) {
                        const int kk = (u * UB + b) * 32 + c32;
                        const t8 k = *reinterpret_cast<const t8 *>(&sK[buf][kp][kk * ROWB + (((2 * x + h) ^ (kk & 7)) << 4)]);
#pragma unroll
                        for (int qp = 0; qp < QP && qp + kp < 3; ++qp) s[u][b] = mfma(k, q[qp][x], s[u][b]);
                    }
            }
        };
        // what a row does not see; the running maximum
        const auto settle = [&](auto uc) {
            constexpr int u = uc.value, k0 = u * UB * 32;
            // (the empty asm keeps these as branches: as selects they would be work of every tile)
            if (base + KT - 1 > w_lo) {
                int upto = pos - base - 4 * h;
                asm volatile("" : "+v"(upto));
#pragma unroll
                for (int b = 0; b < UB; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (k0 + b * 32 + 8 * (i >> 2) + (i & 3) > upto) s[u][b][i] = -INFINITY;
            }
            if (base <= w_old) {
                int from = pos - a.window - base - 4 * h;
                asm volatile("" : "+v"(from));
#pragma unroll
                for (int b = 0; b < UB; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (k0 + b * 32 + 8 * (i >> 2) + (i & 3) <= from) s[u][b][i] = -INFINITY;
            }
            if (PAGED && ok != ALL) {
                uint64_t mine = ok >> (4 * h);
                asm volatile("" : "+v"(mine));
#pragma unroll
                for (int b = 0; b < UB; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (!(mine >> (k0 + b * 32 + 8 * (i >> 2) + (i & 3)) & 1)) s[u][b][i] = -INFINITY;
            }
            float top = s[u][0][0];
#pragma unroll
            for (int b = 0; b < UB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][b][i]);
            const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
            top = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * scale2 - SHIFT;
            // the reference only moves when a score is 2^8 above it: what lies between makes
            // sums and probabilities no less exact, and most tiles need no rescaling
            if (__any(top > mx + 8.0f)) {
                const float mn = fmaxf(mx, top), ref = mn == -INFINITY ? 0.0f : mn, f = __builtin_amdgcn_exp2f(mx - ref);
                mx = mn;
                ls *= f;
#pragma unroll
                for (int x = 0; x < HT; ++x) o[x] *= f;
            }
        };
        const auto weigh = [&](auto uc) {
            constexpr int u = uc.value;
            const float ref = mx == -INFINITY ? 0.0f : mx;
            float sum = 0.0f;
#pragma unroll
            for (int y = 0; y < UB * 2; ++y) {
                typename regs<float, 8>::type x;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][y >> 1][8 * (y & 1) + i], scale2, -ref));
                    sum += x[i];
                }
                // (16-bit types: the one rounding of a probability, half a step of the type that
                // the product takes and that the result is rounded to as well; the sum has it unrounded)
                t8 pp[QP];
                planes<T, QP>(x, pp);
#pragma unroll
                for (int n = 0; n < QP; ++n) p[u][n][y] = pp[n];
            }
            ls += sum;
        };
        // O^T += V^T P^T: the keys in the order of the scores' registers
        const int kr = 4 * h + ((lane & 15) >> 2), c0 = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), sub = (lane & 1) << 3;
        const int swz = (kr & 3) << 1;
        const auto values = [&](auto uc) {
            constexpr int u = uc.value;
#pragma unroll
            for (int y = 0; y < UB * 2; ++y)
#pragma unroll
                for (int x = 0; x < HT; ++x) {
                    if (!FULL && 32 * x >= hd) break;
#pragma unroll
                    for (int kp = 0; kp < KP; ++kp) {
                        const int at = (16 * (u * UB * 2 + y) + kr) * ROWB + (((4 * x + c0) ^ swz) << 4) + sub;
                        typedef __attribute__((address_space(3))) s16x4 lds4;
                        const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)&sV[buf][kp][at]);
                        const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)&sV[buf][kp][at + 8 * ROWB]);
                        typename regs<short, 8>::type vv;
#pragma unroll
                        for (int i = 0; i < 4; ++i) vv[i] = v0[i], vv[4 + i] = v1[i];
                        const t8 vf = __builtin_bit_cast(t8, vv);
#pragma unroll
                        for (int qp = 0; qp < QP && qp + kp < 3; ++qp) o[x] = mfma(vf, p[u][qp][y], o[x]);
                    }
                }
        };
        constexpr std::integral_constant<int, 0> u0;
        scores(u0);
        settle(u0);
        if constexpr (UNITS > 1) {
            constexpr std::integral_constant<int, 1> u1;
            scores(u1);
            weigh(u0);
            values(u0);                                         // (before the reference may move)
            settle(u1);
            weigh(u1);
            values(u1);
        } else {
            weigh(u0);
            values(u0);
        }
    }

    // ── out ──
    const int col = wave * 32 + c32;
    float *dst_part = part + ((slot * a.KVH + kvh) * splits + blockIdx.y) * (BM * (HDP + 2));
    if (__syncthreads_or((int)odd)) {
        for (int c = wave; c < BM && pl.idx0 + c < pl.n_idx; c += WV)
            slow_column<A, C, BM, PAGED>(a, pl, kvh, pl.idx0 + c, pl.first + t_first * KT, pl.first + t_end * KT, splits == 1,
                                         dst_part + c, dst_part + 2 * BM + (int64_t)c * HDP);
        return;
    }
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(ls), __float_as_uint(ls), false, false);
    float l = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    if (idx >= pl.n_idx) return;
    if (splits == 1) {
        const int hq = kvh * G + (idx - i_row * G);
        const int64_t row = pl.s.row0 + i_row;
        float ref = mx == -INFINITY ? 0.0f : mx, f = 1.0f;
        if (a.sinks) {
            const float sk = a.sinks[hq] * PK_LOG2E, top = fmaxf(mx, sk), to = top == -INFINITY ? 0.0f : top;
            f = __builtin_amdgcn_exp2f(mx - to);
            l = __builtin_fmaf(l, f, __builtin_amdgcn_exp2f(sk - to));
            ref = to;
        }
        const float inv = l == 0.0f ? 0.0f : f / l;
        A *dst = (A *)a.out + row * a.out_stride + (int64_t)hq * hd;
#pragma unroll
        for (int x = 0; x < HT; ++x)
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const int e = 32 * x + 8 * y + 4 * h;
                if (e < hd) store4(dst + e, o[x][4 * y] * inv, o[x][4 * y + 1] * inv, o[x][4 * y + 2] * inv, o[x][4 * y + 3] * inv);
            }
        if (a.lse && h == 0) a.lse[row * a.H + hq] = l == 0.0f ? -INFINITY : (ref + __builtin_amdgcn_logf(l)) * PK_LN2;
    } else {
        if (h == 0) dst_part[col] = mx, dst_part[BM + col] = l;
        if (t_first < t_end)
#pragma unroll
            for (int x = 0; x < HT; ++x)
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const int e = 32 * x + 8 * y + 4 * h;
                    if (e < hd)
                        store4(dst_part + 2 * BM + (int64_t)col * HDP + e, o[x][4 * y], o[x][4 * y + 1], o[x][4 * y + 2], o[x][4 * y + 3]);
                }
    }
}

// The parts of split keys, added up in order: four elements of a column per thread, the
// loads of JOIN_AHEAD parts in flight (one after the other: 64 rows after 100,000
// positions, 32 parts, 50 us for 15). Bound by latency, or by the reads of many columns.
constexpr int JOIN_THREADS = 256, JOIN_AHEAD = 8;
template <typename A, int BM, int HDP, int KT>
__global__ __launch_bounds__(JOIN_THREADS) void k_attn_join(pk_attn_args a, int cut, int splits, const float *__restrict__ part) {
    __shared__ int found;
    const int kvh = blockIdx.x % a.KVH, G = a.H / a.KVH;
    const int64_t slot = blockIdx.x / a.KVH;
    const place pl = find<BM, KT>(a, slot, cut, &found);
    if (pl.r < 0) return;
    constexpr int PART = BM * (HDP + 2), QUADS = HDP / 4;
    const int x = blockIdx.y * JOIN_THREADS + threadIdx.x, col = x / QUADS, e = x % QUADS * 4, idx = pl.idx0 + col;
    if (idx >= pl.n_idx || e >= a.hd) return;
    const float *src = part + (slot * a.KVH + kvh) * splits * PART;
    const int i = idx / G, hq = kvh * G + (idx - i * G);
    const float sk = a.sinks ? a.sinks[hq] * PK_LOG2E : -INFINITY;
    float top = sk, l = sk > -INFINITY ? 1.0f : 0.0f;
    f32x4 acc = {0, 0, 0, 0};
    for (int y0 = 0; y0 < splits; y0 += JOIN_AHEAD) {
        float m[JOIN_AHEAD], s[JOIN_AHEAD];
        f32x4 v[JOIN_AHEAD];
#pragma unroll
        for (int y = 0; y < JOIN_AHEAD; ++y) {
            m[y] = -INFINITY;
            if (y0 + y >= splits) continue;
            const float *p = src + (int64_t)(y0 + y) * PART;
            m[y] = p[col], s[y] = p[BM + col];
            v[y] = *reinterpret_cast<const f32x4 *>(p + 2 * BM + (int64_t)col * HDP + e);
        }
        float mn = top;
#pragma unroll
        for (int y = 0; y < JOIN_AHEAD; ++y) mn = fmaxf(mn, m[y]);
        const float ref = mn == -INFINITY ? 0.0f : mn, f0 = __builtin_amdgcn_exp2f(top - ref);
        top = mn;
        l *= f0;
        acc *= f0;
#pragma unroll
        for (int y = 0; y < JOIN_AHEAD; ++y) {
            // (parts without keys hold no sums)
            if (y0 + y >= splits || pl.n_t * (int64_t)(y0 + y) / splits == pl.n_t * (int64_t)(y0 + y + 1) / splits) continue;
            const float f = __builtin_amdgcn_exp2f(m[y] - ref);
            l = __builtin_fmaf(s[y], f, l);
#pragma unroll
            for (int z = 0; z < 4; ++z) acc[z] = __builtin_fmaf(v[y][z], f, acc[z]);
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int64_t row = pl.s.row0 + i;
    store4((A *)a.out + row * a.out_stride + (int64_t)hq * a.hd + e, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
    if (a.lse && e == 0) a.lse[row * a.H + hq] = l == 0.0f ? -INFINITY : ((top == -INFINITY ? 0.0f : top) + __builtin_amdgcn_logf(l)) * PK_LN2;
}

template <typename T, typename A, typename C, int HDP, int WV, int QP, int KP, bool PAGED, bool FULL>
int launch(pk_engine *e, const pk_attn_args &a, int cut, int max_kv) {
    constexpr int BM = 32 * WV, KT = tile_keys(HDP, QP);
    const int64_t G = a.H / a.KVH, slots = (int64_t)a.n_tokens * G / BM + a.n_req, wgs = slots * a.KVH;
    PK_CHECK(wgs <= INT32_MAX, PK_ERR_UNSUPPORTED, "attention: %lld tiles of rows", (long long)wgs);
    // workgroups for all of the device's waves, from keys enough for eight tiles each
    // (and parts for no more than four times as many tile numbers)
    int splits = 1;
    const int64_t busy = std::max<int64_t>(((int64_t)a.n_tokens * G + BM - 1) / BM, 1) * a.KVH;
    const int64_t want = (int64_t)tile_simd(HDP, QP) * 4 / WV * e->n_cu;
    if (PAGED && busy < want) splits = (int)std::max<int64_t>(1, std::min<int64_t>({want / busy, max_kv / (8 * KT), 4 * want / wgs}));
    float *part = nullptr;
    if (splits > 1) {
        PK_TRY(pk_attn_workspace(e, wgs * splits * BM * (HDP + 2), 1));
        part = e->att_ws;
    }
    k_attn_tile<T, A, C, HDP, WV, QP, KP, PAGED, FULL>
        <<<dim3((unsigned)wgs, (unsigned)splits), 64 * WV, 0, e->stream>>>(a, cut, splits, part);
    PK_HIP(hipGetLastError());
    if (splits > 1) {
        k_attn_join<A, BM, HDP, KT><<<dim3((unsigned)wgs, BM * HDP / 4 / JOIN_THREADS), JOIN_THREADS, 0, e->stream>>>(a, cut, splits, part);
        PK_HIP(hipGetLastError());
    }
    return PK_OK;
}

// Four waves per workgroup, or eight where planes are split for them all and the columns
// fill the device either way. Measured, 4 / 8 waves: fp32 prompts of up to 1500 rows,
// heads of 128, 247 / 238 us; 256 rows after 8000 positions, fp32 over bf16, heads of
// 128, 128 / 118; one prompt of 6000 rows, heads of 64, 1420 / 1370; a mixed step's three
// chunks 91 / 95. 16-bit products: 12
// prompts of up to 4096 rows 471 / 476, one of 512 14.2 / 18.1.
template <typename T, typename A, typename C, int HDP, int QP, int KP, bool PAGED>
int by_waves(pk_engine *e, const pk_attn_args &a, int cut, int max_kv) {
    if (a.hd != HDP) return launch<T, A, C, HDP, 4, QP, KP, PAGED, false>(e, a, cut, max_kv);
    if constexpr (QP > 1) {
        constexpr int BM = 32 * 8;
        const int64_t G = a.H / a.KVH, cols = (int64_t)a.n_tokens * G;
        const int64_t parts = PAGED ? std::max<int64_t>(1, max_kv / (8 * tile_keys(HDP, QP))) : 1;
        const bool fills = (cols + BM - 1) / BM * a.KVH * parts >= e->n_cu && cols >= 4 * BM * (int64_t)a.n_req;
        if (fills && cut == 0 && (a.window == 0 || a.window * G >= 4 * BM))
            return launch<T, A, C, HDP, 8, QP, KP, PAGED, true>(e, a, cut, max_kv);
    }
    return launch<T, A, C, HDP, 4, QP, KP, PAGED, true>(e, a, cut, max_kv);
}

template <typename T, typename A, typename C, int QP, int KP, bool PAGED>
int by_shape(pk_engine *e, const pk_attn_args &a, int cut, int max_kv) {
    if (a.hd <= 64) return by_waves<T, A, C, 64, QP, KP, PAGED>(e, a, cut, max_kv);
    return by_waves<T, A, C, 128, QP, KP, PAGED>(e, a, cut, max_kv);
}

}  // namespace

int pk_launch_attn_tile(pk_engine *e, const pk_attn_args &a, int cut, int max_kv) {
    if (a.kv_len) {
        if (a.type == PK_T_F16) return by_shape<pk_f16, pk_f16, pk_f16, 1, 1, true>(e, a, cut, max_kv);
        if (a.type == PK_T_BF16) return by_shape<pk_bf16, pk_bf16, pk_bf16, 1, 1, true>(e, a, cut, max_kv);
        if (a.cache_type == PK_T_BF16) return by_shape<pk_bf16, float, pk_bf16, 3, 1, true>(e, a, cut, max_kv);
        if (a.cache_type == PK_T_F16) return by_shape<pk_bf16, float, pk_f16, 3, 2, true>(e, a, cut, max_kv);
        return by_shape<pk_bf16, float, float, 3, 3, true>(e, a, cut, max_kv);
    }
    if (a.type == PK_T_F16) return by_shape<pk_f16, pk_f16, pk_f16, 1, 1, false>(e, a, cut, max_kv);
    if (a.type == PK_T_BF16) return by_shape<pk_bf16, pk_bf16, pk_bf16, 1, 1, false>(e, a, cut, max_kv);
    return by_shape<pk_bf16, float, float, 3, 3, false>(e, a, cut, max_kv);
}
