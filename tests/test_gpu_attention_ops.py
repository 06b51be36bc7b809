"""attention_packed and attention_paged against 64 bits, row by row within
bounds of the arithmetic (paged_ref.bounds)."""
import math

import pytest
import torch

from paged_ref import attend, bounds, check

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HEADS = [(64, 8, 64), (8, 8, 128), (12, 2, 96), (5, 1, 16), (16, 2, 128), (6, 6, 32), (40, 1, 64), (9, 3, 48)]


@pytest.fixture(scope="module")
def eng(gpu):
    import picchio_amd as pa
    with pa.Engine(pa.gptoss_cfg(n_layers=1, n_experts=4, ctx_len=16, vocab=64)) as e:
        yield e


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def starts(v, first=0):
    c = [first]
    for x in v:
        c.append(c[-1] + x)
    return c


def randn(gen, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)


class Packed:
    def __init__(self, gen, lens, H, KVH, hd, dtype, first=0, behind=0, std=1.0):
        self.lens, self.cu = lens, starts(lens, first)
        T = self.cu[-1] + behind
        x = randn(gen, (T, (H + 2 * KVH) * hd), dtype, std)
        self.q, self.k, self.v = (x[:, :H * hd].unflatten(1, (H, hd)), x[:, H * hd:(H + KVH) * hd].unflatten(1, (KVH, hd)),
                                  x[:, (H + KVH) * hd:].unflatten(1, (KVH, hd)))
        self.out, self.lse = torch.full((T, H, hd), 7.0, device="cuda").to(dtype), torch.full((T, H), 7.0, device="cuda")

    def run(self, eng, max_len=None, cu=None, **kw):
        import picchio_amd as pa
        cu = ints(self.cu) if cu is None else cu
        a = pa.attn_packed(self.q, self.k, self.v, self.out, cu, max(self.lens) if max_len is None else max_len,
                           lse=self.lse, **kw)
        torch.cuda.synchronize()
        eng.attention_packed(a)
        eng.sync()

    def verify(self, window=0, sinks=None, scale=None, what=""):
        T = len(self.q)
        for s, n in enumerate(self.lens):
            r = slice(self.cu[s], self.cu[s] + n)
            if n:
                o, lse, need = attend(self.q[r], self.k[r], self.v[r], 0, window, sinks, scale=scale)
                bo, bs = bounds(o, lse, need, self.q.dtype, self.q.shape[2])
                check(self.out[r], o, bo, (what, s, "out"))
                check(self.lse[r], lse, bs, (what, s, "lse"))
        for rest in (slice(0, self.cu[0]), slice(self.cu[-1], T)):
            assert (self.out[rest] == 7.0).all() and (self.lse[rest] == 7.0).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("H,KVH,hd", HEADS)
@pytest.mark.parametrize("lens,window,sinks", [([1], 0, True), ([5, 0, 1, 64, 33, 0], 0, True), ([150, 257, 63], 0, False),
                                               ([129, 300], 128, True), ([90, 70], 1, False), ([200], 17, True),
                                               ([700], 0, True)])
def test_packed(eng, dtype, H, KVH, hd, lens, window, sinks):
    gen = torch.Generator(device="cuda").manual_seed(H + hd + sum(lens))
    p = Packed(gen, lens, H, KVH, hd, dtype, first=3, behind=70)
    sk = randn(gen, (H,), F32, 2.0) if sinks else None
    p.run(eng, window=window, sinks=sk)
    p.verify(window, sk)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_packed_long(eng, dtype):
    """Prompts of many tiles, windows that end inside them, a scale of its own,
    scores of +-30."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    for lens, window, heads, std in (([2100], 0, (8, 1, 64), 1.0), ([1500, 900], 1000, (4, 2, 128), 1.0),
                                     ([1030, 1], 513, (2, 2, 64), 2.0)):
        p = Packed(gen, lens, *heads, dtype, std=std)
        p.run(eng, window=window, scale=0.25 / std)
        p.verify(window, scale=0.25 / std)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_packed_masked_specials(eng, dtype):
    """Infinities and NaN in keys and values that a row does not see leave it
    alone; rows that see them have them."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    for window, lens in ((0, [300, 100]), (50, [300, 100])):
        for special in (float("nan"), float("inf")):
            p = Packed(gen, lens, 8, 2, 64, dtype)
            p.v[170, 1, 5] = special
            p.v[399, 0] = special
            p.k[330, 0, 7] = float("nan")
            p.run(eng, window=window)
            p.verify(window, what=(window, special))


def test_packed_lowest_and_equal_scores(eng):
    """Scores at the bottom of the type's range, sinks far above and below."""
    for dtype in (F32, BF16):
        gen = torch.Generator(device="cuda").manual_seed(4)
        p = Packed(gen, [100], 4, 2, 64, dtype)
        p.q.fill_(0.0)
        for sinks in ([-1e30, 1e30, 0.0, -3.0e38], [-math.inf] * 4, [50.0, -50.0, 80.0, -80.0]):
            sk = torch.tensor(sinks, device="cuda")
            p.run(eng, sinks=sk)
            p.verify(0, sk)
        p.q.fill_(-1e4)
        p.k.copy_(p.k.abs() * 1e4 if dtype != F16 else p.k)
        p.run(eng)
        assert torch.isfinite(p.out).all() and torch.isfinite(p.lse).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_small_probabilities(eng, dtype):
    """One key far above all others, without a value of its own: the rest, each of a
    probability around 1.03 * 2^-20 and large values, make up the result."""
    gen = torch.Generator(device="cuda").manual_seed(22)
    up = (20 - math.log2(1.03)) * math.log(2.0)
    p = Packed(gen, [1800, 200], 8, 2, 64, dtype)
    g = Paged(gen, [50, 1], [1900, 1700], 8, 2, 64, dtype, dtype, 16)
    for x in (p, g):
        x.q.fill_(1.0)
    for k, v in [(p.k[:1800], p.v[:1800]), (p.k[1800:], p.v[1800:])] + list(zip(g.k, g.v)):
        k.zero_()
        k[0] = up / 8                                              # (64 elements, scale 1 / 8)
        v *= 1024.0
        v[0] = 0.0
    g.fill()
    p.run(eng), g.run(eng)
    p.verify(what="packed"), g.verify(what="paged")


def test_packed_bounds_of_starts(eng):
    """max_len cuts rows; starts beyond the rows or not ascending stay in bounds."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    p = Packed(gen, [100, 40], 8, 2, 64, BF16)
    p.run(eng, max_len=64)
    full_out, full_lse = p.out.clone(), p.lse.clone()
    assert (full_out[64:100] == 7.0).all() and not (full_out[:64] == 7.0).all()
    o, lse, need = attend(p.q[:100], p.k[:100], p.v[:100], 0)
    bo, _ = bounds(o, lse, need, BF16, 64)
    check(p.out[:64], o[:64], bo[:64], "cut")
    for cu in ([0, 90, 1000], [-5, 20, 140], [100, 20, 140]):
        p.out.fill_(7.0)
        p.run(eng, cu=ints(cu), max_len=140)
        a, b = max(cu[1], 0), min(cu[2], 140)
        if cu[0] <= cu[1]:
            o, lse, need = attend(p.q[a:b], p.k[a:b], p.v[a:b], 0)
            check(p.out[a:b], o, bounds(o, lse, need, BF16, 64)[0], cu)


class Paged:
    """Requests with q_lens rows at the end of kv_lens positions; every slot that
    holds no position is NaN."""

    def __init__(self, gen, q_lens, kv_lens, H, KVH, hd, act, cache, page, behind=0, first=0, wide=0, std=1.0):
        self.q_lens, self.kv_lens, self.page, self.hd = q_lens, kv_lens, page, hd
        self.cu = starts(q_lens, first)
        T, n = self.cu[-1] + behind, len(q_lens)
        need = [-(-x // page) for x in kv_lens]
        n_pages = sum(need) + 2
        self.q = randn(gen, (T, H * hd + 8 * wide), act, std)[:, :H * hd].unflatten(1, (H, hd))
        self.K = torch.full((n_pages, KVH, page, hd), float("nan"), device="cuda", dtype=cache)
        self.V = self.K.clone()
        perm = torch.randperm(n_pages, generator=gen, device="cuda").tolist()
        self.tab, at = [], 0
        blocks = max(need + [1]) + 1
        for r in range(n):
            self.tab.append(perm[at:at + need[r]] + [-1] * (blocks - need[r]))
            at += need[r]
        self.k, self.v = [], []
        for r in range(n):
            kk, vv = randn(gen, (kv_lens[r], KVH, hd), cache, std), randn(gen, (kv_lens[r], KVH, hd), cache)
            self.k.append(kk), self.v.append(vv)
        self.fill()
        self.out, self.lse = torch.full((T, H, hd), 7.0, device="cuda").to(act), torch.full((T, H), 7.0, device="cuda")

    def fill(self):
        for r, n in enumerate(self.kv_lens):
            if n:
                j = torch.arange(n, device="cuda")
                pg = torch.tensor(self.tab[r], device="cuda")[j // self.page]
                ok = (pg >= 0) & (pg < len(self.K))
                self.K[pg[ok], :, j[ok] % self.page] = self.k[r][ok]
                self.V[pg[ok], :, j[ok] % self.page] = self.v[r][ok]

    def record(self, max_q=None, max_kv=0, **kw):
        import picchio_amd as pa
        return pa.attn_paged(self.q, self.out, ints(self.cu), ints(self.kv_lens), ints(self.tab), pa.pages(self.K, self.V),
                             max(self.q_lens) if max_q is None else max_q, max_kv, lse=self.lse, **kw)

    def run(self, eng, **kw):
        a = self.record(**kw)
        torch.cuda.synchronize()
        eng.attention_paged(a)
        eng.sync()

    def verify(self, window=0, sinks=None, max_q=None, what=""):
        for r, n in enumerate(self.q_lens):
            if n:
                s = slice(self.cu[r], self.cu[r] + n)
                pg = torch.tensor(self.tab[r], device="cuda")[torch.arange(self.kv_lens[r], device="cuda") // self.page]
                o, lse, need = attend(self.q[s], self.k[r], self.v[r], self.kv_lens[r] - n, window, sinks,
                                      (pg >= 0) & (pg < len(self.K)))
                bo, bs = bounds(o, lse, need, self.q.dtype, self.hd)
                m = n if max_q is None else min(max_q, n)
                check(self.out[s][:m], o[:m], bo[:m], (what, r, "out"))
                check(self.lse[s][:m], lse[:m], bs[:m], (what, r, "lse"))
                assert (self.out[s][m:] == 7.0).all()
        for rest in (slice(0, self.cu[0]), slice(self.cu[-1], len(self.q))):
            assert (self.out[rest] == 7.0).all() and (self.lse[rest] == 7.0).all()


TYPES = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("H,KVH,hd", HEADS)
@pytest.mark.parametrize("q_lens,kv_lens,page,window,sinks", [
    ([1], [1], 16, 0, True), ([1, 1, 1], [37, 500, 8], 8, 0, False), ([1, 0, 1], [300, 40, 129], 32, 128, True),
    ([3, 1, 8], [700, 70, 8], 16, 0, True), ([50, 1, 130], [50, 1000, 333], 64, 0, False),
    ([40, 1, 0, 7], [400, 90, 10, 300], 128, 33, True), ([1], [2300], 256, 0, True)])
def test_paged(eng, act, cache, H, KVH, hd, q_lens, kv_lens, page, window, sinks):
    gen = torch.Generator(device="cuda").manual_seed(H + hd + sum(kv_lens))
    p = Paged(gen, q_lens, kv_lens, H, KVH, hd, act, cache, page, behind=40, first=2, wide=1)
    sk = randn(gen, (H,), F32, 2.0) if sinks else None
    p.run(eng, window=window, sinks=sk)
    p.verify(window, sk)


@pytest.mark.parametrize("act,cache", TYPES)
def test_paged_long(eng, act, cache):
    """One request alone over many positions (the work of a row is split), ragged
    requests beside it, chunks over a long history, windows."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    for q_lens, kv_lens, heads, page, window in (([1], [30011], (8, 1, 64), 16, 0), ([1, 1, 1], [9, 20000, 777], (16, 2, 128), 64, 0),
                                                 ([60], [9000], (8, 2, 64), 32, 0), ([5], [9001], (4, 4, 128), 8, 4000),
                                                 ([1] * 40, [100 + 37 * i for i in range(40)], (8, 1, 64), 16, 0),
                                                 ([300, 1, 1], [5000, 4000, 3], (8, 1, 64), 16, 700)):
        p = Paged(gen, q_lens, kv_lens, *heads, act, cache, page)
        for max_kv in (0, max(kv_lens)):
            p.out.fill_(7.0)
            p.run(eng, window=window, max_kv=max_kv)
            p.verify(window, what=(q_lens[:3], kv_lens[:3], max_kv))


@pytest.mark.parametrize("act,cache", TYPES)
def test_paged_empty_rows_and_bad_pages(eng, act, cache):
    """Rows before position 0, requests without positions, table entries that
    name no page: what is not seen counts nothing, a row that sees nothing is 0."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    for q_lens, kv_lens in (([1, 1, 1], [0, 5, 600]), ([4, 20, 33], [2, 0, 600])):
        for sinks in (None, randn(gen, (8,), F32)):
            p = Paged(gen, q_lens, kv_lens, 8, 2, 64, act, cache, 16)
            p.run(eng, sinks=sinks)
            for r in range(3):
                s, hidden = slice(p.cu[r], p.cu[r + 1]), max(0, q_lens[r] - kv_lens[r])
                want = sinks.expand(hidden, 8) if sinks is not None else torch.full((hidden, 8), -math.inf, device="cuda")
                assert (p.out[s][:hidden] == 0).all()
                # (the sink times log2 e and back: two half steps)
                check(p.lse[s][:hidden], want.double(), 2 * 2.0 ** -24 * want.double().abs(), "empty")
            p.verify(0, sinks)
            for r, b in ((2, 0), (2, 7), (2, 37), (1, 0)):
                p.tab[r][b] = (-1, len(p.K), -2 ** 31, 2 ** 31 - 1)[(r + b) % 4]
            p.run(eng, sinks=sinks)
            p.verify(0, sinks, what="bad pages")
            for b in range(len(p.tab[2])):
                p.tab[2][b] = -1
            p.run(eng, sinks=sinks)
            p.verify(0, sinks, what="no pages")


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("q", [1, 6, 40])
def test_paged_masked_specials(eng, act, cache, q):
    """NaN and infinities in values that some of a request's rows see and others
    do not (later positions, positions that left the window)."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    for window in (0, 60):
        p = Paged(gen, [q, q], [400, 90], 8, 2, 64, act, cache, 16)
        p.v[0][399, 0, 3] = float("nan")
        p.v[0][400 - q, 1, 4] = float("inf")
        p.v[1][90 - q // 2 - 1, 1, 9] = -float("inf")
        p.v[1][max(0, 90 - q - 58), 0, 9] = float("inf")
        p.k[1][89, 1, 1] = float("nan")
        p.fill()
        p.run(eng, window=window)
        p.verify(window)


def test_paged_max_q(eng):
    """Rows beyond max_q are left as they were."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    for q_lens, m in (([9, 1, 3], 2), ([200, 5], 100), ([40], 1)):
        p = Paged(gen, q_lens, [300] * len(q_lens), 8, 2, 64, BF16, BF16, 16)
        p.run(eng, max_q=m)
        p.verify(max_q=m)


def test_paged_rows_beyond_max_q_in_windows(eng):
    """Far more rows than max_q: only the positions of the computed rows count
    (their windows lie far before the request's end), and the call after it, which
    splits its request, is not touched by it."""
    gen = torch.Generator(device="cuda").manual_seed(15)
    a = Paged(gen, [1000, 900], [1000, 5000], 8, 2, 64, BF16, BF16, 16)
    b = Paged(gen, [1, 1], [9000, 700], 8, 2, 64, BF16, BF16, 16)
    for window, m in ((1, 1), (100, 2), (0, 2)):
        a.out.fill_(7.0)
        a.run(eng, max_q=m, window=window)
        a.verify(window, max_q=m)
        b.run(eng)
        b.verify()


@pytest.mark.parametrize("act,cache", [(F32, F16), (BF16, BF16)])
def test_paged_widest_window(eng, act, cache):
    """A window of 2^31 - 1 is none, also beside rows before position 0."""
    gen = torch.Generator(device="cuda").manual_seed(16)
    for q_lens, kv_lens in (([3, 2], [2, 300]), ([50, 40], [20, 300])):
        p = Paged(gen, q_lens, kv_lens, 8, 2, 64, act, cache, 16)
        p.run(eng, window=2 ** 31 - 1)
        p.verify()


# fp32 in workgroups of eight waves: columns for all of the device, whole heads
@pytest.mark.parametrize("H,KVH,hd,lens,window", [(64, 8, 64, [2100], 0), (32, 8, 128, [1100, 1050], 0),
                                                  (16, 16, 64, [4133], 0), (64, 8, 64, [2200], 300)])
def test_packed_fp32_full_device(eng, H, KVH, hd, lens, window):
    gen = torch.Generator(device="cuda").manual_seed(17)
    p = Packed(gen, lens, H, KVH, hd, F32, first=1, behind=9)
    sk = randn(gen, (H,), F32, 2.0)
    p.run(eng, window=window, sinks=sk)
    p.verify(window, sk)


@pytest.mark.parametrize("H,KVH,hd,window", [(64, 8, 64, 0), (32, 8, 128, 0), (32, 8, 128, 700)])
@pytest.mark.parametrize("cache", [F32, F16, BF16])
def test_paged_fp32_full_device(eng, cache, H, KVH, hd, window):
    """A chunk of 300 rows: eight waves, keys split; pages that are none."""
    gen = torch.Generator(device="cuda").manual_seed(18)
    p = Paged(gen, [300], [9000], H, KVH, hd, F32, cache, 16, behind=5)
    for b in (0, 77, 540):
        p.tab[0][b] = -1
    p.run(eng, window=window, max_kv=9000)
    p.verify(window)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("q,kv", [(300, 9000), (600, 600)])
def test_paged_specials_in_split_keys(eng, act, cache, q, kv):
    """Values that are not finite near the causal edge and deep in the history
    of a chunk whose keys are split: rows that see them have them, the others
    are exact."""
    gen = torch.Generator(device="cuda").manual_seed(19)
    p = Paged(gen, [q], [kv], 16, 8, 64, act, cache, 32)
    p.v[0][kv - 1, 0, 3] = float("nan")
    p.v[0][kv - q // 2, 1, 4] = float("inf")
    p.v[0][kv - q + 1, 2, 40] = -float("inf")
    p.v[0][100, 3, 63] = float("inf")
    p.k[0][kv - 7, 4, 0] = float("nan")
    p.fill()
    p.run(eng, max_kv=kv)
    p.verify()


@pytest.mark.parametrize("hd,KVH", [(64, 8), (128, 8)])
def test_packed_fp32_specials_full_device(eng, hd, KVH):
    gen = torch.Generator(device="cuda").manual_seed(20)
    p = Packed(gen, [2100], 8 * KVH if hd == 64 else 4 * KVH, KVH, hd, F32)
    p.v[2099, 1, 5] = float("nan")
    p.v[1500, 3, 6] = float("inf")
    p.v[3, 4, 7] = -float("inf")
    p.run(eng)
    p.verify()


def test_paged_far_offsets(eng):
    """Pages whose elements lie beyond 2^31 and 2^32 elements (and 2^32 bytes)."""
    import picchio_amd as pa
    n_pages, KVH, page, hd = 18000, 8, 256, 128                        # 4.7e9 elements
    gen = torch.Generator(device="cuda").manual_seed(10)
    K = torch.empty((n_pages, KVH, page, hd), device="cuda", dtype=BF16)
    V = torch.empty((n_pages, KVH, page, hd), device="cuda", dtype=BF16)
    ids = [n_pages - 1, 9000, 3, 17000, 8192, 16384]
    for q, lens in ((1, [1500]), (40, [1500]), (1, [700, 800])):
        for i in ids:
            K[i] = randn(gen, K[i].shape, BF16)
            V[i] = randn(gen, V[i].shape, BF16)
        n = len(lens)
        tab = [ids] if n == 1 else [ids[:3], ids[3:]]
        Q, out = randn(gen, (q * n, 16, hd), BF16), torch.zeros((q * n, 16, hd), device="cuda", dtype=BF16)
        call = pa.attn_paged(Q, out, ints(starts([q] * n)), ints(lens), ints(tab), pa.pages(K, V), q)
        torch.cuda.synchronize()
        eng.attention_paged(call)
        # and the store into far pages
        slots = ints([ids[0] * page + 255, ids[3] * page, 8 * page])
        k = randn(gen, (3, KVH, hd), BF16)
        eng.sync()
        for r in range(n):
            t = torch.tensor(tab[r], device="cuda")
            k0, v0 = (x[t].transpose(1, 2).flatten(0, 1)[:lens[r]] for x in (K, V))
            o, lse, need = attend(Q[r * q:(r + 1) * q], k0, v0, lens[r] - q)
            check(out[r * q:(r + 1) * q], o, bounds(o, lse, need, BF16, hd)[0], (q, r))
        torch.cuda.synchronize()
        eng.store_pages(pa.kv_rows(None, k, k, None, ints([0, 0, 0]), slots, pa.pages(K, V)))
        eng.sync()
        for i, s in enumerate(slots.tolist()):
            assert torch.equal(K[s // page, :, s % page], k[i]) and torch.equal(V[s // page, :, s % page], k[i])


@pytest.mark.parametrize("act,cache", [(F32, BF16), (BF16, BF16), (F32, F32)])
def test_paged_captured(eng, act, cache):
    """A captured call reads rows, lengths and tables anew at each replay; two
    graphs of the same engine between each other and eager calls."""
    gen = torch.Generator(device="cuda").manual_seed(11)
    a = Paged(gen, [1, 1, 1], [3000, 20, 700], 8, 1, 64, act, cache, 16)
    b = Paged(gen, [30, 9, 1], [1200, 200, 40], 16, 4, 128, act, cache, 32)
    recs, graphs = [a.record(), b.record()], []
    for p, rec in zip((a, b), recs):
        p.run(eng)                                                     # sizes the workspace
        torch.cuda.synchronize()
        eng.capture_begin()
        eng.attention_paged(rec)
        graphs.append(eng.capture_end())
    for turn in range(4):
        for p, rec, g in zip((a, b), recs, graphs):
            p.q.copy_(randn(gen, p.q.shape, act))
            # another request is the long one
            for x in (p.kv_lens, p.k, p.v, p.tab):
                x.append(x.pop(0))
            for r in range(3):
                p.kv_lens[r] = max(p.q_lens[r], p.kv_lens[r] - turn)
                p.k[r], p.v[r] = p.k[r][:p.kv_lens[r]], p.v[r][:p.kv_lens[r]]
            rec.keep[3].copy_(ints(p.kv_lens)), rec.keep[4].copy_(ints(p.tab))
            p.out.fill_(7.0)
            torch.cuda.synchronize()
            eng.graph_launch(g)
            eng.sync()
            ok = all(k >= q for q, k in zip(p.q_lens, p.kv_lens))
            assert ok
            p.verify(what=turn)
        p = Paged(gen, [2, 40], [900, 300], 8, 2, 64, act, cache, 16)
        p.run(eng)
        p.verify(what=("eager", turn))
    for g in graphs:
        eng.graph_destroy(g)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_same_bits_again(eng, dtype):
    """No sum depends on the order in which workgroups arrive."""
    gen = torch.Generator(device="cuda").manual_seed(12)
    p = Packed(gen, [700, 300], 8, 2, 64, dtype)
    g = Paged(gen, [1, 60, 3], [9000, 4000, 2000], 8, 1, 64, dtype, dtype, 16)
    seen = []
    for _ in range(5):
        p.run(eng), g.run(eng)
        seen.append([x.clone() for x in (p.out, p.lse, g.out, g.lse)])
    for s in seen[1:]:
        assert all(torch.equal(x, y) for x, y in zip(s, seen[0]))


def test_two_engines_at_once(eng, gpu):
    """Calls of two engines run beside each other, each on its own stream with its
    own workspace: split decode steps, mixed steps, and a torch stream's work
    between them."""
    import picchio_amd as pa
    gen = torch.Generator(device="cuda").manual_seed(21)
    with pa.Engine(pa.gptoss_cfg(n_layers=1, n_experts=4, ctx_len=16, vocab=64)) as other:
        a = Paged(gen, [1, 1, 1], [9000, 20, 700], 8, 1, 64, F32, F16, 16)
        b = Paged(gen, [60, 1, 3], [7000, 4000, 2000], 8, 1, 64, F32, F16, 16)
        ra, rb = a.record(), b.record()
        for e in (eng, other):                                         # sizes the workspaces
            e.attention_paged(ra), e.attention_paged(rb)
            e.sync()
        a.out.fill_(7.0), b.out.fill_(7.0)
        noise = torch.zeros(1 << 20, device="cuda")
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        for _ in range(20):
            eng.attention_paged(ra)
            other.attention_paged(rb)
            with torch.cuda.stream(side):
                noise += 1.0
        eng.sync(), other.sync()
        torch.cuda.synchronize()
        a.verify(what="first"), b.verify(what="second")
        assert (noise == 20.0).all()


@pytest.mark.parametrize("n", [64, 65, 100, 128, 129, 200, 256, 257, 1000])
def test_paged_many_requests(eng, n):
    """More requests than a wave's lanes or a workgroup finds at once: some idle,
    one far longer than the others, some of several rows."""
    gen = torch.Generator(device="cuda").manual_seed(13)
    kv = [1 + (37 * i) % 150 for i in range(n)]
    q = [0 if i % 7 == 3 else min(k, 1 + (i % 11 == 5)) for i, k in enumerate(kv)]
    kv[n // 3] = 6000
    p = Paged(gen, q, kv, 8, 2, 64, BF16, BF16, 16)
    p.run(eng)
    p.verify()


@pytest.mark.parametrize("act,cache", [(F32, F16), (F32, BF16), (F16, F16)])
def test_paged_magnitudes(eng, act, cache):
    """Queries from 2^-40 to 2^40 in rows of one call, over keys that bring the
    scores back to around 1 (fp32 queries over a 16-bit cache are scaled and cut
    into planes); values at the ends of the cache's type."""
    gen = torch.Generator(device="cuda").manual_seed(14)
    p = Paged(gen, [1] * 5, [300] * 5, 8, 2, 64, act, cache, 16)
    e = [-40, -20, 0, 20, 40] if act == F32 and cache == BF16 else [-12, -6, 0, 6, 10]
    for r in range(5):
        p.q[r] *= 2.0 ** e[r]
        p.k[r] *= 2.0 ** -e[r]
        p.v[r] *= 2.0 ** (10 if cache == F16 else 60) if r % 2 else 2.0 ** (-10 if cache == F16 else -60)
    p.fill()
    p.run(eng)
    p.verify()
