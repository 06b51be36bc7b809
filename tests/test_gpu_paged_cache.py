"""plan_pages and store_pages against plain Python and 64 bits, and a run of
the paged operators together over several steps."""
import random

import numpy as np
import pytest
import torch

from paged_ref import HALF_STEP, attend, bounds, check, plan, rotate

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng(gpu):
    import picchio_amd as pa
    with pa.Engine(pa.gptoss_cfg(n_layers=1, n_experts=4, ctx_len=300, vocab=64)) as e:
        yield e


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Plan:
    """Device and Python state of the same requests."""

    def __init__(self, eng, n, blocks, n_pages, page, max_tokens, seed=0):
        import picchio_amd as pa
        r = random.Random(seed)
        self.eng, self.page, self.max_tokens = eng, page, max_tokens
        self.table = [[-1] * blocks for _ in range(n)]
        self.ring = r.sample(range(n_pages), n_pages)
        self.state = [r.randrange(n_pages), n_pages]
        self.d = dict(table=ints(self.table).reshape(n, blocks), ring=ints(self.ring), state=ints(self.state + [0, 0]))
        self.old, self.new = ints([0] * n), ints([0] * n)
        self.out = dict(length=ints([0] * n), cu_q=ints([-9] * (n + 1)), slot=ints([-9] * max_tokens),
                        pos=ints([-9] * max_tokens))
        self.call = pa.page_plan(self.old, self.new, self.d["table"], self.d["ring"], self.d["state"], page, **self.out)

    def step(self, old, new, launch=None):
        self.old.copy_(ints(old)), self.new.copy_(ints(new))
        for t in self.out.values():
            t.fill_(-9)
        torch.cuda.synchronize()
        (launch or (lambda: self.eng.plan_pages(self.call)))()
        self.eng.sync()
        want = plan(old, new, self.table, self.ring, self.state, self.page, self.max_tokens)
        for name, w in zip(("length", "cu_q", "slot", "pos"), want):
            assert self.out[name].tolist() == w, name
        assert self.d["table"].tolist() == self.table
        assert self.d["ring"].tolist() == self.ring
        assert self.d["state"].tolist() == self.state + [0, 0]
        return want[0]


def random_steps(p, n, cap, seed, steps, launch=None):
    r, lens = random.Random(seed), [0] * n
    for _ in range(steps):
        new = [r.choice([x, x + 1, x + 1, x + r.randint(0, cap), max(0, x - r.randint(0, 9)), 0]) for x in lens]
        lens = p.step(lens, [min(x, cap + 5) for x in new], launch)


@pytest.mark.parametrize("n,blocks,n_pages,page,tokens", [(1, 1, 1, 8, 8), (5, 9, 20, 16, 100), (64, 4, 100, 32, 700),
                                                          (513, 3, 900, 8, 4000), (4096, 2, 5000, 256, 9000),
                                                          (7, 100, 701, 16, 12000)])
def test_plan_steps(eng, n, blocks, n_pages, page, tokens):
    """Steps at random: growth, idling, giving back, pages and rows running out."""
    random_steps(Plan(eng, n, blocks, n_pages, page, tokens, n), n, blocks * page, n + 1, 6)


def test_plan_many_rows(eng):
    """Rows for more workgroups than arrive on one word, captured and replayed too;
    the rows' arrays off 16 bytes."""
    import picchio_amd as pa
    p = Plan(eng, 20, 300, 6100, 32, 150001, 1)
    random_steps(p, 20, 9600, 2, 4)
    p = Plan(eng, 20, 300, 6100, 32, 150001, 2)
    torch.cuda.synchronize()
    eng.capture_begin()
    eng.plan_pages(p.call)
    g = eng.capture_end()
    random_steps(p, 20, 9600, 3, 4, lambda: eng.graph_launch(g))
    eng.graph_destroy(g)
    p = Plan(eng, 20, 300, 6100, 32, 70001, 3)
    for name in ("slot", "pos"):
        p.out[name] = ints([-9] * 70002)[1:]
    p.call = pa.page_plan(p.old, p.new, p.d["table"], p.d["ring"], p.d["state"], 32, **p.out)
    random_steps(p, 20, 9600, 4, 4)


def test_plan_edges(eng):
    p = Plan(eng, 3, 4, 6, 16, 50)
    assert p.step([0, 0, 0], [16, 17, 1]) == [16, 17, 1]                    # a full page, one over, one row
    assert p.step([16, 17, 1], [49, 17, 2]) == [16, 17, 1]                  # 3 pages wanted, 2 free: nothing behind it either
    assert p.step([16, 17, 1], [48, 0, 1]) == [48, 0, 1]                    # 2 pages taken, 2 given back
    assert p.step([48, 0, 1], [48, 51, 1]) == [48, 0, 1]                    # more rows than there is room for
    assert p.step([48, 0, 1], [-3, -1, 1000]) == [0, 0, 1]                  # lengths are cut to the table
    assert p.step([0, 0, 1], [0, 0, 1]) == [0, 0, 1]                        # nothing to do
    q = Plan(eng, 0, 4, 6, 16, 5)
    assert q.step([], []) == []


def test_plan_bad_entries(eng):
    """A table entry that names no page gives slot -1."""
    p = Plan(eng, 2, 4, 8, 8, 20)
    p.step([0, 0], [4, 4])
    for bad in (-1, 8, 2 ** 31 - 1):
        p.table[1][0] = bad
        p.d["table"].copy_(ints(p.table))
        p.step([4, 4], [6, 6])
        p.step([6, 6], [4, 4])


def test_plan_captured(eng):
    p = Plan(eng, 40, 5, 150, 16, 600, 3)
    torch.cuda.synchronize()
    eng.capture_begin()
    eng.plan_pages(p.call)
    g = eng.capture_end()
    random_steps(p, 40, 80, 5, 8, lambda: eng.graph_launch(g))
    eng.graph_destroy(g)


def rows(gen, T, H, KVH, hd, dtype):
    x = torch.randn((T, (H + 2 * KVH) * hd), generator=gen, device="cuda").to(dtype)
    return (x[:, :H * hd].unflatten(1, (H, hd)), x[:, H * hd:(H + KVH) * hd].unflatten(1, (KVH, hd)),
            x[:, (H + KVH) * hd:].unflatten(1, (KVH, hd)))


TYPES = [(torch.float32, torch.float32), (torch.float32, torch.float16), (torch.float32, torch.bfloat16),
         (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16)]


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("T,H,KVH,hd,page", [(1, 64, 8, 64, 16), (7, 1, 1, 16, 8), (300, 12, 2, 96, 32), (33, 5, 5, 128, 256),
                                             (1000, 10, 5, 32, 64), (2, 300, 100, 48, 8)])
def test_store(eng, act, cache, T, H, KVH, hd, page):
    import picchio_amd as pa
    gen = torch.Generator(device="cuda").manual_seed(T + hd)
    n_pages, far = -(-T // page) + 3, 517
    q, k, v = rows(gen, T, H, KVH, hd, act)
    slot = torch.randperm(n_pages * page, generator=gen, device="cuda")[:T].int()
    pos = torch.randint(0, far, (T,), generator=gen, device="cuda", dtype=torch.int32)
    out = [(5, n_pages * page), (6, -1), (9, -2 ** 31)]          # no slot; positions outside the table
    for i, s in out:
        if i < T:
            slot[i] = s
    for i, s in ((11, far), (12, -1)):
        if i < T:
            pos[i] = s
    rope = torch.randn((far, hd // 2, 2), generator=gen, device="cuda")
    K = torch.randn((n_pages, KVH, page, hd), generator=gen, device="cuda").to(cache)
    V = torch.randn((n_pages, KVH, page, hd), generator=gen, device="cuda").to(cache)
    there = (slot >= 0) & (slot < n_pages * page) & (pos >= 0) & (pos < far)
    at = slot[there].long()

    def flat(x):
        return x.transpose(1, 2).reshape(n_pages * page, KVH, hd)

    for table in (rope, None):
        ok = there if table is not None else (slot >= 0) & (slot < n_pages * page)
        at = slot[ok].long()
        k0, v0, q0 = K.clone(), V.clone(), torch.full((T, H, hd), 7.0, device="cuda").to(act)
        call = pa.kv_rows(q, k, v, q0, pos, slot, pa.pages(k0, v0), rope=table)
        torch.cuda.synchronize()
        eng.store_pages(call)
        eng.sync()
        turn = (lambda x: rotate(x[ok], pos[ok], table)) if table is not None else (lambda x: x[ok].double())
        # a product and a multiply-add of fp32, then one rounding to the type
        def bound(x, w, dtype):
            reach = (x[ok].double().abs().amax(2, keepdim=True) * 2 * (table.abs().max().double() if table is not None else 0))
            return HALF_STEP[dtype] * w.abs() * 1.01 + 2 * 2.0 ** -24 * reach + torch.finfo(dtype).tiny
        check(q0[ok], turn(q), bound(q, turn(q), act), "q_out")
        assert torch.equal(q0[~ok], torch.full_like(q0[~ok], 7.0))
        check(flat(k0)[at], turn(k), bound(k, turn(k), cache), "k")
        assert torch.equal(flat(v0)[at], v[ok].to(cache))
        rest = torch.ones(n_pages * page, dtype=torch.bool, device="cuda")
        rest[at] = False
        assert torch.equal(flat(k0)[rest], flat(K)[rest]) and torch.equal(flat(v0)[rest], flat(V)[rest])
    # in place, and without queries
    k1, v1, qq = K.clone(), V.clone(), q.clone()
    q1 = torch.full((T, H, hd), 7.0, device="cuda").to(act)
    torch.cuda.synchronize()
    eng.store_pages(pa.kv_rows(qq, k, v, qq, pos, slot, pa.pages(k1, v1), rope=rope))
    eng.store_pages(pa.kv_rows(q, k, v, q1, pos, slot, pa.pages(K, V), rope=rope))
    eng.store_pages(pa.kv_rows(None, k, v, None, pos, slot, pa.pages(K, V), rope=rope))
    eng.sync()
    assert torch.equal(k1, K) and torch.equal(v1, V)
    assert torch.equal(qq[there], q1[there]) and torch.equal(qq[~there], q[~there])


def test_store_rounds_and_keeps_specials(eng):
    import picchio_amd as pa
    x = torch.tensor([0.0, -0.0, float("inf"), -float("inf"), float("nan"), 1e-45, 65519.0, 65520.0, 3.3e38, 1 + 2.0 ** -8,
                      1 + 3 * 2.0 ** -8, 1 + 2.0 ** -11, 2.0 ** -25, 6e-8, -1.5, 3.14159], device="cuda").reshape(1, 1, 16)
    for cache in (torch.float16, torch.bfloat16):
        K, V = torch.zeros((1, 1, 8, 16), device="cuda", dtype=cache), torch.zeros((1, 1, 8, 16), device="cuda", dtype=cache)
        torch.cuda.synchronize()
        eng.store_pages(pa.kv_rows(None, x, x, None, ints([0]), ints([3]), pa.pages(K, V)))
        eng.sync()
        for t in (K, V):
            assert torch.equal(t[0, 0, 3].view(torch.int16)[~torch.isnan(x[0, 0])],
                               x[0, 0].to(cache).view(torch.int16)[~torch.isnan(x[0, 0])])
            assert torch.isnan(t[0, 0, 3, 4])


def test_steps_together(eng):
    """Five requests over eight steps (prompts, single tokens, a rejected tail,
    an end, a new request on given-back pages) as a server runs them: plan, store
    with the engine's own rotation table, attend; every step's rows against 64
    bits over each request's own history, and the prompts packed."""
    import picchio_amd as pa
    H, KVH, hd, page, n, blocks, most = 8, 2, 64, 16, 5, 10, 120
    gen, n_pages = torch.Generator(device="cuda").manual_seed(1), 26
    address, far = eng.rope()
    assert far == 300
    p = Plan(eng, n, blocks, n_pages, page, most, 9)
    K = torch.full((n_pages, KVH, page, hd), float("nan"), device="cuda", dtype=torch.bfloat16)
    V = K.clone()
    q_rot, out, lse = (torch.zeros((most, H, hd), device="cuda"), torch.zeros((most, H, hd), device="cuda"),
                       torch.zeros((most, H), device="cuda"))
    sinks = torch.randn(H, generator=gen, device="cuda")
    history = [[] for _ in range(n)]
    x = torch.zeros((most, (H + 2 * KVH) * hd), device="cuda")
    q, k, v = (x[:, :H * hd].unflatten(1, (H, hd)), x[:, H * hd:(H + KVH) * hd].unflatten(1, (KVH, hd)),
               x[:, (H + KVH) * hd:].unflatten(1, (KVH, hd)))
    store = pa.kv_rows(q, k, v, q_rot, p.out["pos"], p.out["slot"], pa.pages(K, V), rope=(address, far))
    att = pa.attn_paged(q_rot, out, p.out["cu_q"], p.out["length"], p.d["table"], pa.pages(K, V), 100, 160, sinks=sinks,
                        lse=lse)
    rope = torch.empty((far, hd // 2, 2), device="cuda")
    import ctypes
    hip = ctypes.CDLL("libamdhip64.so")
    assert hip.hipMemcpy(ctypes.c_void_p(rope.data_ptr()), ctypes.c_void_p(address), ctypes.c_size_t(rope.numel() * 4), 3) == 0
    lens = [0] * n
    for step, new in enumerate([[70, 0, 5, 0, 0], [71, 33, 6, 0, 16], [72, 34, 7, 100, 17], [73, 31, 8, 101, 18],
                                [74, 32, 0, 102, 19], [75, 33, 40, 103, 20], [150, 34, 41, 104, 21], [151, 35, 42, 105, 0]]):
        x.copy_(torch.randn(x.shape, generator=gen, device="cuda"))
        out.fill_(5.0)
        got = p.step(lens, new)
        assert got == new
        eng.store_pages(store)
        eng.attention_paged(att)
        eng.sync()
        cu = p.out["cu_q"].tolist()
        for r in range(n):
            history[r] = history[r][:min(lens[r], new[r])]
            a, b = cu[r], cu[r + 1]
            if b == a:
                continue
            at = torch.arange(lens[r], new[r], device="cuda")
            stored = [z.transpose(1, 2).reshape(n_pages * page, KVH, hd)[p.out["slot"][a:b].long()] for z in (K, V)]
            for z, turned, dtype in ((stored[0], rotate(k[a:b], at, rope), K.dtype),
                                     (q_rot[a:b], rotate(q[a:b], at, rope), q_rot.dtype)):
                check(z, turned, HALF_STEP[dtype] * 1.01 * turned.abs() + 2.0 ** -20, (step, r, "rotation"))
            assert torch.equal(stored[1], v[a:b].to(V.dtype))
            history[r] += list(zip(*stored))
            kk, vv = (torch.stack([z[i] for z in history[r]]) for i in (0, 1))
            o, s, need = attend(q_rot[a:b], kk, vv, lens[r], sinks=sinks)
            bo, bs = bounds(o, s, need, torch.float32, hd)
            check(out[a:b], o, bo, (step, r))
            check(lse[a:b], s, bs, (step, r, "lse"))
        assert (out[cu[-1]:] == 5.0).all()
        lens = got
