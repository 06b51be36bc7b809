"""The paged-cache operators of serving several requests, as timed cases.

A case is a dict of plain values; its "kind" names the operator:

  plan     plan_pages: block tables, free pages, query starts, slots and
           positions of a step, from the requests' lengths before and after
           it; a pass is the step and its way back (what one call takes from
           the free pages the other returns), so that passes can follow
           each other
  store    store_pages: rotary embedding of a step's query and key rows, keys
           and values converted and written to their slots of the paged cache
  packed   attention_packed: causal attention of whole prompts of different
           lengths, packed row behind row
  paged    attention_paged: attention of each request's new rows (one, a few,
           a chunk) over its pages

`own` false: elementary torch operations in 32 bits. `own` true: the calls
that a program makes of this package, which keeps the calls' argument records
beside its buffers as it keeps the buffers.

Head layouts: the GPT-OSS one (64 query heads over 8 KV heads of 64) and
generic ones (heads of 32 to 128, one KV head to one per query head). q, k and
v of a packed prompt or a step are slices of one fused QKV row, as a
projection writes them. Pages are handed out in no order, and table entries
behind a request's pages are -1.
"""
import functools
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
GPTOSS = dict(H=64, KVH=8, hd=64)


def listed():
    return [
        # one decode step of 32 running requests, a few ending or newly admitted
        dict(name="plan_step_32", kind="plan", n=32, page=16, longest=8192, chunk=64, mix=1),
        # a full server: 1000 requests, among them prompt chunks of up to 512 tokens
        dict(name="plan_1000", kind="plan", n=1000, page=32, longest=16384, chunk=512, mix=2),
        # the rows of one decode step, fp32 activations into a bf16 cache
        dict(name="store_step_32", kind="store", T=32, pad=0, page=16, pages=4096, act="f32", cache="bf16", **GPTOSS),
        # the rows of a prompt pass with the captured launch's padding rows behind them
        dict(name="store_prompt_8192", kind="store", T=8192, pad=192, page=32, pages=1024, act="bf16", cache="bf16",
             **GPTOSS),
        # twelve prompts of up to 4096 tokens in one pass
        dict(name="packed_bf16", kind="packed", n=12, longest=4096, type="bf16", window=0, mix=3, **GPTOSS),
        # the sliding-window layer of the same kind of pass
        dict(name="packed_window_f16", kind="packed", n=5, longest=4001, type="f16", window=128, mix=4, **GPTOSS),
        # fp32 prompts, heads of 128
        dict(name="packed_f32", kind="packed", n=4, longest=1500, type="f32", window=0, mix=5, H=32, KVH=8, hd=128),
        # a decode step of 32 requests of up to 8192 positions
        dict(name="paged_step_32", kind="paged", n=32, longest=8192, chunk=1, chunks=0, act="bf16", cache="bf16", page=16,
             window=0, mix=6, **GPTOSS),
        # one request alone after 100,000 positions, fp32 activations over an f16 cache
        dict(name="paged_long_1", kind="paged", n=1, longest=100001, chunk=1, chunks=0, act="f32", cache="f16", page=64,
             window=0, mix=7, **GPTOSS),
        # one short request, fp32 throughout: the call's latency
        dict(name="paged_short_1", kind="paged", n=1, longest=37, chunk=1, chunks=0, act="f32", cache="f32", page=16,
             window=0, mix=8, H=16, KVH=16, hd=128),
        # a chunk of a long prompt beside nothing else
        dict(name="paged_chunk_512", kind="paged", n=1, longest=24000, chunk=512, chunks=1, act="bf16", cache="bf16",
             page=32, window=0, mix=9, **GPTOSS),
        # a mixed step: three prompt chunks among 29 decoding requests, fp32 activations
        dict(name="paged_mixed", kind="paged", n=32, longest=6000, chunk=300, chunks=3, act="f32", cache="bf16", page=16,
             window=0, mix=10, **GPTOSS),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind, mix = rng.choice(["plan", "store", "packed", "packed", "paged", "paged", "paged"]), rng.randrange(1 << 20)
    heads = rng.choice([GPTOSS, GPTOSS, GPTOSS, dict(H=32, KVH=8, hd=128), dict(H=16, KVH=16, hd=128),
                        dict(H=12, KVH=2, hd=96), dict(H=8, KVH=1, hd=64), dict(H=10, KVH=5, hd=32)])
    page, window = rng.choice([8, 16, 16, 32, 64, 128]), rng.choice([0, 0, 0, 128, rng.randint(1, 2000)])
    if kind == "plan":
        return dict(kind=kind, n=_log(rng, 1, 1000), page=page, longest=_log(rng, 64, 16384), chunk=_log(rng, 1, 512), mix=mix)
    act = rng.choice(["f32", "f16", "bf16", "bf16"])
    cache = rng.choice(["f32", "f16", "bf16"]) if act == "f32" else act
    if kind == "store":
        return dict(kind=kind, T=_log(rng, 1, 8192), pad=rng.choice([0, 0, rng.randint(1, 100)]), page=page,
                    pages=_log(rng, 9000 // page + 20, 60000 // page), act=act, cache=cache, **heads)
    if kind == "packed":
        n = _log(rng, 1, 12)
        return dict(kind=kind, n=n, longest=_log(rng, 1, 4096 if act != "f32" else 1500), type=act, window=window, mix=mix,
                    **heads)
    chunk = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 512)])
    n = _log(rng, 1, 32)
    return dict(kind=kind, n=n, longest=_log(rng, chunk + 16, 100000 // n if n > 12 else 24000), chunk=chunk,
                chunks=(rng.randint(1, 3) if n > 12 else 1) if chunk > 8 else n if chunk > 1 else 0, act=act, cache=cache,
                page=page, window=window, mix=mix, **heads)


# ───────────────────────────── lengths ─────────────────────────────

def _lengths(n, longest, mix, lowest=1):
    """n lengths, the longest among them, the others over a factor of 16."""
    r = random.Random(mix)
    v = [longest] + [_log(r, max(lowest, longest // 16), max(lowest, longest)) for _ in range(n - 1)]
    r.shuffle(v)
    return v


def _plan_lengths(case):
    """(lengths before, after) of a step: most requests grow by a token or are
    idle, some by a chunk or are admitted, some end or give tokens back."""
    r, old, new = random.Random(case["mix"]), [], []
    for length in _lengths(case["n"], case["longest"], case["mix"] + 1):
        what, more = r.random(), r.randint(1, case["chunk"])
        a, b = (length - 1, length) if what < 0.6 else (max(0, length - more), length) if what < 0.7 else \
               (0, min(length, more)) if what < 0.8 else (length, 0) if what < 0.9 else \
               (length, max(0, length - more)) if what < 0.95 else (length, length)
        old.append(a), new.append(b)
    return old, new


def _paged_lengths(case):
    """(new rows, cached positions with them) per request; the first `chunks`
    requests have a chunk, the others one row."""
    r = random.Random(case["mix"] + 1)
    q = [case["chunk"] if i == 0 else r.randint(max(1, case["chunk"] // 2), case["chunk"]) for i in range(case["chunks"])]
    q += [1] * (case["n"] - len(q))
    return q, _lengths(case["n"], case["longest"], case["mix"], lowest=case["chunk"])


def _pages(n, page):
    return -(-n // page)


# ───────────────────────────── inputs ─────────────────────────────

def _rand(gen, shape, dtype, std=1.0):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    return out.normal_(0.0, std, generator=gen)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cu(v):
    c = [0]
    for x in v:
        c.append(c[-1] + x)
    return _ints(c)


def _tables(gen, lens, page, spare=3):
    """(block tables padded with -1, number of pages): the requests' pages in no order."""
    need = [_pages(x, page) for x in lens]
    total, width = sum(need) + spare, max(max(need), 1)
    perm = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    have = _ints(need).long()
    col = torch.arange(width, device="cuda")[None]
    at = (torch.cumsum(have, 0) - have)[:, None] + col
    return torch.where(col < have[:, None], perm[at.clamp(max=total - 1)], torch.full_like(perm[:1], -1)), total


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    st, kind = dict(case=case), case["kind"]
    if kind == "plan":
        old, new = _plan_lengths(case)
        page, n = case["page"], case["n"]
        most, width = 2 * sum(max(b - a, 0) + max(a - b, 0) for a, b in zip(old, new)) + 8, _pages(case["longest"], page) + 1
        used = sum(_pages(x, page) for x in old)
        total = used + sum(max(_pages(b, page) - _pages(a, page), 0) for a, b in zip(old, new)) + 5
        perm = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
        have, col = _ints([_pages(x, page) for x in old]).long(), torch.arange(width, device="cuda")[None]
        at = ((torch.cumsum(have, 0) - have)[:, None] + col).clamp(max=total - 1)
        st["table"] = torch.where(col < have[:, None], perm[at], torch.full_like(perm[:1], -1))
        # the free pages wait in a ring, from a place of the seed's on
        head = seed % total
        ring = torch.full((total,), -1, dtype=torch.int32, device="cuda")
        ring[(head + torch.arange(total - used, device="cuda")) % total] = perm[used:]
        st.update(old=_ints(old), new=_ints(new), ring=ring, state=_ints([head, total - used, 0, 0]), most=most)
        for way in ("there", "back"):
            st[way] = dict(length=_ints([0] * n), cu_q=_ints([0] * (n + 1)), slot=_ints([0] * most), pos=_ints([0] * most))
        return st
    H, KVH, hd = case["H"], case["KVH"], case["hd"]
    if kind == "store":
        T, act, page, n_pages = case["T"] + case["pad"], TYPES[case["act"]], case["page"], case["pages"]
        qkv = _rand(gen, (T, (H + 2 * KVH) * hd), act)
        slot = torch.randperm(n_pages * page, generator=gen, device="cuda")[:T].to(torch.int32)
        slot[case["T"]:] = -1
        far = 8192                                        # positions that the table covers
        j = torch.arange(hd // 2, device="cuda", dtype=torch.float64)
        ang = torch.arange(far, device="cuda", dtype=torch.float64)[:, None] * 150000.0 ** (-2.0 * j / hd)
        st.update(qkv=qkv, slot=slot, pos=torch.randint(0, far, (T,), generator=gen, device="cuda", dtype=torch.int32),
                  rope=torch.stack([torch.cos(ang), torch.sin(ang)], 2).float(),
                  k_pages=_rand(gen, (n_pages, KVH, page, hd), TYPES[case["cache"]]),
                  v_pages=_rand(gen, (n_pages, KVH, page, hd), TYPES[case["cache"]]),
                  q_out=torch.zeros((T, H, hd), dtype=act, device="cuda"))
        return st
    if kind == "packed":
        lens, act = _lengths(case["n"], case["longest"], case["mix"]), TYPES[case["type"]]
        T = sum(lens)
        st.update(cu=_cu(lens), qkv=_rand(gen, (T, (H + 2 * KVH) * hd), act))
    else:
        (q_lens, lens), act, cache, page = _paged_lengths(case), TYPES[case["act"]], TYPES[case["cache"]], case["page"]
        T = sum(q_lens)
        table, n_pages = _tables(gen, lens, page)
        st.update(cu=_cu(q_lens), kv_len=_ints(lens), table=table, q=_rand(gen, (T, H, hd), act),
                  k_pages=_rand(gen, (n_pages, KVH, page, hd), cache), v_pages=_rand(gen, (n_pages, KVH, page, hd), cache))
    st.update(sinks=_rand(gen, (H,), torch.float32), out=torch.zeros((T, H, hd), dtype=act, device="cuda"),
              lse=torch.zeros((T, H), dtype=torch.float32, device="cuda"))
    return st


def _qkv(st):
    """The fused rows' q, k and v as strided views."""
    c, x = st["case"], st["qkv"]
    H, KVH, hd = c["H"], c["KVH"], c["hd"]
    return (x[:, :H * hd].unflatten(1, (H, hd)), x[:, H * hd:(H + KVH) * hd].unflatten(1, (KVH, hd)),
            x[:, (H + KVH) * hd:].unflatten(1, (KVH, hd)))


# ─────────────────────────── one pass ───────────────────────────

def run(st):
    if own:
        return _own(st)
    return {"plan": _plain_plan, "store": _plain_store, "packed": _plain_packed, "paged": _plain_paged}[st["case"]["kind"]](st)


@functools.lru_cache(None)
def _engine():
    import picchio_amd as pa
    return pa.Engine(pa.gptoss_cfg(n_layers=1, n_experts=4, ctx_len=16, vocab=64))


def _own(st):
    import picchio_amd as pa
    eng, c, kind = _engine(), st["case"], st["case"]["kind"]
    if kind == "plan":
        if "calls" not in st:
            st["calls"] = [pa.page_plan(a, b, st["table"], st["ring"], st["state"], c["page"], **st[way])
                           for a, b, way in ((st["old"], st["new"], "there"), (st["new"], st["old"], "back"))]
        for call in st["calls"]:
            eng.plan_pages(call)
        return {k: st[k] for k in ("there", "back", "table", "ring", "state")}
    if kind == "store":
        if "call" not in st:
            q, k, v = _qkv(st)
            st["call"] = pa.kv_rows(q, k, v, st["q_out"], st["pos"], st["slot"], pa.pages(st["k_pages"], st["v_pages"]),
                                    rope=st["rope"])
        eng.store_pages(st["call"])
        return {k: st[k] for k in ("q_out", "k_pages", "v_pages")}
    if "call" not in st:
        more = dict(window=c["window"], sinks=st["sinks"], lse=st["lse"])
        if kind == "packed":
            q, k, v = _qkv(st)
            st["call"] = pa.attn_packed(q, k, v, st["out"], st["cu"], c["longest"], **more)
        else:
            st["call"] = pa.attn_paged(st["q"], st["out"], st["cu"], st["kv_len"], st["table"],
                                       pa.pages(st["k_pages"], st["v_pages"]), c["chunk"], c["longest"], **more)
    (eng.attention_packed if kind == "packed" else eng.attention_paged)(st["call"])
    return dict(out=st["out"], lse=st["lse"])


def _plain_plan(st):
    page, out = st["case"]["page"], {}
    for a, b, way in ((st["old"], st["new"], "there"), (st["new"], st["old"], "back")):
        out[way] = _plain_plan_step(st, a.long(), b.long(), page, st["most"])
    return dict(out, table=st["table"], ring=st["ring"], state=st["state"])


def _plain_plan_step(st, old, new, page, most):
    table, ring, state = st["table"], st["ring"], st["state"]
    n_pages = ring.numel()
    head, count = state[0].long(), state[1].long()
    ob, nb = (old + page - 1) // page, (new + page - 1) // page
    need, more = (nb - ob).clamp(min=0), (new - old).clamp(min=0)
    # in order, as long as the free pages and the rows suffice
    fits = (torch.cumsum(need, 0) <= count) & (torch.cumsum(more, 0) <= most)
    length = torch.where((new <= old) | fits, new, old)
    rows = torch.where(fits, more, torch.zeros_like(more))
    cu = torch.cat([torch.zeros_like(rows[:1]), torch.cumsum(rows, 0)])
    take = torch.where(fits, need, torch.zeros_like(need))
    give = (ob - nb).clamp(min=0)
    take0, give0 = torch.cumsum(take, 0) - take, torch.cumsum(give, 0) - give
    col = torch.arange(table.shape[1], device="cuda")[None]
    ob, nb = ob[:, None], nb[:, None]
    grown, shrunk = (col >= ob) & (col < ob + take[:, None]), (col >= nb) & (col < ob)
    got = ring[(head + take0[:, None] + col - ob) % n_pages]
    back = (head + count + give0[:, None] + col - nb) % n_pages
    wide = torch.cat([ring, ring[:1]])                       # one entry more for what is not given back
    wide.scatter_(0, torch.where(shrunk, back, torch.full_like(back, n_pages)).reshape(-1), table.reshape(-1))
    ring.copy_(wide[:n_pages])
    table.copy_(torch.where(grown, got, torch.where(shrunk, torch.full_like(table, -1), table)))
    state[0] = (head + take.sum()) % n_pages
    state[1] = count - take.sum() + give.sum()
    t = torch.arange(most, device="cuda")
    r = (torch.searchsorted(cu, t, right=True) - 1).clamp(max=len(old) - 1)
    pos = old[r] + t - cu[r]
    there = t < cu[-1]
    pos = torch.where(there, pos, torch.zeros_like(pos))
    slot = table[r, (pos // page).clamp(max=table.shape[1] - 1)].long() * page + pos % page
    slot = torch.where(there, slot, torch.full_like(slot, -1))
    return dict(length=length.int(), cu_q=cu.int(), slot=slot.int(), pos=pos.int())


def _plain_store(st):
    c, (q, k, v) = st["case"], _qkv(st)
    half, page = c["hd"] // 2, c["page"]
    there = (st["slot"] >= 0)[:, None, None]
    cs = st["rope"][st["pos"].long()][:, None]
    turn = lambda x: torch.cat([x[..., :half] * cs[..., 0] - x[..., half:] * cs[..., 1],
                                x[..., :half] * cs[..., 1] + x[..., half:] * cs[..., 0]], 2)
    st["q_out"].copy_(torch.where(there, turn(q.float()).to(q.dtype), st["q_out"]))
    n = c["T"]                                            # padding rows are behind the step's
    slot = st["slot"][:n].long()
    for pages, rows in ((st["k_pages"], turn(k.float())[:n]), (st["v_pages"], v[:n])):
        pages[slot // page, :, slot % page] = rows.to(pages.dtype)
    return {k: st[k] for k in ("q_out", "k_pages", "v_pages")}


def _softmax_product(q, k, v, seen, sinks, rows):
    """q [n, KVH, G, Q, hd], k and v [n, KVH, L, hd], seen [n, Q, L] -> (out [n, Q, H, hd], lse [n, Q, H]), some KV
    heads at a time so that the scores stay below a few GB."""
    n, KVH, G, Q, hd = q.shape
    L, outs, lses = k.shape[2], [], []
    step = max(1, min(KVH, (1 << 30) // max(1, n * G * Q * L)))
    for h in range(0, KVH, step):
        s = torch.matmul(q[:, h:h + step].reshape(n, -1, G * Q, hd), k[:, h:h + step].transpose(2, 3).contiguous())
        s = s.reshape(n, -1, G, Q, L) * (1.0 / math.sqrt(hd))
        s = torch.where(seen[:, None, None], s, torch.full_like(s[:1, :1, :1, :1, :1], -math.inf))
        sk = sinks.reshape(KVH, G)[None, h:h + step, :, None, None]
        m = torch.maximum(s.amax(4, keepdim=True), sk)
        s = torch.exp(s - m)
        den = s.sum(4, keepdim=True) + torch.exp(sk - m)
        o = torch.matmul(s.reshape(n, -1, G * Q, L), v[:, h:h + step]).reshape(n, -1, G, Q, hd) / den
        outs.append(o)
        lses.append((m + torch.log(den))[..., 0])
    out, lse = torch.cat(outs, 1), torch.cat(lses, 1)
    return out.permute(0, 3, 1, 2, 4).reshape(n, Q, KVH * G, hd)[rows], lse.permute(0, 3, 1, 2).reshape(n, Q, KVH * G)[rows]


def _spread(x, cu, longest):
    """Packed rows [T, ...] as [n, longest, ...], and which entries are rows."""
    at = cu[:-1, None].long() + torch.arange(longest, device="cuda")[None]
    there = at < cu[1:, None]
    return x[at.clamp(max=len(x) - 1)], there


def _heads(x):
    return x.float().permute(0, 2, 1, 3).contiguous()


def _plain_packed(st):
    c, (q, k, v) = st["case"], _qkv(st)
    L, KVH, hd = c["longest"], c["KVH"], c["hd"]
    (q, there), k, v = _spread(q, st["cu"], L), _spread(k, st["cu"], L)[0], _spread(v, st["cu"], L)[0]
    i = torch.arange(L, device="cuda")
    seen = i[None] <= i[:, None]
    if c["window"]:
        seen = seen & (i[None] > i[:, None] - c["window"])
    n = len(q)
    out, lse = _softmax_product(_heads(q).reshape(n, KVH, -1, L, hd), _heads(k), _heads(v), seen[None], st["sinks"], there)
    return dict(out=out.to(TYPES[c["type"]]), lse=lse)


def _plain_paged(st):
    c = st["case"]
    Q, L, KVH, hd, page = c["chunk"], c["longest"], c["KVH"], c["hd"], c["page"]
    q, there = _spread(st["q"], st["cu"], Q)
    n = len(q)
    at = st["table"].long().clamp(min=0)
    k, v = (x[at].permute(0, 2, 1, 3, 4).reshape(n, KVH, -1, hd)[:, :, :L].float() for x in (st["k_pages"], st["v_pages"]))
    L = k.shape[2]
    col = torch.arange(L, device="cuda")[None, None]
    row = (st["kv_len"] - (st["cu"][1:] - st["cu"][:-1]))[:, None, None] + torch.arange(Q, device="cuda")[None, :, None]
    seen = (col <= row) & (col < st["kv_len"][:, None, None])
    if c["window"]:
        seen = seen & (col > row - c["window"])
    out, lse = _softmax_product(_heads(q).reshape(n, KVH, -1, Q, hd), k, v, seen, st["sinks"], there)
    return dict(out=out.to(TYPES[c["act"]]), lse=lse)


# ───────────────────────── work of a pass ─────────────────────────

def _pairs(q, kv, window):
    """(query, key) pairs that one head computes, and the keys that any of them sees."""
    pairs = sum(min(p + 1, window) if window else p + 1 for p in range(kv - q, kv))
    return pairs, min(kv, window + q - 1) if window else kv


def work(case):
    k = case["kind"]
    if k == "plan":
        old, new = _plan_lengths(case)
        page = case["page"]
        moved = sum(abs(_pages(a, page) - _pages(b, page)) for a, b in zip(old, new))
        rows = sum(abs(a - b) for a, b in zip(old, new))
        most = 2 * rows + 8
        # per way: the lengths in, lengths and starts out, the pages from or to the ring and the table, all rows' slots and positions
        return dict(bytes=2 * (4 * case["n"] * 4 + moved * 8 + most * 8), flops=2 * (10 * case["n"] + 6 * most))
    H, KVH, hd = case["H"], case["KVH"], case["hd"]
    if k == "store":
        act, cache = SIZE[case["act"]], SIZE[case["cache"]]
        row = (2 * H + 2 * KVH) * hd * act + 2 * KVH * hd * cache + hd * 4 + 8
        return dict(bytes=case["T"] * row, flops=case["T"] * (H + KVH) * hd * 3)
    if k == "packed":
        lens, e = _lengths(case["n"], case["longest"], case["mix"]), SIZE[case["type"]]
        pairs = sum(_pairs(x, x, case["window"])[0] for x in lens)
        return dict(bytes=sum(lens) * ((2 * H + 2 * KVH) * hd * e + H * 4), flops=4 * H * hd * pairs)
    q, lens = _paged_lengths(case)
    seen = [_pairs(a, b, case["window"]) for a, b in zip(q, lens)]
    return dict(bytes=sum(s for _, s in seen) * 2 * KVH * hd * SIZE[case["cache"]]
                + sum(q) * H * (2 * hd * SIZE[case["act"]] + 4), flops=4 * H * hd * sum(p for p, _ in seen))


# ───────────────── the same in 64 bits, request by request ─────────────────

def _exact_rows(q, k, v, first, window, sinks):
    """Rows q [Q, H, hd] (fp64) at positions first.. over k, v [L, KVH, hd]."""
    Q, H, hd = q.shape
    G, out, lse = H // k.shape[1], torch.empty_like(q), torch.empty((Q, H), dtype=torch.float64, device=q.device)
    pos, key = torch.arange(first, first + Q, device=q.device)[:, None], torch.arange(k.shape[0], device=q.device)[None]
    hidden = key > pos
    if window:
        hidden = hidden | (key <= pos - window)
    for h in range(H):
        a = q[:, h] @ k[:, h // G].T / math.sqrt(hd)
        a = torch.cat([a.masked_fill(hidden, -math.inf), sinks[h].double().expand(Q, 1)], 1)
        lse[:, h] = torch.logsumexp(a, 1)
        out[:, h] = torch.exp(a - lse[:, h:h + 1])[:, :-1] @ v[:, h // G]
    return out, lse


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind == "plan":
        return None                                        # whole numbers only
    if kind == "store":
        q, k, v = (x.double() for x in _qkv(st))
        z = torch.complex(*(st["rope"][st["pos"].long()].double().unbind(2)))[:, None]
        half, n, out = case["hd"] // 2, case["T"], {}
        rot = lambda x: torch.view_as_real(torch.complex(x[..., :half], x[..., half:]) * z).transpose(2, 3).flatten(2)
        out["q_out"] = rot(q)
        out["q_out"][n:] = 0.0
        for name, rows in (("k_pages", rot(k)), ("v_pages", v)):
            flat = st[name].double().transpose(1, 2).reshape(-1, case["KVH"], case["hd"])
            flat[st["slot"][:n].long()] = rows[:n]
            out[name] = flat.reshape(case["pages"], case["page"], case["KVH"], case["hd"]).transpose(1, 2).contiguous()
        return out
    outs = []
    if kind == "packed":
        q, k, v = _qkv(st)
        a = 0
        for n in _lengths(case["n"], case["longest"], case["mix"]):
            outs.append(_exact_rows(q[a:a + n].double(), k[a:a + n].double(), v[a:a + n].double(), 0, case["window"],
                                    st["sinks"]))
            a += n
    else:
        a, page = 0, case["page"]
        for r, (n, length) in enumerate(zip(*_paged_lengths(case))):
            ids = st["table"][r, :_pages(length, page)].long()
            k, v = (st[x].index_select(0, ids).transpose(1, 2).flatten(0, 1)[:length].double() for x in ("k_pages", "v_pages"))
            outs.append(_exact_rows(st["q"][a:a + n].double(), k, v, length - n, case["window"], st["sinks"]))
            a += n
    return dict(out=torch.cat([o for o, _ in outs]), lse=torch.cat([s for _, s in outs]))
