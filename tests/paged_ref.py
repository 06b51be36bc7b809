"""The paged-cache operators in 64 bits, request by request, and how far the
fp32 arithmetic may be from them."""
import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def attend(q, k, v, first, window=0, sinks=None, seen=None, scale=None):
    """Rows q [Q, H, hd] at positions first.. over k, v [L, KVH, hd]; `seen` [L]
    leaves positions out. Returns out, lse and a dict of what the bounds need,
    all fp64: mass = sum_j p_j |v_j|, reach = max_j scale |q|.|k_j| per row."""
    Q, H, hd = q.shape
    if not len(k):                               # a position that no row sees
        k = v = torch.zeros((1, *k.shape[1:]), device=q.device)
        seen = torch.tensor([False], device=q.device)
    L, KVH, _ = k.shape
    q, k, v = q.double(), k.double(), v.double()
    scale = 1 / math.sqrt(hd) if scale is None else scale
    pos, key = torch.arange(first, first + Q, device=q.device)[:, None], torch.arange(L, device=q.device)[None]
    on = key <= pos
    if window:
        on = on & (key > pos - window)
    if seen is not None:
        on = on & seen[None]
    out, mass = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((Q, H), -math.inf, dtype=torch.float64, device=q.device)
    reach, n = torch.zeros_like(lse), on.sum(1)
    for h in range(H):
        g = h // (H // KVH)
        # (what no row sees may hold anything)
        kk, vv = (torch.where(on.any(0)[:, None], x[:, g], torch.zeros_like(x[:, g])) for x in (k, v))
        s = (q[:, h] @ kk.T * scale).masked_fill(~on, -math.inf)
        a = s if sinks is None else torch.cat([s, sinks[h].double().expand(Q, 1)], 1)
        lse[:, h] = torch.logsumexp(a, 1)
        p = torch.where(on, torch.exp(s - lse[:, h:h + 1]), torch.zeros_like(s))
        # 0 x infinity: a position that a row does not see adds nothing to it
        fine = torch.isfinite(vv).all(1)
        out[:, h] = p[:, fine] @ vv[fine]
        mass[:, h] = p[:, fine] @ vv[fine].abs()
        for j in torch.nonzero(~fine)[:, 0].tolist():
            rows = on[:, j]
            out[rows, h] += p[rows, j:j + 1] * vv[j]
        reach[:, h] = (q[:, h].abs() @ kk.abs().T * scale).masked_fill(~on, 0.0).nan_to_num(0.0).amax(1)
    return out, lse, dict(mass=mass, reach=reach, n=n.double())


def bounds(out, lse, need, dtype, hd):
    """(bound of out, bound of lse) elementwise. A score is off by at most (hd +
    4) half steps of fp32 of its largest possible sum; a probability by that twice
    (numerator and denominator), by the running maximum's roundings (as a sink or
    a score times log2 e, and in the difference: 3 half steps of a value that
    |lse| bounds where it is a sink, and |q|.|k| where it is a score: exp(x (1 +
    d)) = exp(x) (1 + x d)), and exp2's and the rescalings' few half steps per 64
    positions; a sum of n terms by n half steps; with a 16-bit type each
    probability by a half step of the type for its product with V; the result by a
    half step of its type."""
    u = 2.0 ** -24
    ds = (hd + 4) * u * need["reach"] + 3 * u * lse.abs().nan_to_num(posinf=0.0)
    rel = 2 * ds + u * (need["n"][:, None] + 16 + need["n"][:, None] / 16)
    if dtype != torch.float32:
        rel = rel + HALF_STEP[dtype]
    tiny = torch.finfo(dtype).tiny
    return (rel[..., None] * need["mass"] * (1 + HALF_STEP[dtype]) + HALF_STEP[dtype] * out.abs() + tiny,
            ds + u * (need["n"][:, None] + 16 + 2 * lse.abs().nan_to_num(posinf=0.0)))


def check(got, want, bound, what):
    got = got.double()
    both = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), (what, "NaN")
    rest = ~both & ~torch.isnan(want)
    assert torch.equal(got[rest], want[rest]), (what, "infinities")
    off = (got - want).abs()[both]
    if off.numel():
        worst = (off / bound[both].clamp(min=1e-300)).max().item()
        assert worst <= 1.0, f"{what}: off by {worst:.3g} times the bound"


def rotate(x, pos, rope):
    """x [T, heads, hd] turned by rope [positions, hd / 2, 2] in fp64."""
    c, s = rope[pos.long()].double().unbind(2)
    c, s = c[:, None], s[:, None]
    a, b = x.double().chunk(2, 2)
    return torch.cat([a * c - b * s, a * s + b * c], 2)


def plan(old, new, table, ring, state, page, max_tokens):
    """pk_plan_pages on Python lists: returns (len, cu, slot, pos), changes table,
    ring and state."""
    cap, n_pages = len(table[0]) * page if table else 0, len(ring)
    head, count = state[0], state[1]
    free = [ring[(head + i) % n_pages] for i in range(count)]
    given, lens, cu, slot, pos, taken, rows, shut = [], [], [0], [], [], 0, 0, False
    for r, (a, b) in enumerate(zip(old, new)):
        a, b = min(max(a, 0), cap), min(max(b, 0), cap)
        ob, nb = -(-a // page), -(-b // page)
        if b > a:
            shut = shut or taken + nb - ob > count or rows + b - a > max_tokens
            if shut:
                b = a
            else:
                table[r][ob:nb] = free[taken:taken + nb - ob]
                taken += nb - ob
                rows += b - a
        else:
            given += table[r][nb:ob]
            table[r][nb:ob] = [-1] * (ob - nb)
        lens.append(b)
        for p in range(a, b):
            g = table[r][p // page]
            pos.append(p)
            slot.append(g * page + p % page if 0 <= g < n_pages else -1)
        cu.append(rows)
    for i, g in enumerate(given):
        ring[(head + count + i) % n_pages] = g
    state[0], state[1] = (head + taken) % n_pages, count - taken + len(given)
    return lens, cu, slot + [-1] * (max_tokens - rows), pos + [0] * (max_tokens - rows)
