"""The paged-cache operators' argument checks, on the host side alone
(hip_host): what they refuse launches nothing, what they take launches."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest
import torch

from hip_host import run

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SETUP = """
h = engine(small(vocab=512, ctx_len=64), synthetic=False)
launches()
def A(v, by=0):
    return vp(v.value + by)
buf = dev(1 << 20)
def pages(**kw):
    p = pa.PkPages(A(buf), A(buf), pa.T_BF16, 64, 16, 2, 64)
    for k, v in kw.items(): setattr(p, k, v)
    return p
def plan(**kw):
    a = [A(buf, 4096 * i) for i in range(9)]
    p = pa.PkPagePlan(8, 4, 64, 16, 100, *a)
    for k, v in kw.items(): setattr(p, k, v)
    return p
def rows(pg=None, **kw):
    p = pa.PkKvRows(5, 4, pa.T_BF16, 64, A(buf), A(buf), A(buf), A(buf), 256, 128, 128, 256, A(buf), A(buf), A(buf), pg or pages())
    for k, v in kw.items(): setattr(p, k, v)
    return p
def packed(**kw):
    p = pa.PkAttnPacked(pa.T_F16, 4, 2, 64, 10, 2, 8, 0, 0.0, A(buf), A(buf), A(buf), A(buf), 256, 128, 128, 256, A(buf), None, None)
    for k, v in kw.items(): setattr(p, k, v)
    return p
def paged(pg=None, **kw):
    p = pa.PkAttnPaged(pa.T_BF16, 4, 10, 2, 8, 5, 0, 0, 0.0, A(buf), A(buf), 256, 256, A(buf), A(buf), A(buf), None, None, pg or pages())
    for k, v in kw.items(): setattr(p, k, v)
    return p
def takes(f, rec, n=None):
    assert f(h, C.byref(rec)) == 0, L.pk_last_error()
    got = len(launches())
    assert got >= 1 if n is None else got == n, got
def refuses(f, rec, code):
    rc = f(h, C.byref(rec))
    assert rc == code, (rc, code, L.pk_last_error())
    assert not launches() and L.pk_last_error()
f_plan, f_rows, f_packed, f_paged = L.pk_plan_pages, L.pk_store_pages, L.pk_attention_packed, L.pk_attention_paged
"""


def checked(code):
    run(SETUP + code)


def test_null_arguments():
    checked("""
for f, make in ((f_plan, plan), (f_rows, rows), (f_packed, packed), (f_paged, paged)):
    takes(f, make())
    assert f(None, C.byref(make())) == -1 and f(h, None) == -1
    for name, kind in make()._fields_:
        if kind is C.c_void_p and name not in ("rope_dev", "sinks_dev", "lse_dev"):
            refuses(f, make(**{name: None}), -1)
for pg in (pages(k_dev=None), pages(v_dev=None)):
    refuses(f_rows, rows(pg), -1)
    refuses(f_paged, paged(pg), -1)
takes(f_rows, rows(rope_dev=None, rope_len=0))
takes(f_rows, rows(n_heads=0, q_dev=None, q_out_dev=None))
assert not L.pk_engine_rope(None, None)
""")


def test_nothing_to_do():
    checked("""
takes(f_plan, plan(n_req=0, old_len_dev=None, new_len_dev=None, table_dev=None, len_dev=None))
takes(f_plan, plan(max_tokens=0, slot_dev=None, pos_dev=None))
takes(f_rows, rows(n_tokens=0), 0)
for kw in (dict(n_tokens=0), dict(n_seq=0), dict(max_len=0)):
    takes(f_packed, packed(**kw), 0)
for kw in (dict(n_tokens=0), dict(n_req=0), dict(max_q=0)):
    takes(f_paged, paged(**kw), 0)
""")


def test_shapes_and_types():
    checked("""
for kw, rc in ((dict(n_req=-1), -1), (dict(n_req=4097), -4), (dict(max_tokens=-1), -1), (dict(max_blocks=0), -1),
               (dict(n_pages=0), -1), (dict(page_size=0), -4), (dict(page_size=12), -4), (dict(page_size=512), -4),
               (dict(page_size=4), -4), (dict(n_pages=1 << 27), -1), (dict(max_blocks=1 << 27), -1)):
    refuses(f_plan, plan(**kw), rc)
takes(f_plan, plan(n_req=4096, n_pages=(1 << 27) - 1))
p = plan()
for name in ("old_len_dev", "new_len_dev"):                       # len_dev may not overlap the lengths that it follows from
    refuses(f_plan, plan(len_dev=getattr(p, name)), -1)
    refuses(f_plan, plan(len_dev=getattr(p, name) + 7 * 4), -1)
    takes(f_plan, plan(len_dev=getattr(p, name) + 8 * 4))
bad_pages = ((dict(type=3), -1), (dict(type=-1), -1), (dict(page_size=24), -4), (dict(page_size=512), -4), (dict(n_pages=0), -1),
             (dict(n_pages=1 << 27), -1), (dict(n_kv_heads=0), -1), (dict(head_dim=8), -4), (dict(head_dim=72), -4),
             (dict(head_dim=144), -4), (dict(k_dev=buf.value + 8), -1), (dict(v_dev=buf.value + 2), -1))
for kw, rc in bad_pages:
    refuses(f_rows, rows(pages(**kw)), rc)
    refuses(f_paged, paged(pages(**kw)), rc)
for act in range(3):
    for cache in range(3):
        ok = act in (0, cache)
        for f, make in ((f_rows, rows), (f_paged, paged)):
            (takes(f, make(pages(type=cache), type=act)) if ok else refuses(f, make(pages(type=cache), type=act), -4))
for kw in (dict(n_tokens=-1), dict(n_heads=-1), dict(rope_len=0), dict(rope_dev=buf.value + 8), dict(type=9),
           dict(q_stride=248), dict(q_stride=260), dict(k_stride=120), dict(k_dev=buf.value + 8), dict(q_out_stride=0)):
    refuses(f_rows, rows(**kw), -1)
both = (dict(n_tokens=-1), dict(window=-1), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
        dict(n_heads=0), dict(n_heads=5), dict(q_stride=255), dict(out_stride=128), dict(type=3), dict(q_dev=buf.value + 4))
for kw in both + (dict(n_seq=-1), dict(max_len=-1), dict(n_kv_heads=0), dict(n_kv_heads=3), dict(k_stride=64)):
    refuses(f_packed, packed(**kw), -1)
for kw in both + (dict(n_req=-1), dict(max_q=-1), dict(max_kv=-1), dict(max_blocks=0), dict(max_blocks=1 << 28)):
    refuses(f_paged, paged(**kw), -1)
big = 1 << 26
for kw in (dict(q_stride=big + 8), dict(out_stride=big + 8), dict(k_stride=big + 8), dict(v_stride=1 << 40)):
    refuses(f_packed, packed(**kw), -1)
takes(f_packed, packed(q_stride=big, k_stride=big, v_stride=big, out_stride=big))
refuses(f_paged, paged(q_stride=big + 8), -1)
refuses(f_rows, rows(v_stride=big + 8), -1)
refuses(f_paged, paged(max_blocks=(1 << 26) + 1), -1)             # 2^30 positions of 16
refuses(f_packed, packed(n_seq=(1 << 17) + 1), -4)
refuses(f_paged, paged(n_req=(1 << 17) + 1), -4)
takes(f_paged, paged(n_req=1 << 17))
refuses(f_packed, packed(n_tokens=(1 << 29) + 1), -4)             # two heads to a key head
refuses(f_paged, paged(n_tokens=(1 << 29) + 1), -4)
for f, make in ((f_packed, packed), (f_paged, paged)):
    takes(f, make(window=2 ** 31 - 1))
for hd in (8, 24, 100, 144, 256):
    refuses(f_packed, packed(head_dim=hd), -4)
refuses(f_packed, packed(n_heads=1026, q_stride=1 << 17, out_stride=1 << 17), -4)
""")


def test_every_layout_launches():
    """Head layouts, head sizes, lengths and bounds from one to large: every call
    is one that the device takes (grids within its limits)."""
    checked("""
for t in range(3):
    for H, KVH in ((1, 1), (64, 8), (12, 2), (40, 1), (1024, 1), (7, 7)):
        for hd in (16, 48, 64, 96, 128):
            for n, T, longest in ((1, 1, 1), (3, 200, 150), (4096, 70000, 70000), (70000, 1 << 20, 40000)):
                takes(f_packed, packed(type=t, n_heads=H, n_kv_heads=KVH, head_dim=hd, n_tokens=T, n_seq=n, max_len=longest,
                                       q_stride=H * hd, k_stride=KVH * hd, v_stride=KVH * hd, out_stride=H * hd))
                for max_q in (1, 2, 9, longest):
                    for kv in (0, 1, 5000):
                        takes(f_paged, paged(pages(type=t, n_kv_heads=KVH, head_dim=hd), type=t, n_heads=H, n_tokens=T, n_req=n,
                                             max_q=max_q, max_kv=kv, max_blocks=1 << 13, q_stride=H * hd, out_stride=H * hd))
""")


def test_workspaces_and_captures():
    """What a captured call addresses outlives the calls that need more; a capture
    whose call would need more is refused, not enlarged."""
    checked("""
def call(n, T, max_q, pg=None):
    return paged(pg, n_tokens=T, n_req=n, max_q=max_q, max_blocks=1 << 13)
takes(f_paged, call(1, 1, 1))
pa.check(L.pk_capture_begin(h))
pa.check(f_paged(h, C.byref(call(1, 1, 1))))
g = vp()
pa.check(L.pk_capture_end(h, C.byref(g)))
for n, T, max_q in ((2, 2, 1), (100, 100, 1), (2, 900, 600), (4000, 4000, 1), (300, 9000, 700)):
    takes(f_paged, call(n, T, max_q))
    pa.check(L.pk_graph_launch(h, g))
    assert hh.hh_stale() == 0
pa.check(L.pk_graph_destroy(g))
pa.check(L.pk_engine_destroy(h))
assert hh.hh_in_use() == 4 << 20, hh.hh_in_use()
""")


def test_records_check_their_tensors():
    """The Python records: shapes, types, strides and devices."""
    import picchio_amd as pa
    z = lambda *s, t=torch.bfloat16: torch.zeros(s, dtype=t)
    i = lambda n: torch.zeros(n, dtype=torch.int32)
    pg = pa.pages(z(4, 2, 16, 64), z(4, 2, 16, 64))
    assert (pg.type, pg.n_pages, pg.page_size, pg.n_kv_heads, pg.head_dim) == (pa.T_BF16, 4, 16, 2, 64)
    for k, v in ((z(4, 2, 16), z(4, 2, 16)), (z(4, 2, 16, 64), z(3, 2, 16, 64)), (z(4, 2, 16, 64), z(4, 2, 16, 64, t=torch.float16)),
                 (z(4, 16, 2, 64).transpose(1, 2), z(4, 16, 2, 64).transpose(1, 2)), (z(4, 2, 16, 64, t=torch.int32),) * 2):
        with pytest.raises(ValueError):
            pa.pages(k, v)
    x = z(5, (4 + 2 + 2) * 64)
    q, k, v = x[:, :256].unflatten(1, (4, 64)), x[:, 256:384].unflatten(1, (2, 64)), x[:, 384:].unflatten(1, (2, 64))
    r = pa.kv_rows(q, k, v, torch.zeros_like(q), i(5), i(5), pg, rope=z(9, 32, 2, t=torch.float32))
    assert (r.q_stride, r.k_stride, r.rope_len, r.n_heads, r.n_tokens) == (512, 512, 9, 4, 5)
    assert pa.kv_rows(None, k, v, None, i(5), i(5), pg, rope=(1234, 7)).rope_len == 7
    for bad in (dict(q=q.float()), dict(q=q[:4]), dict(k=q), dict(v=v.transpose(0, 1)), dict(pos=i(4)), dict(slot=i(5).long()),
                dict(rope=z(9, 32, 2)), dict(rope=z(9, 16, 2, t=torch.float32)), dict(q_out=z(5, 4, 128)[..., ::2])):
        with pytest.raises(ValueError):
            pa.kv_rows(**{**dict(q=q, k=k, v=v, q_out=torch.zeros_like(q), pos=i(5), slot=i(5), pages=pg), **bad})
    out = z(5, 4, 64)
    a = pa.attn_packed(q, k, v, out, i(3), 5)
    assert (a.n_seq, a.n_tokens, a.k_stride, a.out_stride) == (2, 5, 512, 256)
    for bad in (dict(k=k.half()), dict(out=out.float()), dict(cu=i(3).long()), dict(sinks=torch.zeros(3)),
                dict(lse=torch.zeros(5, 5)), dict(v=v[:4])):
        with pytest.raises(ValueError):
            pa.attn_packed(**{**dict(q=q, k=k, v=v, out=out, cu=i(3), max_len=5), **bad})
    b = pa.attn_paged(q, out, i(4), i(3), i(6).reshape(3, 2), pg, 3)
    assert (b.n_req, b.max_blocks, b.max_q) == (3, 2, 3)
    for bad in (dict(cu_q=i(3)), dict(table=i(6).reshape(2, 3)), dict(q=z(5, 4, 32)), dict(kv_len=i(3).long())):
        with pytest.raises(ValueError):
            pa.attn_paged(**{**dict(q=q, out=out, cu_q=i(4), kv_len=i(3), table=i(6).reshape(3, 2), pages=pg, max_q=3), **bad})
    p = pa.page_plan(i(3), i(3), i(6).reshape(3, 2), i(4), i(4), 16, i(3), i(4), i(9), i(9))
    assert (p.n_req, p.max_blocks, p.n_pages, p.max_tokens) == (3, 2, 4, 9)
    with pytest.raises(ValueError):
        pa.page_plan(i(3), i(3), i(6).reshape(3, 2), i(4), i(3), 16, i(3), i(4), i(9), i(9))


def test_record_layouts_match_the_header():
    import picchio_amd as pa
    names = {"pk_pages": pa.PkPages, "pk_page_plan": pa.PkPagePlan, "pk_kv_rows": pa.PkKvRows, "pk_attn_packed": pa.PkAttnPacked,
             "pk_attn_paged": pa.PkAttnPaged}
    lines = [f'printf("{n} {f} %zu\\n", offsetof({n}, {f}));' for n, c in names.items() for f, _ in c._fields_]
    lines += [f'printf("{n} size %zu\\n", sizeof({n}));' for n in names]
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "l.c"), os.path.join(d, "l")
        open(c, "w").write('#include <stdio.h>\n#include <stddef.h>\n#include "picchio_hip.h"\nint main(void) {' + "\n".join(lines) + "}")
        subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe])
        for line in subprocess.check_output([exe], text=True).splitlines():
            n, f, v = line.split()
            assert int(v) == (C.sizeof(names[n]) if f == "size" else getattr(names[n], f).offset), line
