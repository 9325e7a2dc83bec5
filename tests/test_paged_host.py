"""The paged operators' refusals and host side, without a GPU: the C entries
check their arguments before anything is launched, and the rotation's
frequencies are computed on the host."""
import ctypes as C
import math

import pytest
import torch

import orchkv_b200 as okv
from orchkv_b200 import _lib, paged

INVALID = okv.ERR["INVALID"]
A = 1 << 20                                       # any aligned address: never read


def call(**kw):
    """A valid call's arguments, by name, with some replaced."""
    v = dict(k=A, v=A, page_stride=16 * 4 * 128, head_stride=128, token_stride=4 * 128, n_pages=9,
             page_tokens=16, n_kv_heads=4, d_head=128, dtype=1, table=A, width=4096, n=2, lens=A, starts=A,
             rows=6, hq=8, q=A, out=2 * A, row_stride=8 * 128, q_head=128, kr=A, vr=A, rot=128, turns=A,
             ws=A, short=0)
    assert set(kw) <= set(v)
    v.update(kw)
    L = okv.lib()
    pg = _lib.Pages(v["k"], v["v"], v["page_stride"], v["head_stride"], v["token_stride"], v["n_pages"],
                    v["page_tokens"], v["n_kv_heads"], v["d_head"], v["dtype"])
    b = _lib.Batch(v["table"], v["width"], 0, v["width"], v["n"], v["lens"], v["starts"], v["rows"], v["rows"])
    q = _lib.Rows(v["q"], v["row_stride"], v["q_head"])
    o = _lib.Rows(v["out"], v["row_stride"], v["q_head"])
    kr, vr = (_lib.Rows(v[x], 4 * 128, 128) for x in ("kr", "vr"))
    ap = _lib.AppendArgs(q, o, kr, vr, v["hq"], v["rot"], 0, 1.0, v["turns"], 0, 0, 0, 0, 1e-6)
    at = _lib.AttendArgs(q, o, 0, v["hq"], 1.0, 0)
    ms = _lib.MassArgs(q, A, v["out"], v["hq"], 1.0, 0)
    need = L.orchkv_paged_attend_workspace(C.byref(pg), C.byref(b), C.byref(at))
    return need, dict(
        append=lambda: L.orchkv_paged_append(C.byref(pg), C.byref(b), C.byref(ap), None),
        attend=lambda: L.orchkv_paged_attend(C.byref(pg), C.byref(b), C.byref(at), v["ws"],
                                             max(0, need - v["short"]), None),
        mass=lambda: L.orchkv_paged_block_mass(C.byref(pg), C.byref(b), C.byref(ms), v["ws"], 1 << 30, None))


EVERY = ("append", "attend", "mass")


@pytest.mark.parametrize("bad,ops", [
    (dict(k=0), EVERY), (dict(k=A + 8), EVERY), (dict(v=0), ("append", "attend")),
    (dict(page_stride=16 * 4 * 128 + 4), EVERY), (dict(head_stride=132), EVERY),
    (dict(token_stride=4 * 128 + 1), EVERY), (dict(n_pages=0), EVERY), (dict(n_pages=1 << 31), EVERY),
    (dict(page_tokens=0), EVERY), (dict(n_kv_heads=0), EVERY), (dict(d_head=0), EVERY),
    (dict(d_head=100), EVERY), (dict(d_head=264), EVERY), (dict(dtype=3), EVERY), (dict(dtype=-1), EVERY),
    (dict(table=0), EVERY), (dict(width=0), EVERY), (dict(width=1 << 27), EVERY), (dict(lens=0), EVERY),
    (dict(starts=0), EVERY), (dict(rows=1 << 31), EVERY), (dict(hq=9), ("attend", "mass")),
    (dict(hq=0), ("attend", "mass")), (dict(q=0), EVERY), (dict(q=A + 2), EVERY), (dict(out=0), EVERY),
    (dict(row_stride=8 * 128 + 1), EVERY), (dict(q_head=129), EVERY), (dict(kr=0), ("append",)),
    (dict(vr=A + 8), ("append",)), (dict(rot=127), ("append",)), (dict(rot=130), ("append",)),
    (dict(page_stride=-16 * 4 * 128), EVERY), (dict(token_stride=-128), EVERY), (dict(row_stride=-1024), EVERY),
    (dict(out=A), ("attend",)),
    (dict(turns=0), ("append",)), (dict(ws=0), ("attend",)), (dict(ws=A + 16), ("attend",)),
    (dict(short=1), ("attend",)),
])
def test_refusals(bad, ops):
    _, fn = call(**bad)
    for op in ops:
        assert fn[op]() == INVALID, op


def test_nothing_to_do():
    for kw in (dict(n=0, table=0, lens=0, starts=0), dict(rows=0, q=0)):
        need, fn = call(**kw)
        assert need == 0
        assert fn["append"]() == 0 and fn["attend"]() == 0
    assert call(n=0, table=0, lens=0, starts=0)[1]["mass"]() == 0
    assert call()[0] > 0
    assert call(width=4, rows=2)[0] == 0          # short: no workspace
    assert call(d_head=100)[0] == 0


def pages(shape=(4, 16, 2, 64), dtype=torch.float16, **kw):
    x = torch.zeros(shape, dtype=dtype, **kw)
    return x, x.clone()


@pytest.mark.parametrize("make,layout,msg", [
    (lambda: pages(), "tokens", "layout"),
    (lambda: pages(dtype=torch.float64), "nhd", "not supported"),
    (lambda: (pages()[0], pages((4, 16, 2, 32))[0]), "nhd", "alike"),
    (lambda: (pages()[0], pages()[0].float()), "nhd", "alike"),
    (lambda: pages(), "slab", "3 dimensions"),
    (lambda: pages((4, 16, 64)), "hnd", "4 dimensions"),
    (lambda: pages((4, 16, 2, 100)), "nhd", "16 bytes"),
    (lambda: pages((2, 16, 2, 264)), "nhd", "256"),
    (lambda: pages((0, 16, 2, 64)), "nhd", "empty"),
    (lambda: tuple(x.transpose(2, 3) for x in pages((4, 16, 64, 64))), "nhd", "side by side"),
    (lambda: tuple(x[..., 1:65] for x in pages((4, 16, 2, 72))), "nhd", "16 bytes"),
    (lambda: tuple(x[..., :64] for x in pages((4, 16, 2, 65))), "nhd", "16 bytes"),
    (lambda: pages(), "nhd", "CUDA"),
])
def test_pages_refused(make, layout, msg):
    k, v = make()
    with pytest.raises(ValueError, match=msg):
        paged.PagedKV(k, v, layout)


def test_frequencies():
    d, base = 64, 10000.0
    plain, one = paged.Rotary.frequencies(d, base)
    assert one == 1.0 and plain.dtype == torch.float64
    assert all(abs(float(f) - base ** (-2 * i / d)) < 1e-15 for i, f in enumerate(plain))
    lin, one = paged.Rotary.frequencies(d, base, {"type": "linear", "factor": 4})
    assert one == 1.0 and torch.allclose(lin, plain / 4, rtol=1e-15)
    ntk, _ = paged.Rotary.frequencies(d, base, {"type": "ntk", "factor": 4})
    assert float(ntk[0]) == 1.0 and math.isclose(float(ntk[-1]), float(plain[-1]) / 4, rel_tol=1e-12)
    n = 4096
    yarn, mul = paged.Rotary.frequencies(d, base, {"type": "yarn", "factor": 16, "original": n})
    assert math.isclose(mul, 0.1 * math.log(16) + 1)
    ratio = yarn / plain
    turns = n * plain / (2 * math.pi)
    assert (ratio[turns > 40] == 1).all() and torch.allclose(ratio[turns < 0.7], torch.tensor(1 / 16, dtype=torch.float64))
    assert (ratio[1:] <= ratio[:-1] + 1e-15).all()
    band, _ = paged.Rotary.frequencies(d, base, {"type": "banded", "factor": 8, "original": n})
    ratio = band / plain
    assert (ratio[turns >= 4] == 1).all() and torch.allclose(ratio[turns <= 1], torch.tensor(1 / 8, dtype=torch.float64))
    mid = (turns > 1) & (turns < 4)
    assert torch.allclose(ratio[mid], 1 / 8 + (1 - 1 / 8) * (turns[mid] - 1) / 3)
    same, mul = paged.Rotary.frequencies(d, base, {"type": "yarn", "factor": 1, "original": n})
    assert mul == 1.0 and torch.allclose(same, plain)


@pytest.mark.parametrize("kw,msg", [
    (dict(rotary_dim=63), "even"), (dict(rotary_dim=0), "positive"), (dict(rotary_dim=66), "of a head"),
    (dict(scaling={"type": "cubic", "factor": 2}), "unknown"),
    (dict(scaling={"type": "linear", "factor": 0.5}), "below 1"),
    (dict(scaling={"type": "banded", "factor": 2, "original": 99, "low": 4, "high": 4}), "high above low"),
    (dict(rotary_dim=2, scaling={"type": "ntk", "factor": 2}), "4 or more"),
    (dict(inv_freq=torch.ones(3, 3)), "one dimension"), (dict(inv_freq=torch.ones(40)), "of a head"),
    (dict(inv_freq=torch.ones(8), rotary_dim=8), "rotate 16"),
    (dict(inv_freq=torch.ones(8), scaling={"type": "linear", "factor": 2}), "as it is"),
])
def test_rotary_refused(kw, msg):
    with pytest.raises(ValueError, match=msg):
        paged.Rotary(64, device="cpu", **kw)


def test_rotary_keeps_what_it_is_given():
    r = paged.Rotary(64, 32, interleaved=True, device="cpu")
    assert r.rotary_dim == 32 and r.interleaved and r.scale == 1.0 and r.turns.dtype == torch.float64
    assert math.isclose(float(r.turns[0]), 1 / (2 * math.pi))
    y = paged.Rotary(64, device="cpu", scaling={"type": "yarn", "factor": 4, "original": 64, "attention": 0.7})
    assert y.scale == 0.7
