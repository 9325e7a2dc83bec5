"""The paged operators where lengths, values and memory are unusual: lengths
past the table, infinities and NaN, faint weights, gradients, overlapping
tensors.  Bounds are those of tests/paged_cases.py."""
import math

import pytest

from oracle import paged_model as M
from tests import paged_cases as P

pytestmark = pytest.mark.gpu


def kv(c):
    from orchkv_b200 import paged
    return paged.PagedKV(c["kp"], c["vp"], c["layout"])


def call(c):
    return c["table"], c["lens"], c["starts"]


# ---- lengths that the table does not cover -----------------------------------------

def past_the_table(torch, new, lens, tokens, **kw):
    """Sequences of new[i] rows and lens[i] tokens over tables of `tokens`, of
    which the first min(lens[i], tokens) lie in pages."""
    there = [min(n, tokens) for n in lens]
    c = P.make(torch, [0] * len(new), there, width=tokens // kw.get("block", 16), **kw)
    c["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    c["starts"] = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    hq, d = c["q"].shape[1:]
    c["q"] = torch.randn(sum(new), hq, d, generator=c["gen"], device="cuda").to(c["dt"])
    return c


@pytest.mark.parametrize("new,lens,tokens,hq,hk", [
    ([2048], [3000], 960, 32, 8), ([2048], [9000], 960, 32, 8), ([3000], [900], 960, 8, 1),
    ([1500, 70], [2500, 4000], 960, 16, 4), ([1200, 900], [1000, 5000], 960, 8, 1), ([2000], [5000], 4000, 8, 2),
    ([1, 1, 1], [500, 2000, 9000], 960, 8, 2), ([5, 3], [2, 3000], 960, 8, 2),
])
@pytest.mark.parametrize("window", [0, 700])
def test_lengths_past_the_table_or_below_the_rows(cuda, new, lens, tokens, hq, hk, window):
    """Every row is written: tokens past the table hold nothing, and rows
    before a sequence's first token attend to nothing."""
    torch = cuda
    d = 64
    c = past_the_table(torch, new, lens, tokens, hq=hq, hk=hk, d=d, seed=sum(new))
    out = torch.full_like(c["q"], 7.0)
    got, lse = kv(c).attend(c["q"], *call(c), window=window, return_lse=True, out=out)
    assert got is out
    P.check_attend(c, out, lse, d ** -0.5, window)
    mass = torch.full((len(new), hk, tokens // 16), 7.0, device="cuda")
    kv(c).block_mass(c["q"], lse, *call(c), window=window, out=mass)
    P.check_mass(c, mass, lse, d ** -0.5, window)


# ---- faint weights --------------------------------------------------------------------

@pytest.mark.parametrize("new,held,block", [([1], 32000, 16), ([40], 32000, 16), ([600], 32000, 16),
                                            ([40], 32000, 24), ([1] * 48, 6000, 16)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("where", ["first", "last"])
def test_one_large_weight_among_many_faint_ones(cuda, new, held, block, d, dtype, where):
    """One key of weight 1 whose value is 0, and thousands of weight e^-17 =
    2^-24.5: the result is theirs alone, so each must be held to half a step
    of the pages' type."""
    torch = cuda
    c = P.make(torch, new, [held] * len(new), hq=8, hk=2, d=d, block=block, dtype=dtype, stale=0.0)
    c["kp"].zero_()
    c["q"].zero_()
    c["q"][:, :, 0] = 4.0
    at = 0 if where == "first" else held - 1
    page = c["table"][:, at // block].long()
    c["kp"][page, at % block, :, 0] = 4.25
    c["vp"].copy_(1 + 0.25 * torch.rand(c["vp"].shape, generator=c["gen"], device="cuda"))
    c["vp"][page, at % block] = 0
    out, lse = kv(c).attend(c["q"], *call(c), scale=1.0, return_lse=True)
    P.check_attend(c, out, lse, 1.0)


@pytest.mark.parametrize("new", [1, 40, 600])
@pytest.mark.parametrize("rise", [0.5, 2.0, 3.5, 6.0])
def test_scores_that_rise_along_the_keys(cuda, new, rise):
    """Scores that grow by `rise` nats every 128 keys: the reference that
    weights are taken against lags behind or is moved, and fp16 holds both."""
    torch = cuda
    c = P.make(torch, [new], [2000], hq=8, hk=2, d=64, dtype="fp16", stale=0.0)
    c["q"].zero_()
    c["q"][:, :, 0] = 1.0
    tok = torch.arange(2000 + new, device="cuda")
    row = c["table"][0, tok // 16].long()
    c["kp"].mul_(0.25)
    c["kp"][row, tok % 16, :, 0] = (rise * (tok // 128)).to(c["dt"])[:, None]
    out, lse = kv(c).attend(c["q"], *call(c), scale=1.0, return_lse=True)
    assert torch.isfinite(out).all()
    P.check_attend(c, out, lse, 1.0)


# ---- masses of values that are not finite --------------------------------------------

@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("fp16", 64)])
@pytest.mark.parametrize("of", ["q", "lse"])
def test_a_nan_row_reaches_every_block_it_attends_to(cuda, dtype, d, of):
    """A NaN query or lse in every place of a tile of 128 rows: all blocks
    that the row attends to, and those of its KV head alone."""
    torch = cuda
    c = P.make(torch, [64], [512], hq=8, hk=2, d=d, dtype=dtype)
    _, lse = kv(c).attend(c["q"], *call(c), return_lse=True)
    clean = kv(c).block_mass(c["q"], lse, *call(c))
    P.check_mass(c, clean, lse, d ** -0.5)
    for col in range(128):
        row, g = col // 4 + 32 * (col & 1), col % 4
        h = col // 64
        q, l = c["q"].clone(), lse.clone()
        if of == "q":
            q[row, h * 4 + g, col % d] = math.nan
        else:
            l[row, h * 4 + g] = math.nan
        mass = kv(c).block_mass(q, l, *call(c))
        blocks = (512 + row) // 16 + 1
        assert torch.isnan(mass[0, h, :blocks]).all(), col
        assert torch.equal(mass[0, h, blocks:], clean[0, h, blocks:]), col
        assert torch.equal(mass[0, 1 - h], clean[0, 1 - h]), col


@pytest.mark.parametrize("new", [1, 20, 64])
def test_masses_under_another_lse(cuda, new):
    """An lse that is not the row's own: the weights go by the formula, up to
    infinity and down to 0."""
    torch = cuda
    c = P.make(torch, [new], [512], hq=8, hk=2)
    _, lse = kv(c).attend(c["q"], *call(c), return_lse=True)
    for off in (-50.0, 30.0):
        mass = kv(c).block_mass(c["q"], lse + off, *call(c))
        P.check_mass(c, mass, lse + off, 128 ** -0.5)
    there = (512 + new + 15) // 16
    mass = kv(c).block_mass(c["q"], lse - 200, *call(c))
    assert (mass[:, :, :there] == math.inf).all() and (mass[:, :, there:] == 0).all()
    mass = kv(c).block_mass(c["q"], lse + 200, *call(c))
    assert (mass >= 0).all() and (mass < 1e-30).all()
    # one row's lse too small, in every place of a tile of 128 rows
    if new < 64:
        return
    for col in range(128):
        row, h = col // 4, col % 4
        l = lse.clone()
        l[row, h] -= 200
        mass = kv(c).block_mass(c["q"], l, *call(c))
        seen = (512 + row) // 16 + 1
        assert (mass[0, 0, :seen] == math.inf).all(), col
        assert torch.isfinite(mass[0, 1]).all() and (mass >= 0).all(), col


# ---- append: elements that do not turn -------------------------------------------------

@pytest.mark.parametrize("d,rot,inter", [(128, 0, False), (64, 32, False), (128, 64, True), (72, 20, False),
                                         (256, 2, True), (40, 6, True), (128, 112, False), (64, 64, False)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("normed", [False, True])
def test_append_elements_that_do_not_turn(cuda, d, rot, inter, dtype, normed):
    """An infinite or NaN element that is not rotated stays where it is and
    reaches no other; without a norm, such elements keep their very bits."""
    torch = cuda
    from orchkv_b200 import paged
    c = P.make(torch, [9, 20], [0, 30], hq=6, hk=3, d=d, dtype=dtype, stale=3.0, seed=d + rot)
    tail = torch.arange(rot, d, device="cuda")
    for x in (c["q"], c["k"]):
        for r in range(x.shape[0]):
            for h in range(x.shape[1]):
                if len(tail):
                    at = tail[(7 * r + 3 * h) % len(tail)]
                    x[r, h, at] = (math.inf, -math.inf, math.nan, -0.0)[(r + h) % 4]
    w = torch.rand(d, generator=c["gen"], device="cuda").add(0.5).to(c["dt"]) if normed else None
    freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / max(rot, 1)) if rot else None
    ro = paged.Rotary(d, inv_freq=freq, interleaved=inter, scale=1.25) if rot else None
    want = M.append(c["kp"], c["vp"], c["layout"], *call(c), c["k"], c["v"], c["q"], freq, inter, 1.25, None, w, w)
    got = kv(c).append(c["k"], c["v"], *call(c), q=c["q"], rotary=ro, q_norm=w, k_norm=w)
    u = P.half_step(c["dt"])
    for a, b in ((got, want[2]), (c["kp"], want[0])):
        fin = torch.isfinite(b)
        assert torch.equal(torch.isnan(a), torch.isnan(b))
        assert torch.equal(a[torch.isinf(b)].double(), b[torch.isinf(b)])
        amax = torch.where(fin, b, torch.zeros_like(b)).abs().amax(-1, keepdim=True)
        tol = u * 1.01 * b.abs() + (d + 16) * 2.0 ** -24 * 1.25 * math.sqrt(2) * amax + 2.0 ** -25
        assert ((a.double() - b).abs() <= tol)[fin].all()
    if not normed:
        same, x = got[..., rot:], c["q"][..., rot:]
        ok = ~torch.isnan(x)
        assert torch.equal(same[ok], x[ok]) and torch.equal(torch.signbit(same[ok]), torch.signbit(x[ok]))


@pytest.mark.parametrize("hq,hk", [(7, 1), (28, 4), (40, 1), (4, 4), (16, 1)])
@pytest.mark.parametrize("new,block", [(1, 16), (1, 7), (5, 16), (70, 16), (300, 64)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_keys_of_no_weight(cuda, hq, hk, new, block, dtype):
    """Keys whose score is minus infinity for every row weigh nothing, also
    where a tile has places that hold no row."""
    torch = cuda
    d = 64
    c = P.make(torch, [new], [500], hq=hq, hk=hk, d=d, block=block, dtype=dtype)
    c["q"][:, :, 0] = c["q"][:, :, 0].abs() + 0.125
    tok = torch.tensor([0, 3, 100, 101, 255, 256, 499], device="cuda")
    c["kp"][c["table"][0, tok // block].long(), tok % block, :, 0] = -math.inf
    out, lse = kv(c).attend(c["q"], *call(c), return_lse=True)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    mass = kv(c).block_mass(c["q"], lse, *call(c))
    want = M.block_mass(c["kp"], c["layout"], *call(c), c["q"], lse, d ** -0.5)
    # the bound of check_mass, its largest score taken over the other keys
    kp = c["kp"].clone()
    kp[torch.isinf(kp)] = 0
    _, _, _, top = M.attend(kp, kp, c["layout"], *call(c), c["q"], d ** -0.5)
    big = float(lse.abs().max())
    rel = float(P.score_slack(torch.tensor(float(top.max()) + 2 * big / (d + 4), dtype=torch.float64), d)) + 2.0 ** -18
    assert ((mass.double() - want).abs() <= rel * want + 1e-30).all()


# ---- gradients ----------------------------------------------------------------------------

def test_gradients_are_refused_and_never_dropped(cuda):
    torch = cuda
    from orchkv_b200 import paged
    c = P.make(torch, [2, 1], [5, 30], hq=4, hk=2)
    x, a, d = kv(c), call(c), 128
    w = torch.ones(d, dtype=c["dt"], device="cuda")
    leaf = w.clone().requires_grad_()
    freq = torch.ones(d // 2, device="cuda").requires_grad_()
    lse = torch.zeros(3, 4, device="cuda")
    grad_lse = lse.clone().requires_grad_()
    learned = paged.Rotary(d, inv_freq=freq)
    hot = paged.PagedKV(c["kp"].float().requires_grad_().to(c["dt"]), c["vp"])
    calls = [
        lambda **k: x.append(c["k"], c["v"], *a, q=c["q"], q_norm=leaf),
        lambda **k: x.append(c["k"], c["v"], *a, k_norm=leaf),
        lambda **k: x.append(c["k"], c["v"], *a, rotary=learned),
        lambda **k: x.block_mass(c["q"], grad_lse, *a),
        lambda **k: hot.append(c["k"], c["v"], *a),
        lambda **k: hot.attend(c["q"], *a),
        lambda **k: hot.block_mass(c["q"], lse, *a),
    ]
    for i, fn in enumerate(calls):
        with pytest.raises(ValueError, match="gradient"):
            fn()
        with torch.no_grad():
            fn()


def test_forward_gradients_are_refused(cuda):
    torch = cuda
    import torch.autograd.forward_ad as fwd
    c = P.make(torch, [2, 1], [5, 30], hq=4, hk=2)
    x, a = kv(c), call(c)
    w = torch.ones(128, dtype=c["dt"], device="cuda")
    lse = torch.zeros(3, 4, device="cuda")
    with fwd.dual_level():
        def dual(t):
            return fwd.make_dual(t, torch.ones_like(t))
        for fn in (lambda: x.attend(dual(c["q"]), *a), lambda: x.append(dual(c["k"]), c["v"], *a),
                   lambda: x.append(c["k"], c["v"], *a, k_norm=dual(w)),
                   lambda: x.block_mass(c["q"], dual(lse), *a)):
            with pytest.raises(ValueError, match="gradient"):
                fn()


def test_a_tensor_saved_for_a_backward_pass_and_overwritten_is_noticed(cuda):
    torch = cuda
    c = P.make(torch, [2, 1], [5, 30], hq=4, hk=2, dtype="fp32")
    x, a = kv(c), call(c)
    leaf = torch.ones((), device="cuda", requires_grad=True)
    lse = torch.zeros(3, 4, device="cuda")

    def written(t, fn):
        """fn writes into t, which the product has saved."""
        y = (leaf * t).sum()
        fn()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()

    q = c["q"].clone()
    written(q, lambda: x.append(c["k"], c["v"], *a, q=q, q_out=q))
    written(c["kp"], lambda: x.append(c["k"], c["v"], *a))
    written(c["vp"], lambda: x.append(c["k"], c["v"], *a))
    out = torch.empty_like(c["q"])
    written(out, lambda: x.attend(c["q"], *a, out=out))
    mass = torch.empty(2, 2, c["table"].shape[1], device="cuda")
    written(mass, lambda: x.block_mass(c["q"], lse, *a, out=mass))


def test_inference_tensors(cuda):
    torch = cuda
    with torch.inference_mode():
        c = P.make(torch, [2, 1], [5, 30], hq=4, hk=2)
        q = kv(c).append(c["k"], c["v"], *call(c), q=c["q"], q_out=c["q"])
        out, lse = kv(c).attend(q, *call(c), return_lse=True, out=torch.empty_like(q))
    P.check_attend(c, out, lse, 128 ** -0.5)
    kv(c).append(c["k"], c["v"], *call(c), q=c["q"], q_out=c["q"])   # and outside of it


# ---- tensors that share memory ---------------------------------------------------------

def test_overlapping_tensors_are_refused(cuda):
    torch = cuda
    c = P.make(torch, [3, 1], [5, 30], hq=4, hk=2)
    x, a, d = kv(c), call(c), 128
    buf = torch.zeros(40, d, dtype=c["dt"], device="cuda")
    q = buf[:16].view(4, 4, d)
    later, one = buf[4:20].view(4, 4, d), buf[:4].view(1, 4, d).expand(4, 4, d)
    flat = buf[:4].view(4, 1, d).expand(4, 4, d)
    for out in (later, buf[15:31].view(4, 4, d), q):
        with pytest.raises(ValueError, match="overlap"):
            x.attend(q, *a, out=out)
    for out in (later, one, flat):
        with pytest.raises(ValueError, match="overlap"):
            x.append(c["k"], c["v"], *a, q=q, q_out=out)
    for out in (one, flat):
        with pytest.raises(ValueError, match="overlap"):
            x.attend(c["q"], *a, out=out)
    k = buf[8:16].view(4, 2, d)
    with pytest.raises(ValueError, match="k and v"):
        x.append(k, c["v"], *a, q=c["q"], q_out=buf[:16].view(4, 4, d))
    with pytest.raises(ValueError, match="k and v"):
        x.append(c["k"], k, *a, q=c["q"], q_out=buf[:16].view(4, 4, d))
    # a broadcast input is an ordinary one
    P.check_attend(dict(c, q=one), *x.attend(one, *a, return_lse=True), d ** -0.5)


@pytest.mark.parametrize("how", ["rows", "heads", "columns", "in place"])
def test_interleaved_tensors_are_taken(cuda, how):
    """q and the results in one buffer, but in places of their own."""
    torch = cuda
    from orchkv_b200 import paged
    c = P.make(torch, [3, 40], [5, 30], hq=4, hk=2)
    T, d = 43, 128
    if how == "rows":
        buf = torch.zeros(2 * T, 4, d, dtype=c["dt"], device="cuda")
        q, out = buf[0::2], buf[1::2]
    elif how == "heads":
        buf = torch.zeros(T, 4, 2, d, dtype=c["dt"], device="cuda")
        q, out = buf[:, :, 0], buf[:, :, 1]
    else:
        buf = torch.zeros(T, 12, d, dtype=c["dt"], device="cuda")
        q, out = buf[:, :4], buf[:, 4:8]
        if how == "in place":
            c["k"], c["v"] = buf[:, 8:10].copy_(c["k"]), buf[:, 10:].copy_(c["v"])
    q.copy_(c["q"])
    ro = paged.Rotary(d)
    want = kv(c).append(c["k"], c["v"], *call(c), q=c["q"], rotary=ro)
    if how == "in place":
        assert kv(c).append(c["k"], c["v"], *call(c), q=q, rotary=ro, q_out=q) is q
        assert torch.equal(q, want)
    else:
        assert kv(c).append(c["k"], c["v"], *call(c), q=q, rotary=ro, q_out=out) is out
        assert torch.equal(out, want) and torch.equal(q, c["q"])
    got = kv(c).attend(q, *call(c), out=out)
    assert torch.equal(got, kv(c).attend(q.contiguous(), *call(c)))


# ---- units of one half behind a unit of two ------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_infinite_values_before_many_short_sequences(cuda, dtype, bad):
    """Long sequences with a value that is not finite on their diagonal, each
    before dozens of short ones that need half a tile only: the rows that
    attend to it are not finite, all others are as without it."""
    torch = cuda
    new = ([300] + [40] * 60) * 6
    held = [30] * len(new)
    c = P.make(torch, new, held, hq=8, hk=8, dtype=dtype, seed=3)
    want, wl = kv(c).attend(c["q"], *call(c), return_lse=True)
    at = 30 + 200
    for i in range(0, len(new), 61):
        page = int(c["table"][i, at // 16])
        c["vp"][page, at % 16, :, 5:8] = bad
    for _ in range(5):
        out, lse = kv(c).attend(c["q"], *call(c), return_lse=True)
        assert torch.equal(lse, wl)
        hit = torch.zeros_like(out, dtype=torch.bool)
        for i in range(0, len(new), 61):
            r = int(c["starts"][i])
            hit[r + 200:r + 300, :, 5:8] = True
        assert not torch.isfinite(out[hit]).any()
        assert torch.equal(out[~hit], want[~hit])


def test_broadcast_pages_are_read_and_not_written(cuda):
    """K and V shared by all heads: attended over like any, refused for an
    append, whose heads would write one place; masses over their inputs."""
    torch = cuda
    c = P.make(torch, [2, 40], [90, 30], hq=4, hk=1)
    shared = dict(c, kp=c["kp"].expand(-1, -1, 4, -1), vp=c["vp"].expand(-1, -1, 4, -1))
    out, lse = kv(shared).attend(c["q"], *call(c), return_lse=True)
    P.check_attend(shared, out, lse, 128 ** -0.5)
    k4 = c["k"].expand(-1, 4, -1).contiguous()
    with pytest.raises(ValueError, match="broadcast"):
        kv(shared).append(k4, k4, *call(c))
    with pytest.raises(ValueError, match="overlap"):
        kv(c).block_mass(c["q"], lse, *call(c), out=lse.flatten()[:2 * c["table"].shape[1]].view(2, 1, -1))
