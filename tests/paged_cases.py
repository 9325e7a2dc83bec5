"""Inputs and error bounds shared by the tests of the paged operators."""
import torch

from oracle import paged_model as M

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def half_step(dt):
    return torch.finfo(dt).eps / 2


def make(torch, new, held, hq=8, hk=2, d=128, block=16, layout="nhd", dtype="bf16", seed=0, spare=3,
         extra_rows=0, width=None, stale=float("nan"), qscale=1.0):
    """A ragged call: new[i] rows on top of held[i] tokens.  Places of the
    pages that no token was written to hold `stale`."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[dtype]
    n = len(new)
    lens = [a + b for a, b in zip(new, held)]
    W = width or max(1, max(-(-L // block) for L in lens))
    per = hk if layout == "slab" else 1
    need = [[-(-L // block)] * per for L in lens]
    count = sum(map(sum, need))
    pages = count + spare
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    table = torch.full((n, per, W), -1, dtype=torch.int32)
    shape = {"nhd": (pages, block, hk, d), "hnd": (pages, hk, block, d), "slab": (pages, block, d)}[layout]
    kp = torch.full(shape, stale, dtype=dt, device="cuda")
    vp = torch.full(shape, stale, dtype=dt, device="cuda")
    k = 0
    for i in range(n):
        for h in range(per):
            for b in range(need[i][h]):
                table[i, h, b] = order[k]
                toks = slice(0, min(block, lens[i] - b * block))
                ix = (order[k], slice(None), toks) if layout == "hnd" else (order[k], toks)
                for p in (kp, vp):
                    p[ix] = torch.randn(p[ix].shape, generator=g, device="cuda").to(dt)
                k += 1
    if layout != "slab":
        table = table[:, 0]
    T = sum(new) + extra_rows
    return dict(kp=kp, vp=vp, table=table.contiguous().cuda(), layout=layout, T=T, dt=dt,
                lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                starts=torch.tensor([sum(new[:i]) for i in range(n + 1)], dtype=torch.int32, device="cuda"),
                q=(torch.randn(T, hq, d, generator=g, device="cuda") * qscale).to(dt),
                k=torch.randn(T, hk, d, generator=g, device="cuda").to(dt),
                v=torch.randn(T, hk, d, generator=g, device="cuda").to(dt),
                max_new=max(new), d=d, gen=g)


def score_slack(top, d):
    """Largest relative error of a weight exp(s - lse): a score is a sum of d
    products in fp32, each partial sum off by 2^-23 (a tensor core may cut
    instead of round) of at most `top` = sum |q k|; the power of two and the
    fp32 bookkeeping around it add under 2^-19 more."""
    return torch.expm1(2 * (d + 4) * 2.0 ** -23 * top) + 2.0 ** -19


def check_attend(c, out, lse, scale, window=0, p_bits=None):
    """out and lse against the 64-bit form.  Bound of an output: half a step
    of its own rounding; the weights' rounding to the pages' type (half a step
    each of sum p |v|; the fp32 path rounds to fp32); their fp32 errors on
    numerator and denominator."""
    o, l, bulk, top = M.attend(c["kp"], c["vp"], c["layout"], c["table"], c["lens"], c["starts"], c["q"],
                               scale, window)
    n = int(c["starts"][-1])
    o, l, bulk, top = o[:n], l[:n], bulk[:n], top[:n]
    u = half_step(c["dt"])
    sl = score_slack(top, c["d"])[..., None]
    tol = u * o.abs() * 1.01 + bulk * (u * 1.01 + 2 * sl) + 1e-30
    if c["dt"] == torch.float16:
        tol = tol + 2.0 ** -25                   # half a step of a subnormal result
    err = (out[:n].double() - o).abs()
    assert not torch.isnan(out[:n]).any()
    assert (err <= tol).all(), float((err / tol).max())
    if lse is not None:
        empty = torch.isinf(l)
        assert torch.equal(torch.isinf(lse[:n]) & (lse[:n] < 0), empty)
        e = (lse[:n].double() - l).abs()[~empty]
        t = (score_slack(top, c["d"]) + 2.0 ** -22 * l.abs())[~empty]
        assert (e <= t).all(), float((e / t).max())
    return o, l


def check_mass(c, mass, lse, scale, window=0):
    """Every term is within score_slack of the exact one; the sum of a block
    of positive terms adds 2^-24 a term and level (under 2^-18)."""
    want = M.block_mass(c["kp"], c["layout"], c["table"], c["lens"], c["starts"], c["q"], lse, scale, window)
    n = int(c["starts"][-1])
    _, l, _, top = M.attend(c["kp"], c["kp"], c["layout"], c["table"], c["lens"], c["starts"], c["q"],
                            scale, window)
    worst = float(top[:n].max()) if n else 0.0
    # lse * log2(e) in fp32 is off by 2^-23 of it
    big = float(lse[:n][~torch.isinf(lse[:n])].abs().max()) if n and (~torch.isinf(lse[:n])).any() else 0.0
    rel = float(score_slack(torch.tensor(worst + 2 * big / (c["d"] + 4), dtype=torch.float64), c["d"])) + 2.0 ** -18
    assert not torch.isnan(mass).any()
    err = (mass.double() - want).abs()
    assert (err <= rel * want + 1e-30).all(), float((err / (want + 1e-30)).max())
    return want
