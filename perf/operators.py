"""Cases that time the operators over the paged KV cache: the append with the
norms and the rotation, the attention of new tokens over the pages, and the
attention mass of every block.

`own = False` computes each operator in its plain form with elementary torch
operations, in 32 bits (the rotation's angles in 64) and rounded once; `own =
True` makes the framework's calls.  The head counts, the 128- and 64-wide
heads and the 16- and 64-token blocks are the ones this repository's tests
and benchmark use.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- cases ---------------------------------------------------------------------
# op      append | attend | mass
# n       sequences; new: most new tokens of one; held: most tokens held before
# mix     0: every sequence has `new` and `held`; else the seed of ragged ones
# hq, hk  query and KV heads; d: head width; block: tokens of a page
# layout  nhd | hnd: one page holds every KV head; slab: one page a KV head
# window  attended tokens (0: all); lse: the call also returns it
# rot     rotated elements; inter: adjacent pairs; norm: q and k norms; far: position offset

def _append(name, **kw):
    c = dict(name=name, op="append", n=1, new=1, held=0, mix=0, hq=32, hk=8, d=128, block=16,
             layout="hnd", dtype="bf16", rot=128, inter=False, norm=False, factor=1.0, far=0)
    c.update(kw)
    return c


def _attend(name, **kw):
    c = dict(name=name, op="attend", n=1, new=1, held=0, mix=0, hq=32, hk=8, d=128, block=16,
             layout="hnd", dtype="bf16", window=0, lse=False)
    c.update(kw)
    return c


def _mass(name, **kw):
    c = _attend(name, **kw)
    c["op"] = "mass"
    return c


def listed():
    return [
        # one request's next token, one layer: latency alone
        _append("append 1 token", held=700),
        # the decode step of the benchmark's 32 requests, one layer
        _append("append 32 x 1 token", n=32, held=8191, hq=28, hk=4, layout="slab"),
        # a prefill of four prompts with q and k norms, positions of a long context, scaled
        _append("append 8k tokens, norms", n=4, new=2700, held=5000, mix=3, hq=64, hk=8,
                layout="nhd", norm=True, factor=8.0, far=100000),
        # 32-bit cache of narrow heads, half of each rotated in adjacent pairs, odd lengths
        _append("append ragged fp32", n=9, new=333, held=77, mix=5, hq=14, hk=2, d=64, block=64,
                dtype="fp32", rot=32, inter=True),
        # one request's next token over a short context: latency alone
        _attend("attend 1 token", held=900, lse=True),
        # the decode step of the benchmark's 32 requests, one layer
        _attend("attend 32 x 1 token", n=32, held=8191, hq=28, hk=4, layout="slab", lse=True),
        # decode of many requests of very different lengths, a sliding window, 64-token blocks
        _attend("attend ragged decode", n=61, held=16000, mix=7, hq=64, hk=8, block=64,
                layout="nhd", dtype="fp16", window=6000),
        # a prefill chunk late in a long prompt
        _attend("attend 4k over 32k", new=4096, held=28672, layout="nhd"),
        # prompts' chunks and single tokens in one batch, odd lengths, narrow heads
        _attend("attend mixed batch", n=24, new=1100, held=4000, mix=11, hq=28, hk=4, d=64, block=64,
                dtype="fp16", lse=True),
        # block scores of one request's step: latency alone
        _mass("mass 1 token", held=900),
        # block scores of the benchmark's decode step, one layer
        _mass("mass 32 x 1 token", n=32, held=8191, hq=28, hk=4, layout="slab"),
        # block scores of a prefill chunk
        _mass("mass 2k over 16k", new=2048, held=14336, layout="nhd"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "mass"])
    hq, hk = rng.choice([(32, 8), (28, 4), (64, 8), (8, 8), (14, 2)])
    c = dict(op=op, mix=rng.randrange(1, 10 ** 6), hq=hq, hk=hk, d=rng.choice([128, 128, 64]),
             block=rng.choice([16, 16, 32, 64]), layout=rng.choice(["nhd", "hnd", "slab"]),
             dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if op == "append":
        c.update(n=_log(rng, 1, 64), held=_log(rng, 1, 4000), norm=rng.random() < 0.5,
                 inter=rng.random() < 0.5, factor=rng.choice([1.0, 8.0]), far=rng.choice([0, 100000]))
        c["rot"] = rng.choice([c["d"], c["d"], c["d"] // 2])
        if rng.random() < 0.25:
            c["dtype"] = "fp32"
        c["new"] = _log(rng, 1, min(4000, 8000 // c["n"]))
        return c
    if rng.random() < 0.5:                        # decode
        c.update(n=_log(rng, 1, 64), new=1, held=_log(rng, 1, 16000))
        if rng.random() < 0.2:
            c["dtype"] = "fp32"
    else:                                         # chunks
        c.update(n=_log(rng, 1, 16), held=_log(rng, 1, 16000))
        c["new"] = _log(rng, 2, 3000)
    c.update(window=rng.choice([0, 0, _log(rng, 1, 8000)]), lse=rng.random() < 0.5)
    most = 2.0e9                                  # scores of the padded plain form
    while c["n"] * c["new"] * (c["new"] + c["held"]) * c["hq"] > most:
        if c["n"] > 1:
            c["n"] = (c["n"] + 1) // 2
        else:
            c["new"] = (c["new"] + 1) // 2
    return c


def _lengths(case):
    """(new tokens, tokens held before) of every sequence."""
    n, new, held = case["n"], case["new"], case["held"]
    if not case["mix"]:
        return [(new, held)] * n
    r = random.Random(case["mix"])
    out = [(max(1, int(new * r.random() ** 2)) if r.random() < 0.8 else 1,
            int(held * r.random())) for _ in range(n)]
    out[r.randrange(n)] = (new, held)
    return out


# ---- inputs --------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["dtype"]]
    n, hq, hk, d, bs = case["n"], case["hq"], case["hk"], case["d"], case["block"]
    lens = _lengths(case)
    new = [a for a, _ in lens]
    total = [a + b for a, b in lens]
    T = sum(new)
    width = max(-(-t // bs) for t in total)
    per_head = case["layout"] == "slab"

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dt)

    # pages in random order of a pool with some to spare
    cols = torch.arange(width, device="cuda")
    need = torch.tensor([-(-t // bs) for t in total], device="cuda")
    used = cols[None, :] < need[:, None]
    if per_head:
        used = used[:, None, :].expand(n, hk, width)
    count = int(used.sum())
    pages = count + 7
    order = torch.randperm(pages, generator=g, device="cuda")[:count].to(torch.int32)
    table = torch.full(used.shape, -1, dtype=torch.int32, device="cuda")
    table[used] = order
    if per_head:
        pool = randn(pages, 2, bs, d)
        kp, vp = pool[:, 0], pool[:, 1]
    else:
        shape = (pages, bs, hk, d) if case["layout"] == "nhd" else (pages, hk, bs, d)
        kp, vp = randn(*shape), randn(*shape)
    s = dict(case=case, kp=kp, vp=vp, table=table,
             lens=torch.tensor(total, dtype=torch.int32, device="cuda"),
             starts=torch.tensor([sum(new[:i]) for i in range(n + 1)], dtype=torch.int32, device="cuda"),
             max_new=max(new), max_len=max(total))
    if case["op"] == "append":
        qkv = randn(T, (hq + 2 * hk) * d)         # the projection's output, q, k and v side by side
        s["q"] = qkv[:, :hq * d].view(T, hq, d)
        s["k"] = qkv[:, hq * d:(hq + hk) * d].view(T, hk, d)
        s["v"] = qkv[:, (hq + hk) * d:].view(T, hk, d)
        rot = case["rot"]
        base = 500000.0 if case["far"] else 10000.0
        s["inv_freq"] = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot) / case["factor"]
        s["qn"] = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(dt) if case["norm"] else None
        s["kn"] = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(dt) if case["norm"] else None
        s["pos"] = None
        if case["far"]:
            at = s["starts"].long()
            row = torch.arange(T, device="cuda")
            i = torch.searchsorted(at, row, right=True) - 1
            s["pos"] = row - at[i + 1] + s["lens"].long()[i] + case["far"]
    else:
        s["q"] = randn(T, hq, d, scale=1.5)
        s["scale"] = d ** -0.5
        if case["op"] == "mass":
            s["lse"] = _lse(s)
    if own:
        from orchkv_b200 import paged
        s["kv"] = paged.PagedKV(kp, vp, layout=case["layout"])
        if case["op"] == "append":
            s["rotary"] = paged.Rotary(d, inv_freq=s["inv_freq"], interleaved=case["inter"])
    return s


# ---- plain forms ---------------------------------------------------------------

def _rows(s):
    """Sequence, index in it and cache position of every row."""
    at = s["starts"].long()
    row = torch.arange(s["q"].shape[0], device="cuda")
    i = torch.searchsorted(at, row, right=True) - 1
    return i, row - at[i], row - at[i + 1] + s["lens"].long()[i]


def _spread(s, x, fill=0.0):
    """[T, hq, ...] -> [n, hk, group, max_new, ...]: the rows of every sequence, padded."""
    c = s["case"]
    i, j, _ = _rows(s)
    y = x.new_full((c["n"], s["max_new"]) + x.shape[1:], fill)
    y[i, j] = x
    y = y.unflatten(2, (c["hk"], c["hq"] // c["hk"]))
    return y.movedim(1, 3)


def _cached(s, pages):
    """The pages of every sequence in 32 bits, [n, hk, width * block, d]."""
    c, t = s["case"], s["table"].long().clamp(min=0)
    if c["layout"] == "slab":
        return pages[t].float().flatten(2, 3)
    x = pages[t]
    x = x.movedim(3, 1) if c["layout"] == "nhd" else x.movedim(2, 1)
    return x.float().flatten(2, 3)


def _allowed(s):
    """[n, 1, 1, max_new, width * block]: the tokens that each row attends to."""
    c = s["case"]
    L = s["table"].shape[-1] * c["block"]
    at = s["starts"].long()
    m = at[1:] - at[:-1]
    pos = s["lens"].long()[:, None] - m[:, None] + torch.arange(s["max_new"], device="cuda")[None, :]
    t = torch.arange(L, device="cuda")
    ok = t[None, None, :] <= pos[:, :, None]
    if c["window"]:
        ok &= t[None, None, :] > pos[:, :, None] - c["window"]
    ok &= (torch.arange(s["max_new"], device="cuda")[None, :] < m[:, None])[:, :, None]
    return ok[:, None, None]


def _scores(s):
    x = torch.matmul(_spread(s, s["q"].float() * s["scale"]), _cached(s, s["kp"])[:, :, None].transpose(-1, -2))
    return x.masked_fill_(~_allowed(s), -math.inf)


def _lse(s):
    x = _scores(s)
    top = x.amax(-1, keepdim=True).clamp_(min=-1e30)
    y = x.sub_(top).exp_().sum(-1).log_() + top[..., 0]
    return _gathered(s, y)


def _gathered(s, y):
    """[n, hk, group, max_new, ...] -> [T, hq, ...]"""
    i, j, _ = _rows(s)
    return y.movedim(3, 1).flatten(2, 3)[i, j]


def _turn(x, cos, sin, rot, inter):
    y = x.clone()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., :rot // 2], x[..., rot // 2:rot])
    u, w = a * cos - b * sin, b * cos + a * sin
    if inter:
        y[..., 0:rot:2], y[..., 1:rot:2] = u, w
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = u, w
    return y


def _normed(x, w):
    x = x.float()
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float()


def _write(s, pages, x):
    """Rows x [T, hk, d] to their places in the pages."""
    c = s["case"]
    i, _, at = _rows(s)
    b, o = at // c["block"], at % c["block"]
    x = x.to(pages.dtype)
    if c["layout"] == "slab":
        pages[s["table"].long()[i, :, b], o[:, None]] = x
    elif c["layout"] == "nhd":
        pages[s["table"].long()[i, b], o] = x
    else:
        pages.transpose(1, 2)[s["table"].long()[i, b], o] = x


def run(s):
    c = s["case"]
    if own:
        kv = s["kv"]
        if c["op"] == "append":
            q = kv.append(s["k"], s["v"], s["table"], s["lens"], s["starts"], q=s["q"], rotary=s["rotary"],
                          positions=s["pos"], q_norm=s["qn"], k_norm=s["kn"], eps=1e-6)
            return [q, s["kp"], s["vp"]]
        if c["op"] == "attend":
            return kv.attend(s["q"], s["table"], s["lens"], s["starts"], scale=s["scale"], window=c["window"],
                             max_new=s["max_new"], return_lse=c["lse"])
        return kv.block_mass(s["q"], s["lse"], s["table"], s["lens"], s["starts"], scale=s["scale"],
                             window=c["window"], max_new=s["max_new"])
    if c["op"] == "append":
        pos = _rows(s)[2] if s["pos"] is None else s["pos"]
        angle = torch.remainder(pos.double()[:, None] * s["inv_freq"], 2 * math.pi)
        cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
        q = _turn(_normed(s["q"], s["qn"]), cos, sin, c["rot"], c["inter"]).to(s["q"].dtype)
        _write(s, s["kp"], _turn(_normed(s["k"], s["kn"]), cos, sin, c["rot"], c["inter"]))
        _write(s, s["vp"], s["v"])
        return [q, s["kp"], s["vp"]]
    x = _scores(s)
    if c["op"] == "attend":
        top = x.amax(-1, keepdim=True).clamp_(min=-1e30)
        x = x.sub_(top).exp_()
        l = x.sum(-1, keepdim=True)
        y = torch.matmul(x, _cached(s, s["vp"])[:, :, None]) / l.clamp(min=1e-38)
        out = _gathered(s, y).to(s["q"].dtype)
        return [out, _gathered(s, l.log()[..., 0] + top[..., 0])] if c["lse"] else out
    lse = _spread(s, s["lse"][..., None], math.inf)
    p = x.sub_(lse).exp_()
    return p.sum((2, 3)).unflatten(-1, (-1, c["block"])).sum(-1)


# ---- the least that a pass has to do ------------------------------------------------

def work(case):
    lens = _lengths(case)
    e = TYPES[case["dtype"]].itemsize
    hq, hk, d, w = case["hq"], case["hk"], case["d"], case.get("window", 0)
    T = sum(a for a, _ in lens)
    if case["op"] == "append":
        return {"bytes": e * T * d * (2 * hq + 4 * hk), "flops": T * d * (hq + hk) * (6 + 4 * case["norm"])}
    pairs = keys = 0
    for m, held in lens:
        total = m + held
        if w:
            full = sum(min(w, held + j + 1) for j in range(m))
            keys += min(total, m + w - 1)
        else:
            full = m * held + m * (m + 1) // 2
            keys += total
        pairs += full
    width = max(-(-(a + b) // case["block"]) for a, b in lens)
    if case["op"] == "attend":
        return {"bytes": e * d * (2 * T * hq + 2 * hk * keys) + 4 * T * hq * case["lse"],
                "flops": 4 * d * hq * pairs}
    return {"bytes": e * d * (T * hq + hk * keys) + 4 * T * hq + 4 * case["n"] * hk * width,
            "flops": 2 * d * hq * pairs}


# ---- in 64 bits, sequence by sequence ---------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    lens = _lengths(case)
    hq, hk, bs = case["hq"], case["hk"], case["block"]
    grp = hq // hk
    f64 = torch.float64
    if case["op"] == "append":
        out_q = torch.empty(s["q"].shape, dtype=f64, device="cuda")
        kp, vp = s["kp"].to(f64), s["vp"].to(f64)
        row = 0
        half = case["rot"] // 2
        for i, (m, held) in enumerate(lens):
            at = torch.arange(held, held + m, device="cuda")
            # the angle in parts: whole thousands of positions and the rest, added as rotations
            p = (at + case["far"]).to(f64)[:, None]
            f = s["inv_freq"][None, :]
            hi = torch.floor(p / 1024) * 1024
            c = torch.cos(hi * f) * torch.cos((p - hi) * f) - torch.sin(hi * f) * torch.sin((p - hi) * f)
            z = torch.sin(hi * f) * torch.cos((p - hi) * f) + torch.cos(hi * f) * torch.sin((p - hi) * f)
            first = torch.arange(half, device="cuda") * (2 if case["inter"] else 1)
            second = first + (1 if case["inter"] else half)
            for x, w, heads in ((s["q"], s["qn"], hq), (s["k"], s["kn"], hk)):
                y = x[row:row + m].to(f64)
                if w is not None:
                    y = y / torch.sqrt((y ** 2).sum(-1, keepdim=True) / case["d"] + 1e-6) * w.to(f64)
                r = y.clone()
                r[:, :, first] = y[:, :, first] * c[:, None] - y[:, :, second] * z[:, None]
                r[:, :, second] = y[:, :, first] * z[:, None] + y[:, :, second] * c[:, None]
                if heads == hq and x is s["q"]:
                    out_q[row:row + m] = r
                else:
                    kr = r
            b, o = at // bs, at % bs
            v = s["v"][row:row + m].to(f64)
            for h in range(hk):
                if case["layout"] == "slab":
                    page = s["table"][i, h].long()[b]
                    kp[page, o], vp[page, o] = kr[:, h], v[:, h]
                elif case["layout"] == "nhd":
                    page = s["table"][i].long()[b]
                    kp[page, o, h], vp[page, o, h] = kr[:, h], v[:, h]
                else:
                    page = s["table"][i].long()[b]
                    kp[page, h, o], vp[page, h, o] = kr[:, h], v[:, h]
            row += m
        return [out_q, kp, vp]
    T = s["q"].shape[0]
    out = torch.zeros(T, hq, case["d"], dtype=f64, device="cuda")
    lse = torch.zeros(T, hq, dtype=f64, device="cuda")
    mass = torch.zeros(case["n"], hk, s["table"].shape[-1], dtype=f64, device="cuda")
    row = 0
    for i, (m, held) in enumerate(lens):
        total = m + held
        nb = -(-total // bs)
        key = torch.arange(total, device="cuda")
        pos = torch.arange(held, total, device="cuda")
        hide = key[None, :] > pos[:, None]
        if case["window"]:
            hide |= key[None, :] <= pos[:, None] - case["window"]
        for h in range(hk):
            if case["layout"] == "slab":
                page = s["table"][i, h, :nb].long()
                k, v = s["kp"][page], s["vp"][page]
            else:
                page = s["table"][i, :nb].long()
                k, v = (s["kp"][page][:, :, h], s["vp"][page][:, :, h]) if case["layout"] == "nhd" else \
                    (s["kp"][page][:, h], s["vp"][page][:, h])
            k, v = k.reshape(-1, case["d"])[:total].to(f64), v.reshape(-1, case["d"])[:total].to(f64)
            for a in range(grp):
                z = (s["q"][row:row + m, h * grp + a].to(f64) @ k.T) * s["scale"]
                z[hide] = -math.inf
                if case["op"] == "mass":
                    z = torch.exp(z - s["lse"][row:row + m, h * grp + a].to(f64)[:, None]).sum(0)
                    z = torch.nn.functional.pad(z, (0, nb * bs - total))
                    mass[i, h, :nb] += z.view(nb, bs).sum(1)
                else:
                    lse[row:row + m, h * grp + a] = torch.logsumexp(z, 1)
                    out[row:row + m, h * grp + a] = torch.softmax(z, 1) @ v
        row += m
    if case["op"] == "mass":
        return mass
    return [out, lse] if case["lse"] else out
