"""Plain restatement, in 64 bits, of the operators over a paged KV cache:
append with norm and rotation, attention over the pages, block masses.

Sequence by sequence and head by head, with no regard for speed; tensors may
live on any device.  `pages` are indexed through `place`, the only part that
knows a layout.
"""
import math

import torch


def place(layout, page, tok, head):
    """Index of token `tok` of page `page` for KV head `head`."""
    if layout == "slab":
        return (page, tok)
    return (page, tok, head) if layout == "nhd" else (page, head, tok)


def page_tokens(pages, layout):
    return pages.shape[2] if layout == "hnd" else pages.shape[1]


def kv_heads(pages, layout, table):
    return {"slab": lambda: table.shape[1], "nhd": lambda: pages.shape[2],
            "hnd": lambda: pages.shape[1]}[layout]()


def sequences(lens, starts):
    """(index, first row, rows, tokens held) of every sequence."""
    st = starts.tolist()
    return [(i, st[i], st[i + 1] - st[i], L) for i, L in enumerate(lens.tolist())]


def tokens_of(pages, layout, table, i, h, length):
    """(rows [length, d] in 64 bits, which of them lie in a page)."""
    bs = page_tokens(pages, layout)
    tab = (table[i, h] if layout == "slab" else table[i]).tolist()
    d = pages.shape[-1]
    out = torch.zeros(length, d, dtype=torch.float64, device=pages.device)
    there = torch.zeros(length, dtype=torch.bool, device=pages.device)
    for b in range(-(-length // bs)):
        if b >= len(tab) or not 0 <= tab[b] < pages.shape[0]:
            continue
        a, e = b * bs, min(length, (b + 1) * bs)
        out[a:e] = pages[place(layout, tab[b], slice(0, e - a), h)].double()
        there[a:e] = True
    return out, there


def rotate(x, pos, inv_freq, interleaved, scale=1.0):
    """x [rows, heads, d] (float64) turned by pos [rows] * inv_freq radians."""
    n = inv_freq.numel()
    ang = pos.double()[:, None] * inv_freq.double()[None].to(pos.device)
    c, s = torch.cos(ang)[:, None] * scale, torch.sin(ang)[:, None] * scale
    first = torch.arange(n, device=x.device) * (2 if interleaved else 1)
    second = first + (1 if interleaved else n)
    y = x.clone()
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., second] * c + x[..., first] * s
    return y


def norm(x, w, eps):
    x = x.double()
    if w is None:
        return x
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()


def append(kp, vp, layout, table, lens, starts, k, v, q=None, inv_freq=None, interleaved=False,
           scale=1.0, positions=None, q_norm=None, k_norm=None, eps=1e-6):
    """(kp, vp, q) in 64 bits after the append; rows of no sequence keep NaN
    in q."""
    kp, vp = kp.double(), vp.double()
    bs = page_tokens(kp, layout)
    qo = None if q is None else torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    for i, r0, m, L in sequences(lens, starts):
        at = torch.arange(L - m, L, device=k.device)
        pos = at if positions is None else positions[r0:r0 + m]
        kk = norm(k[r0:r0 + m], k_norm, eps)
        qq = None if q is None else norm(q[r0:r0 + m], q_norm, eps)
        if inv_freq is not None:
            kk = rotate(kk, pos, inv_freq, interleaved, scale)
            qq = None if q is None else rotate(qq, pos, inv_freq, interleaved, scale)
        if q is not None:
            qo[r0:r0 + m] = qq
        for h in range(k.shape[1]):
            tab = (table[i, h] if layout == "slab" else table[i]).tolist()
            for j, t in enumerate(at.tolist()):
                if t < 0 or t // bs >= len(tab) or not 0 <= tab[t // bs] < kp.shape[0]:
                    continue
                ix = place(layout, tab[t // bs], t % bs, h)
                kp[ix], vp[ix] = kk[j, h], v[r0 + j, h].double()
    return kp, vp, qo


def attend(kp, vp, layout, table, lens, starts, q, scale, window=0):
    """out, lse and, for error bounds, sum p |v| and the largest scaled
    sum |q k| of each row, all [rows, heads, ...]; NaN in rows of no sequence."""
    T, hq, d = q.shape
    heads = kv_heads(kp, layout, table)
    g = hq // heads
    f64 = dict(dtype=torch.float64, device=q.device)
    out, bulk = (torch.full((T, hq, d), math.nan, **f64) for _ in range(2))
    lse, top = (torch.full((T, hq), math.nan, **f64) for _ in range(2))
    for i, r0, m, L in sequences(lens, starts):
        pos = torch.arange(L - m, L, device=q.device)
        t = torch.arange(L, device=q.device)
        for h in range(heads):
            k, there = tokens_of(kp, layout, table, i, h, L)
            v, _ = tokens_of(vp, layout, table, i, h, L)
            ok = there[None, :] & (t[None, :] <= pos[:, None])
            if window:
                ok &= t[None, :] > pos[:, None] - window
            for a in range(h * g, (h + 1) * g):
                qa = q[r0:r0 + m, a].double()
                kz = torch.where(there[:, None], k, torch.zeros_like(k))
                s = qa @ kz.T * scale
                s = torch.where(ok, s, torch.full_like(s, -math.inf))
                some = ok.any(1)
                mx = torch.where(some, s.amax(1) if L else torch.zeros(m, **f64), torch.zeros(m, **f64))
                e = torch.where(ok, torch.exp(s - mx[:, None]), torch.zeros_like(s))
                l = e.sum(1)
                p = e / torch.where(some, l, torch.ones_like(l))[:, None]
                used = ok.any(0)
                vz = torch.where(used[:, None], v, torch.zeros_like(v))
                out[r0:r0 + m, a] = p @ vz
                bulk[r0:r0 + m, a] = p @ vz.abs()
                lse[r0:r0 + m, a] = torch.where(some, mx + torch.log(torch.where(some, l, torch.ones_like(l))),
                                                torch.full_like(l, -math.inf))
                w = qa.abs() @ torch.where(used[:, None], kz, torch.zeros_like(kz)).abs().T * abs(scale)
                top[r0:r0 + m, a] = torch.where(ok, w, torch.zeros_like(w)).amax(1) if L else 0.0
    return out, lse, bulk, top


def block_mass(kp, layout, table, lens, starts, q, lse, scale, window=0):
    """[sequences, KV heads, width]."""
    heads = kv_heads(kp, layout, table)
    bs, g = page_tokens(kp, layout), q.shape[1] // heads
    mass = torch.zeros(lens.shape[0], heads, table.shape[-1], dtype=torch.float64, device=q.device)
    for i, r0, m, L in sequences(lens, starts):
        pos = torch.arange(L - m, L, device=q.device)
        t = torch.arange(L, device=q.device)
        for h in range(heads):
            k, there = tokens_of(kp, layout, table, i, h, L)
            ok = there[None, :] & (t[None, :] <= pos[:, None])
            if window:
                ok &= t[None, :] > pos[:, None] - window
            for a in range(h * g, (h + 1) * g):
                s = q[r0:r0 + m, a].double() @ torch.where(there[:, None], k, torch.zeros_like(k)).T * scale
                p = torch.where(ok, torch.exp(s - lse[r0:r0 + m, a].double()[:, None]), torch.zeros_like(s))
                for b in range(min(table.shape[-1], -(-L // bs))):
                    mass[i, h, b] += p[:, b * bs:(b + 1) * bs].sum()
    return mass
