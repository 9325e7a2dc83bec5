"""Operators over a paged KV cache, on the pages where they lie.

``PagedKV`` stands for one layer's pages (a vLLM-style cache tensor, or the
data plane's slab pool) and has the three operators a decode or prefill step
runs on them:

* ``append``: the new tokens' keys and values into their pages, with each
  head's RMS norm and the position rotation on the way, and the rotated
  queries out, in one launch;
* ``attend``: attention of the new tokens over the pages, from one token a
  sequence to long chunks, several sequences of any lengths in one call;
* ``block_mass``: every block's attention mass, the input of
  ``tm_report_attn_batch_dev``, without an attention map in memory.

A call's sequences are ragged: the new tokens of sequence i are rows
``starts[i]:starts[i+1]`` of the row tensors and the last of its ``lens[i]``
tokens; token t of KV head h lies in page ``table[i, t // page_tokens]``
(``table[i, h, ...]`` where pages hold one head).  Table entries that name no
page (negative, or past the last) hold nothing: such tokens are not written
and not attended to, so a cache whose cold blocks have left the GPU is
attended over what is there.  Lengths and tables are read on the device: a
captured call follows them.

Everything runs on torch's current stream of the cache's device and keeps no
state between calls.  The operators have no gradient.
"""
from __future__ import annotations

import math

import torch

from . import core

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


class Rotary:
    """Position rotation of the first `rotary_dim` elements of a head.

    Pairs are (p, p + rotary_dim / 2), or (2p, 2p + 1) when `interleaved`;
    pair p turns by position * frequency[p], frequency[p] = base ** (-2 p /
    rotary_dim) unless `inv_freq` gives them.  `scaling` stretches them for
    contexts longer than trained on:

    ``{"type": "linear", "factor": f}``
        every frequency / f
    ``{"type": "ntk", "factor": f}``
        base * f ** (rotary_dim / (rotary_dim - 2)): the slowest / f, the
        fastest as it was
    ``{"type": "yarn", "factor": f, "original": n, "beta_fast": 32, "beta_slow": 1}``
        pairs that turn more than beta_fast times within the original context
        n stay, those below beta_slow turns are / f, a linear ramp over the
        pair index between; results scaled by 0.1 ln f + 1 (or
        ``"attention"``)
    ``{"type": "banded", "factor": f, "original": n, "low": 1, "high": 4}``
        wavelengths below n / high stay, above n / low are / f, between them
        a ramp linear in n / wavelength
    """

    def __init__(self, head_dim: int, rotary_dim: int | None = None, base: float = 10000.0, *,
                 inv_freq: torch.Tensor | None = None, interleaved: bool = False,
                 scaling: dict | None = None, scale: float = 1.0, device="cuda"):
        if inv_freq is None:
            rotary_dim = head_dim if rotary_dim is None else rotary_dim
            freq, extra = self.frequencies(rotary_dim, base, scaling)
            scale = scale * extra
        else:
            if scaling is not None:
                raise ValueError("scaling is for computed frequencies: inv_freq is taken as it is")
            if inv_freq.dim() != 1:
                raise ValueError("inv_freq must have one dimension")
            freq = inv_freq
            if rotary_dim is not None and rotary_dim != 2 * freq.numel():
                raise ValueError(f"{freq.numel()} frequencies rotate {2 * freq.numel()} elements, "
                                 f"not {rotary_dim}")
            if inv_freq.is_cuda:
                device = inv_freq.device
        self.rotary_dim = 2 * freq.numel()
        if not 0 < self.rotary_dim <= head_dim:
            raise ValueError(f"{self.rotary_dim} rotated elements of a head of {head_dim}")
        self.interleaved = bool(interleaved)
        self.scale = float(scale)
        self.turns = (freq.to(torch.float64) / (2 * math.pi)).to(device).contiguous()

    @staticmethod
    def frequencies(rotary_dim: int, base: float = 10000.0,
                    scaling: dict | None = None) -> tuple[torch.Tensor, float]:
        """Radians per position of each pair (float64, CPU), and the factor of
        the rotated results."""
        if rotary_dim <= 0 or rotary_dim % 2:
            raise ValueError("rotary_dim must be positive and even")
        p = torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim
        if scaling is None:
            return base ** -p, 1.0
        kind, f = scaling.get("type"), float(scaling["factor"])
        if f < 1.0:
            raise ValueError("scaling factor below 1")
        if kind == "linear":
            return base ** -p / f, 1.0
        if kind == "ntk":
            if rotary_dim < 4:
                raise ValueError("ntk scaling needs a rotary_dim of 4 or more")
            return (base * f ** (rotary_dim / (rotary_dim - 2))) ** -p, 1.0
        freq = base ** -p
        n = float(scaling["original"]) if kind in ("yarn", "banded") else 0.0
        if kind == "yarn":
            def index(turns):                     # pair that turns so often in n positions
                return rotary_dim * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(base))
            lo = max(math.floor(index(float(scaling.get("beta_fast", 32)))), 0)
            hi = min(math.ceil(index(float(scaling.get("beta_slow", 1)))), rotary_dim - 1)
            ramp = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - lo)
                    / max(hi - lo, 1e-3)).clamp(0, 1)
            extra = scaling.get("attention")
            if extra is None:
                extra = 0.1 * math.log(f) + 1.0 if f > 1 else 1.0
            return freq * (1 - ramp) + freq / f * ramp, float(extra)
        if kind == "banded":
            low, high = float(scaling.get("low", 1)), float(scaling.get("high", 4))
            if not high > low:
                raise ValueError("banded scaling needs high above low")
            keep = ((n * freq / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
            return freq * keep + freq / f * (1 - keep), 1.0
        raise ValueError(f"unknown scaling type {kind!r}")


def _need(ok: bool, msg: str):
    if not ok:
        raise ValueError(msg)


class PagedKV:
    """One layer's pages.  `layout`:

    ``"nhd"``   k, v [pages, page tokens, KV heads, head_dim]
    ``"hnd"``   k, v [pages, KV heads, page tokens, head_dim]
    ``"slab"``  k, v [pages, page tokens, head_dim]: a page holds one head,
                tables are [sequences, KV heads, width]

    fp16, bf16 or fp32; equal strides, each a multiple of 16 bytes, the head's
    elements side by side; head_dim at most 256 and a multiple of 16 bytes."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, layout: str = "nhd"):
        _need(layout in ("nhd", "hnd", "slab"), f"unknown layout {layout!r}")
        _need(k.dtype in _DTYPES, f"pages of {k.dtype} are not supported")
        _need(k.shape == v.shape and k.dtype == v.dtype and k.stride() == v.stride()
              and k.device == v.device, "k and v pages must be alike")
        _need(k.dim() == (3 if layout == "slab" else 4), f"{layout} pages have "
              f"{3 if layout == 'slab' else 4} dimensions, not {k.dim()}")
        _need(k.numel() > 0, "empty pages")
        _need(k.stride(-1) == 1, "the elements of a head must lie side by side")
        st, sh = k.stride(), k.shape
        if layout == "nhd":
            tokens, heads, s_tok, s_head = sh[1], sh[2], st[1], st[2]
        elif layout == "hnd":
            tokens, heads, s_tok, s_head = sh[2], sh[1], st[2], st[1]
        else:
            tokens, heads, s_tok, s_head = sh[1], None, st[1], 0
        e = k.element_size()
        _need(sh[-1] <= 256 and sh[-1] * e % 16 == 0,
              "head_dim must be at most 256 and a multiple of 16 bytes")
        _need(not (s_tok * e % 16 or s_head * e % 16 or st[0] * e % 16
                   or k.data_ptr() % 16 or v.data_ptr() % 16),
              "pages and their strides must be multiples of 16 bytes")
        _need(k.is_cuda, "pages must be on a CUDA device")
        self.k, self.v, self.layout = k, v, layout
        self._set(k.get_device(), k.data_ptr(), v.data_ptr(), (st[0], s_head, s_tok), sh[0], tokens,
                  heads, sh[-1], k.dtype)

    def _set(self, device, k_ptr, v_ptr, strides, n_pages, tokens, heads, head_dim, dtype):
        self._C = core()
        self._dev = device
        self.n_pages, self.page_tokens, self.head_dim, self.dtype = n_pages, tokens, head_dim, dtype
        self.n_kv_heads = heads                   # None: as many as the call's tables have
        self._args = (k_ptr, v_ptr) + strides + (n_pages, tokens)
        self._align = 16 // dtype.itemsize
        self._by_heads = {}

    def _pages(self, heads: int):
        _need(heads > 0, "a table of no heads")
        pg = self._by_heads[heads] = self._C.Pages(*self._args, heads, self.head_dim,
                                                   _DTYPES[self.dtype])
        return pg

    # -- argument checks -----------------------------------------------------

    def _batch(self, table, lens, starts, rows, max_new):
        """(pages handle, KV heads, the batch's arguments)."""
        i32, dev, slab = torch.int32, self._dev, self.n_kv_heads is None
        shape = table.shape
        if table.dtype != i32 or lens.dtype != i32 or starts.dtype != i32:
            raise ValueError("table, lens and starts must be int32")
        if len(shape) != (3 if slab else 2):
            raise ValueError("table must be [sequences, KV heads, width]" if slab
                             else "table must be [sequences, width]")
        n, width = shape[0], shape[-1]
        if lens.shape != (n,) or starts.shape != (n + 1,):
            raise ValueError("table, lens and starts must have n, n and n + 1 entries")
        st = table.stride()
        if st[-1] != 1 or not lens.is_contiguous() or not starts.is_contiguous():
            raise ValueError("table rows, lens and starts must be contiguous")
        if width == 0:
            raise ValueError("a table of no blocks")
        if table.get_device() != dev or lens.get_device() != dev or starts.get_device() != dev:
            raise ValueError("every tensor must be on the pages' device")
        if max_new is None:
            max_new = rows
        elif max_new < 0:
            raise ValueError("max_new must not be negative")
        heads = shape[1] if slab else self.n_kv_heads
        pg = self._by_heads.get(heads) or self._pages(heads)
        return pg, heads, (table.data_ptr(), st[0], st[1] if slab else 0, width, n, lens.data_ptr(),
                           starts.data_ptr(), rows, max_new)

    def _rows(self, x, name, heads=None, rows=None):
        """Checks a row tensor; its (pointer, row stride, head stride)."""
        shape = x.shape
        if (len(shape) != 3 or shape[2] != self.head_dim or (heads is not None and shape[1] != heads)
                or (rows is not None and shape[0] != rows)):
            raise ValueError(f"{name} must be [rows, heads, {self.head_dim}]"
                             + ("" if heads is None else f" with {heads} heads")
                             + ("" if rows is None else f" and {rows} rows"))
        if x.dtype != self.dtype:
            raise ValueError(f"{name} must be {self.dtype} as the pages are")
        p, s, align = x.data_ptr(), x.stride(), self._align
        if (s[2] != 1 or s[0] % align or s[1] % align or p % 16) and x.numel():
            raise ValueError(f"{name}: heads must be contiguous, pointer and strides multiples of "
                             "16 bytes")
        if x.get_device() != self._dev:
            raise ValueError(f"{name} must be on the pages' device")
        if x.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} requires a gradient, which these operators do not have")
        return p, s[0], s[1]

    def _heads(self, hq, heads, window):
        if hq == 0 or hq % heads:
            raise ValueError(f"{hq} query heads do not share {heads} KV heads")
        if window < 0:
            raise ValueError("window must not be negative")

    def _call(self, fn, *args):
        dev = self._dev
        if torch.cuda.current_device() == dev:
            rc = fn(*args, torch.cuda.current_stream(dev).cuda_stream)
        else:
            with torch.cuda.device(dev):
                rc = fn(*args, torch.cuda.current_stream(dev).cuda_stream)
        if rc != 0:
            raise RuntimeError(f"orchkv_{fn.__name__} failed: {rc}")

    # -- the operators -------------------------------------------------------

    def append(self, k, v, table, lens, starts, *, q=None, rotary: Rotary | None = None,
               positions=None, q_norm=None, k_norm=None, eps: float = 1e-6, q_out=None):
        """The new tokens' k, v [rows, KV heads, head_dim] into the pages; lens
        count them already.  q [rows, query heads, head_dim] is returned
        rotated (in q_out if given, which may be q).  q_norm, k_norm
        [head_dim]: RMS norm of each head first.  positions [rows] (int32 or
        int64): where the rotation takes a token to be, by default its place
        in its sequence.  Rows behind the last sequence are left alone."""
        rows = k.shape[0]
        pg, heads, batch = self._batch(table, lens, starts, rows, None)
        ka, va = self._rows(k, "k", heads), self._rows(v, "v", heads, rows)
        qa = oa = (0, 0, 0)
        hq = 0
        if q is not None:
            qa = self._rows(q, "q", None, rows)
            hq = q.shape[1]
            if q_out is None:
                q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            oa = self._rows(q_out, "q_out", hq, rows)
        else:
            _need(q_out is None and q_norm is None, "q_out and q_norm go with q")
        pos, pos64 = 0, 0
        if positions is not None:
            _need(positions.dtype in (torch.int32, torch.int64) and positions.shape == (rows,)
                  and positions.is_contiguous() and positions.get_device() == self._dev,
                  "positions must be int32 or int64 [rows], contiguous, on the pages' device")
            pos, pos64 = positions.data_ptr(), int(positions.dtype == torch.int64)
        norms = []
        for w, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
            if w is not None:
                if (w.shape != (self.head_dim,) or w.dtype != self.dtype or not w.is_contiguous()
                        or w.get_device() != self._dev):
                    raise ValueError(f"{name} must be [{self.head_dim}] {self.dtype}, contiguous, on "
                                     "the pages' device")
            norms.append(0 if w is None else w.data_ptr())
        rot, inter, scale, turns = 0, 0, 1.0, 0
        if rotary is not None:
            rot, inter, scale = rotary.rotary_dim, int(rotary.interleaved), rotary.scale
            _need(rot <= self.head_dim and rotary.turns.get_device() == self._dev,
                  "rotary wider than a head, or on another device")
            turns = rotary.turns.data_ptr()
        self._call(self._C.paged_append, pg, batch, qa, oa, ka, va,
                   (hq, rot, inter, scale, turns, pos, pos64, norms[0], norms[1], eps))
        return q_out

    def attend(self, q, table, lens, starts, *, scale: float | None = None, window: int = 0,
               max_new: int | None = None, return_lse: bool = False, out=None):
        """softmax(scale * q k) v of every row of q [rows, query heads,
        head_dim] over its sequence's tokens up to its own place (the last
        `window` of them if not 0); scale is head_dim ** -0.5 by default.
        Returns out, or (out, lse) with lse [rows, query heads] fp32.  A row
        with nothing to attend to gets 0 and -inf.  max_new: the most new
        tokens of one sequence, if the caller knows it (decode: 1), lets the
        call leave out what only longer ones need."""
        rows = q.shape[0]
        qa = self._rows(q, "q")
        hq = q.shape[1]
        pg, heads, batch = self._batch(table, lens, starts, rows, max_new)
        self._heads(hq, heads, window)
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        oa = self._rows(out, "out", hq, rows)
        lse = torch.empty(rows, hq, dtype=torch.float32, device=q.device) if return_lse else None
        args = (hq, self.head_dim ** -0.5 if scale is None else scale, window)
        need = self._C.paged_attend_workspace(pg, batch, args)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        self._call(self._C.paged_attend, pg, batch, qa, oa, lse.data_ptr() if return_lse else 0, args,
                   ws.data_ptr(), need)
        return (out, lse) if return_lse else out

    def block_mass(self, q, lse, table, lens, starts, *, scale: float | None = None, window: int = 0,
                   max_new: int | None = None, out=None):
        """The attention mass of every block: [sequences, KV heads, table
        width] fp32, the sum over the sequence's rows, the KV head's query
        heads and the block's tokens of exp(scale * q k - lse), with the lse
        that attend returned for the same arguments."""
        rows = q.shape[0]
        qa = self._rows(q, "q")
        hq = q.shape[1]
        pg, heads, batch = self._batch(table, lens, starts, rows, max_new)
        self._heads(hq, heads, window)
        if (lse.dtype != torch.float32 or lse.shape != (rows, hq) or not lse.is_contiguous()
                or lse.get_device() != self._dev):
            raise ValueError(f"lse must be fp32 [{rows}, {hq}], contiguous, on the pages' device")
        shape = (lens.shape[0], heads, table.shape[-1])
        if out is None:
            out = torch.empty(shape, dtype=torch.float32, device=q.device)
        else:
            if (out.shape != shape or out.dtype != torch.float32 or not out.is_contiguous()
                    or out.get_device() != self._dev):
                raise ValueError(f"out must be fp32 {list(shape)}, contiguous, on the pages' device")
        args = (hq, self.head_dim ** -0.5 if scale is None else scale, window)
        need = self._C.paged_block_mass_workspace(pg, batch, qa, args)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        self._call(self._C.paged_block_mass, pg, batch, qa, lse.data_ptr(), out.data_ptr(), args,
                   ws.data_ptr() if need else 0, need)
        return out
