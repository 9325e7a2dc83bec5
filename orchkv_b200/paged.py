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
state between calls.  Waits inside the kernels end after two seconds;
``orchkv_b200.lib().orchkv_paged_status()`` is not 0 once one has, and its call's
results are then not complete.  The operators have no gradient: an input that requires
one (a norm's weight, frequencies, lse and the pages among them) is refused
unless gradients are off, and tensors that a call writes into count as changed
in place.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import core, lib, torch_ops
from ._lib import Pages

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


def _pool_device() -> int:
    """The device of the data plane's GPU pool, once it is initialised."""
    return C.cast(lib().orchkv_gpu_tier(), C.POINTER(C.c_int))[0]         # its first field


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
        self.n_pages, self.page_tokens, self.head_dim, self.dtype = n_pages, tokens, head_dim, dtype
        self.n_kv_heads = heads                   # None: as many as the call's tables have
        self._ops = torch_ops().Pages(device, k_ptr, v_ptr, *strides, n_pages, tokens, heads or 0,
                                      head_dim, _DTYPES[dtype], self.k, self.v)

    @classmethod
    def over_pool(cls) -> "PagedKV":
        """The pages of the data plane's GPU pool (orchkv_init): slabs of one
        head, with tables from ``pool_table``.  Valid until its shutdown."""
        pg = Pages()
        rc = lib().orchkv_pool_pages(1, C.byref(pg))
        if rc != 0:
            raise RuntimeError(f"orchkv_pool_pages failed: {rc}")
        dtype = {v: k for k, v in _DTYPES.items()}.get(pg.dtype)
        _need(dtype is not None, "the pool's type is not supported")
        _need(pg.d_head <= 256 and pg.d_head * dtype.itemsize % 16 == 0,
              "d_head must be at most 256 and a multiple of 16 bytes")
        self = cls.__new__(cls)
        self.k = self.v = None
        self.layout = "slab"
        self._set(_pool_device(), pg.k, pg.v,
                  (pg.page_stride, pg.head_stride, pg.token_stride), pg.n_pages, pg.page_tokens, None,
                  pg.d_head, dtype)
        return self

    def append(self, k, v, table, lens, starts, *, q=None, rotary: Rotary | None = None,
               positions=None, q_norm=None, k_norm=None, eps: float = 1e-6, q_out=None):
        """The new tokens' k, v [rows, KV heads, head_dim] into the pages; lens
        count them already.  q [rows, query heads, head_dim] is returned
        rotated (in q_out if given, which may be q itself, and overlaps none
        of q, k and v otherwise).  q_norm, k_norm
        [head_dim]: RMS norm of each head first.  positions [rows] (int32 or
        int64): where the rotation takes a token to be, by default its place
        in its sequence.  Rows behind the last sequence are left alone."""
        turns, inter, scale = (None, False, 1.0) if rotary is None else (
            rotary.turns, rotary.interleaved, rotary.scale)
        return self._ops.append(k, v, table, lens, starts, q, turns, inter, scale, positions, q_norm,
                                k_norm, eps, q_out)

    def attend(self, q, table, lens, starts, *, scale: float | None = None, window: int = 0,
               max_new: int | None = None, return_lse: bool = False, out=None):
        """softmax(scale * q k) v of every row of q [rows, query heads,
        head_dim] over its sequence's tokens up to its own place (the last
        `window` of them if not 0); scale is head_dim ** -0.5 by default.
        Returns out (not q), or (out, lse) with lse [rows, query heads] fp32.  A row
        with nothing to attend to gets 0 and -inf.  out must overlap neither q
        nor itself.  max_new: the most new tokens of one sequence, if the
        caller knows it (decode: 1), lets the call leave out what only longer
        ones need (a decode step without it takes 7 to 70 % longer); the rows
        of a sequence with more of them may not be computed."""
        return self._ops.attend(q, table, lens, starts, scale, window, max_new, return_lse, out)

    def block_mass(self, q, lse, table, lens, starts, *, scale: float | None = None, window: int = 0,
                   max_new: int | None = None, out=None):
        """The attention mass of every block: [sequences, KV heads, table
        width] fp32, the sum over the sequence's rows, the KV head's query
        heads and the block's tokens of exp(scale * q k - lse), with the lse
        that attend returned for the same arguments."""
        return self._ops.block_mass(q, lse, table, lens, starts, scale, window, max_new, out)


def pool_table(requests, layer: int, row_len: int, n_kv_heads: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Table [requests, KV heads, blocks] and lens of one layer of data-plane
    requests (handles of ``orchkv_core.request_create``): the slabs of the
    blocks that lie on the GPU, -1 for the others, for the first `row_len`
    tokens.  Runs on the data plane's stream, which is the current stream
    after ``orchkv_core.set_stream`` and ordered with the default stream
    otherwise; take it again after blocks were allocated or moved."""
    cpp, pg = core(), Pages()
    rc = lib().orchkv_pool_pages(max(n_kv_heads, 1), C.byref(pg))
    if rc != 0:
        raise RuntimeError(f"orchkv_pool_pages failed: {rc}")
    _need(n_kv_heads > 0 and row_len > 0 and len(requests) > 0, "requests, heads and row_len must not be 0")
    device = torch.device("cuda", _pool_device())
    table = torch.empty(len(requests), n_kv_heads, -(-row_len // pg.page_tokens), dtype=torch.int32, device=device)
    lens = torch.empty(len(requests), dtype=torch.int32, device=device)
    rc = cpp.slab_table(list(requests), layer, n_kv_heads, row_len, table.data_ptr(), lens.data_ptr())
    if rc != 0:
        raise RuntimeError(f"orchkv_slab_table failed: {rc}")
    return table, lens
