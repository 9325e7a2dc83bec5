"""The operators over a paged KV cache (orchkv_b200/paged.py) against their
64-bit restatement (oracle/paged_model.py)."""
import math

import pytest

from oracle import paged_model as M
from tests import paged_cases as P

pytestmark = pytest.mark.gpu


def kv(c):
    from orchkv_b200 import paged
    return paged.PagedKV(c["kp"], c["vp"], c["layout"])


def attend(c, **kw):
    return kv(c).attend(c["q"], c["table"], c["lens"], c["starts"], return_lse=True, **kw)


# ---- append --------------------------------------------------------------------

@pytest.mark.parametrize("layout", ["nhd", "hnd", "slab"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("d,rot,inter", [(128, 128, False), (128, 64, True), (64, 64, True), (64, 32, False),
                                         (80, 80, False), (72, 20, False), (72, 72, True), (256, 256, False),
                                         (256, 2, True), (32, 0, False), (16, 16, False)])
def test_append(cuda, layout, dtype, d, rot, inter):
    torch = cuda
    from orchkv_b200 import paged
    block = 7 if layout == "hnd" else 16
    c = P.make(torch, [1, 5, 0, 37], [0, 15, 9, 100], hq=6, hk=3, d=d, block=block, layout=layout,
               dtype=dtype, extra_rows=2, stale=3.0, seed=d + rot)
    normed = rot != 64
    w = [(1 + 0.2 * torch.randn(d, generator=c["gen"], device="cuda")).to(c["dt"]) if normed else None
         for _ in range(2)]
    freq = None
    if rot:
        freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    ro = paged.Rotary(d, inv_freq=freq, interleaved=inter, scale=1.25) if rot else None
    want = M.append(c["kp"], c["vp"], c["layout"], c["table"], c["lens"], c["starts"], c["k"], c["v"], c["q"],
                    freq, inter, 1.25, None, w[0], w[1], 1e-5)
    q_out = torch.full_like(c["q"], 7.0)
    got = kv(c).append(c["k"], c["v"], c["table"], c["lens"], c["starts"], q=c["q"], rotary=ro, q_norm=w[0],
                       k_norm=w[1], eps=1e-5, q_out=q_out)
    assert got is q_out
    n = int(c["starts"][-1])
    # one rounding, and fp32 work on at most two products of magnitude |y|
    # (norm: sum of d squares, 1 / sqrt, two products)
    u = P.half_step(c["dt"])
    big = 1.25 * math.sqrt(2)
    for name, a, b in (("q", q_out[:n], want[2][:n]), ("k", c["kp"], want[0]), ("v", c["vp"], want[1])):
        amax = b.abs().amax(-1, keepdim=True)
        tol = u * 1.01 * b.abs() + (d + 16) * 2.0 ** -24 * big * amax + 2.0 ** -25 * (c["dt"] == torch.float16)
        assert ((a.double() - b).abs() <= tol).all(), name
    assert (q_out[n:] == 7.0).all()              # rows behind the last sequence
    assert torch.equal(c["vp"].double(), want[1])


@pytest.mark.parametrize("pos64", [False, True])
def test_append_far_positions(cuda, pos64):
    """Angles of positions in the hundreds of millions, in place of q, strided
    rows of one projection."""
    torch = cuda
    from orchkv_b200 import paged
    d, hq, hk = 128, 4, 2
    c = P.make(torch, [9, 70], [3, 0], hq=hq, hk=hk, d=d, dtype="fp32", stale=0.0)
    T = c["T"]
    qkv = torch.randn(T, (hq + 2 * hk) * d, device="cuda", generator=c["gen"])
    q = qkv[:, :hq * d].view(T, hq, d)
    k = qkv[:, hq * d:(hq + hk) * d].view(T, hk, d)
    v = qkv[:, (hq + hk) * d:].view(T, hk, d)
    pos = torch.arange(T, device="cuda") * 2_500_003 + 100_000_007
    pos = pos if pos64 else pos.to(torch.int32)
    freq = 500000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
    q0 = q.clone()
    want = M.append(c["kp"], c["vp"], "nhd", c["table"], c["lens"], c["starts"], k, v, q0, freq, False, 1.0,
                    pos.long())
    got = kv(c).append(k, v, c["table"], c["lens"], c["starts"], q=q, rotary=paged.Rotary(d, inv_freq=freq),
                       positions=pos, q_out=q)
    assert got is q
    # the fraction of a turn is kept in double: pos * turns is below 2^29, so
    # it is off by 2^-24 of a turn at most, and rounded to fp32 by 2^-26
    tol = 2 * math.pi * 2.0 ** -23 + 8 * 2.0 ** -24
    for a, b in ((q, want[2]), (c["kp"], want[0])):
        assert (a.double() - b).abs().max() <= tol * math.sqrt(2) * b.abs().max()
    assert torch.equal(c["vp"].double(), want[1])


def test_append_leaves_the_rest(cuda):
    """Tokens without a page are dropped, nothing else is touched, and k alone
    works without q, rotation and norms."""
    torch = cuda
    c = P.make(torch, [20, 3], [0, 30], d=64, block=16, stale=5.0)
    c["table"][0, 1] = -1
    c["table"][1, 2] = c["kp"].shape[0]          # one past the last page
    before = c["kp"].clone()
    want = M.append(c["kp"], c["vp"], "nhd", c["table"], c["lens"], c["starts"], c["k"], c["v"])
    assert kv(c).append(c["k"], c["v"], c["table"], c["lens"], c["starts"]) is None
    assert torch.equal(c["kp"].double(), want[0]) and torch.equal(c["vp"].double(), want[1])
    assert (c["kp"] != before).any()


def test_append_many_sequences(cuda):
    """More sequences than one probe of the search holds, empty ones between."""
    torch = cuda
    new = [(i * 7) % 3 for i in range(1500)]
    c = P.make(torch, new, [i % 5 for i in range(1500)], hq=2, hk=1, d=16, block=4, stale=0.0)
    want = M.append(c["kp"], c["vp"], "nhd", c["table"], c["lens"], c["starts"], c["k"], c["v"])
    kv(c).append(c["k"], c["v"], c["table"], c["lens"], c["starts"])
    assert torch.equal(c["kp"].double(), want[0])


# ---- attend --------------------------------------------------------------------

@pytest.mark.parametrize("layout,block", [("nhd", 16), ("hnd", 64), ("slab", 16), ("nhd", 7), ("slab", 1),
                                          ("hnd", 128), ("nhd", 256), ("hnd", 24)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("hq,hk", [(8, 2), (4, 4), (7, 1), (16, 1)])
def test_attend_one_token(cuda, layout, block, dtype, hq, hk):
    """One new token a sequence: lengths of one, of a page less or more, long."""
    torch = cuda
    held = [0, 1, block - 1, block, 127, 128, 1000, 333]
    c = P.make(torch, [1] * len(held), held, hq=hq, hk=hk, block=block, layout=layout, dtype=dtype,
               seed=block + hq)
    out, lse = attend(c, max_new=1)
    P.check_attend(c, out, lse, 128 ** -0.5)


@pytest.mark.parametrize("d", [8, 16, 40, 64, 80, 96, 128, 192, 256])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("new,held", [([1, 1], [70, 300]), ([33, 2, 150], [5, 0, 90])])
def test_attend_head_widths(cuda, d, dtype, new, held):
    torch = cuda
    c = P.make(torch, new, held, hq=6, hk=2, d=d, dtype=dtype, seed=d)
    out, lse = attend(c, scale=0.2)
    P.check_attend(c, out, lse, 0.2)


@pytest.mark.parametrize("layout,block", [("nhd", 16), ("hnd", 64), ("slab", 16), ("slab", 32), ("nhd", 128),
                                          ("hnd", 256), ("nhd", 20)])
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("fp16", 64), ("bf16", 64), ("fp16", 128)])
@pytest.mark.parametrize("window", [0, 1, 50, 300])
def test_attend_chunks(cuda, layout, block, dtype, d, window):
    """Ragged chunks with single tokens, an empty sequence and padding rows
    among them, causal, with and without a window."""
    torch = cuda
    new, held = [1, 300, 0, 129, 17, 64, 1], [77, 0, 40, 200, 511, 128, 0]
    c = P.make(torch, new, held, hq=14, hk=2, d=d, block=block, layout=layout, dtype=dtype, extra_rows=5,
               seed=window)
    out = torch.full_like(c["q"], 9.0)
    got, lse = attend(c, window=window, out=out)
    assert got is out
    P.check_attend(c, out, lse, d ** -0.5, window)
    assert (out[int(c["starts"][-1]):] == 9.0).all()


@pytest.mark.parametrize("new", [1, 40, 300])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("layout", ["nhd", "slab"])
def test_attend_over_resident_blocks(cuda, new, dtype, layout):
    """Blocks that have left the GPU hold nothing: holes, a hole at the end,
    a whole row with nothing left."""
    torch = cuda
    c = P.make(torch, [new, new, new], [700, 33, 0], hq=8, hk=2, layout=layout, dtype=dtype, seed=new)
    t = c["table"]
    g = torch.Generator(device="cuda").manual_seed(1)
    gone = torch.rand(t[0].shape, device="cuda", generator=g) < 0.5
    t[0][gone] = -1
    t[1] = c["kp"].shape[0] + 5                  # nothing at all
    out, lse = attend(c)
    o, l = P.check_attend(c, out, lse, 128 ** -0.5)
    rows = slice(new, 2 * new)
    assert (out[rows] == 0).all() and torch.isinf(lse[rows]).all()


@pytest.mark.parametrize("new", [1, 5, 200])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_attend_infinite_and_nan_keys_behind_the_mask(cuda, new, dtype):
    """Keys of later tokens may hold anything; places behind the length and
    pages of no sequence are NaN in every test here."""
    torch = cuda
    c = P.make(torch, [new], [130], hq=4, hk=1, dtype=dtype)
    kp = c["kp"]
    last = 130 + new - 1                         # the last token's key: only the last row sees it
    if new > 1:
        page = int(c["table"][0, last // 16])
        ok = c["q"][:-1].clone()
        out0, _ = attend(c)
        kp[page, last % 16] = math.nan
        out, lse = attend(c)
        assert torch.equal(out[:new - 1], out0[:new - 1])
        assert torch.isnan(out[new - 1]).all() and torch.isnan(lse[new - 1]).all()
    else:
        out, lse = attend(c)
        P.check_attend(c, out, lse, 128 ** -0.5)


@pytest.mark.parametrize("new,held", [(1, 200), (3, 130), (5, 27), (9, 700), (200, 130), (700, 300)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("window", [0, 40])
def test_attend_infinite_values_reach_their_rows_alone(cuda, new, held, dtype, bad, window):
    """A value that is infinite or NaN at one token (and one far before every
    window): the rows that attend to it, and they alone, are not finite there;
    every other number is as without it."""
    torch = cuda
    c = P.make(torch, [new, 2], [held, 60], hq=14, hk=2, dtype=dtype, seed=new)
    want, wl = attend(c, window=window)
    at = held + new // 2                          # the value's token
    page = c["table"][0].tolist()
    c["vp"][page[at // 16], at % 16, :, 7:10] = bad
    if window:
        c["vp"][page[0], 0] = bad                 # token 0: outside all windows but the first rows'
    out, lse = attend(c, window=window)
    assert torch.equal(lse, wl)
    for r in range(new + 2):
        sees = r < new and held + r >= at and (not window or held + r < at + window)
        first = bool(window) and r < new and held + r < window
        cols = torch.zeros(128, dtype=torch.bool, device="cuda")
        if sees:
            cols[7:10] = True
        if first:
            cols[:] = True
        assert (~torch.isfinite(out[r][:, cols])).all(), r
        assert torch.equal(out[r][:, ~cols], want[r][:, ~cols]), r


def test_attend_large_scores(cuda):
    """Scores in the hundreds: the maximum moves all the time."""
    torch = cuda
    for new in (1, 260):
        c = P.make(torch, [new], [900], hq=8, hk=2, qscale=20.0, seed=3)
        page = c["table"][0].tolist()
        for t in range(0, 900, 50):              # keys that grow along the sequence
            c["kp"][page[t // 16], t % 16] *= 1 + t / 300
        out, lse = attend(c)
        P.check_attend(c, out, lse, 128 ** -0.5)


def test_attend_strided_rows(cuda):
    torch = cuda
    for new in (1, 190):
        c = P.make(torch, [new, new], [50, 9], hq=8, hk=2, seed=new)
        wide = torch.randn(c["T"], 8 + 4, 128, device="cuda", generator=c["gen"]).to(c["dt"])
        c["q"] = wide[:, 2:10]
        hold = torch.full((8, c["T"], 136), 4.0, dtype=c["dt"], device="cuda")
        out = hold[:, :, :128].transpose(0, 1)
        got, lse = attend(c, out=out)
        P.check_attend(c, out, lse, 128 ** -0.5)
        assert (hold[:, :, 128:] == 4.0).all()


def test_attend_repeats_bit_for_bit(cuda):
    torch = cuda
    for new in (1, 33, 500):
        c = P.make(torch, [new] * 3, [4000, 100, 2500], hq=8, hk=2, seed=new)
        a, la = attend(c)
        for _ in range(3):
            b, lb = attend(c)
            assert torch.equal(a, b) and torch.equal(la, lb)


def test_attend_many_sequences(cuda):
    torch = cuda
    n = 700
    new = [1 if i % 4 else 2 for i in range(n)]
    new[13] = 0
    held = [(i * 37) % 90 for i in range(n)]
    held[400] = 3000
    c = P.make(torch, new, held, hq=4, hk=1, d=64, seed=9)
    out, lse = attend(c, max_new=2)
    P.check_attend(c, out, lse, 64 ** -0.5)


def test_attend_lengths_below_the_rows(cuda):
    """lens that count fewer tokens than the rows: the first rows have no place
    and attend to nothing."""
    torch = cuda
    c = P.make(torch, [6], [10], hq=4, hk=2, dtype="bf16")
    c["lens"][0] = 4
    out, lse = attend(c)
    assert (out[:2] == 0).all() and torch.isinf(lse[:2]).all()
    assert torch.isfinite(lse[2:]).all() and not torch.isnan(out).any()


# ---- block mass ------------------------------------------------------------------

@pytest.mark.parametrize("layout,block", [("nhd", 16), ("hnd", 64), ("slab", 16), ("nhd", 7), ("slab", 1),
                                          ("hnd", 128), ("nhd", 256), ("hnd", 24)])
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("fp16", 64), ("fp32", 128), ("bf16", 80)])
@pytest.mark.parametrize("new,held", [([1, 1, 1], [0, 100, 1000]), ([130, 1, 0, 40], [300, 9, 50, 0])])
@pytest.mark.parametrize("window", [0, 70])
def test_block_mass(cuda, layout, block, dtype, d, new, held, window):
    torch = cuda
    c = P.make(torch, new, held, hq=8, hk=2, d=d, block=block, layout=layout, dtype=dtype, extra_rows=1,
               seed=d, width=max(1, max(-(-(a + b) // block) for a, b in zip(new, held))) + 3)
    if block <= 16:
        c["table"][-1, ..., 1] = -1              # a block that left
    out, lse = attend(c, window=window)
    mass = kv(c).block_mass(c["q"], lse, c["table"], c["lens"], c["starts"], window=window)
    P.check_mass(c, mass, lse, d ** -0.5, window)
    # every row's weights add to one
    total = mass.sum((1, 2))
    for i, (m, h) in enumerate(zip(new, held)):
        rows = torch.isfinite(lse[int(c["starts"][i]):int(c["starts"][i + 1])]).sum()
        assert abs(float(total[i]) - float(rows)) <= 1e-3 * max(1, float(rows))


def test_block_mass_is_what_the_report_sums(cuda):
    """The masses equal tm_report_attn_probs' sums of a stored map: two
    managers, one fed the map, the other the masses."""
    torch = cuda
    import orchkv_b200 as okv
    from orchkv_b200 import paged
    n, hq, hk, d, block = 2, 8, 2, 64, 16
    c = P.make(torch, [1] * n, [319] * n, hq=hq, hk=hk, d=d, block=block)
    out, lse = attend(c, max_new=1)
    mass = kv(c).block_mass(c["q"], lse, c["table"], c["lens"], c["starts"], max_new=1)
    T, nb = 320, 320 // block
    probs = torch.zeros(n, hq, T, dtype=torch.float32, device="cuda")
    for i in range(n):
        for h in range(hk):
            k, _ = M.tokens_of(c["kp"], "nhd", c["table"], i, h, T)
            s = c["q"][i, h * 4:(h + 1) * 4].double() @ k.T * d ** -0.5
            probs[i, h * 4:(h + 1) * 4] = torch.softmax(s, 1).float()
    ids = torch.arange(n * hk * nb, dtype=torch.int32, device="cuda")
    a, b = okv.Manager(tracker_cap=1024), okv.Manager(tracker_cap=1024)
    try:
        L = okv.lib()
        for m in (a, b):
            for x in range(ids.numel()):
                assert m.register_id(x) == 0
        assert L.tm_report_attn_probs(a.ref, probs.data_ptr(), n, hq, hk, T, block, None, ids.data_ptr()) == 0
        assert L.tm_report_attn_batch_dev(b.ref, ids.data_ptr(), mass.data_ptr(), ids.numel()) == 0
        torch.cuda.synchronize()
        sa, sb = a.state()["sum"][:ids.numel()], b.state()["sum"][:ids.numel()]
        assert sa.sum() > 0
        # both within 2^-17 of the exact sum
        assert (abs(sa - sb) <= 2.0 ** -16 * abs(sa)).all()
    finally:
        a.close()
        b.close()


# ---- together, streams, graphs ----------------------------------------------------

def step(c, ro, pos=None, stream=None):
    x = kv(c)
    q = x.append(c["k"], c["v"], c["table"], c["lens"], c["starts"], q=c["q"], rotary=ro)
    out, lse = x.attend(q, c["table"], c["lens"], c["starts"], return_lse=True)
    return q, out, lse, x.block_mass(q, lse, c["table"], c["lens"], c["starts"])


@pytest.mark.parametrize("layout", ["nhd", "slab"])
def test_step_by_step_equals_one_chunk(cuda, layout):
    """A prompt appended and attended token by token gives what one chunk
    gives, to the rounding of the weights."""
    torch = cuda
    from orchkv_b200 import paged
    m, d = 90, 128
    ro = paged.Rotary(d, scaling={"type": "yarn", "factor": 4.0, "original": 32})
    whole = P.make(torch, [m], [0], hq=8, hk=2, layout=layout, stale=0.0, seed=4)
    q1, out1, _, mass1 = step(whole, ro)
    one = dict(whole, kp=torch.zeros_like(whole["kp"]), vp=torch.zeros_like(whole["vp"]))
    total = torch.zeros_like(mass1)
    for t in range(m):
        c = dict(one, k=whole["k"][t:t + 1], v=whole["v"][t:t + 1], q=whole["q"][t:t + 1],
                 lens=torch.tensor([t + 1], dtype=torch.int32, device="cuda"),
                 starts=torch.tensor([0, 1], dtype=torch.int32, device="cuda"))
        q, out, lse, mass = step(c, ro)
        assert torch.equal(q[0], q1[t])
        total += mass
        # two roundings of the weights and two of the result, against values of a few units
        assert (out[0].double() - out1[t].double()).abs().max() <= 4 * P.half_step(c["dt"]) * 5
    assert torch.equal(one["kp"], whole["kp"]) and torch.equal(one["vp"], whole["vp"])
    assert ((total - mass1).abs() <= 2.0 ** -14 * mass1 + 1e-30).all()


def test_captured_step_follows_its_lengths(cuda):
    """A captured step replays with lengths and tables changed in place, on
    another stream, beside an eager call in flight."""
    torch = cuda
    from orchkv_b200 import paged
    ro = paged.Rotary(128)
    c = P.make(torch, [1] * 4, [700, 30, 5, 64], hq=8, hk=2, width=50, stale=0.0, seed=6, spare=60)
    for i in range(4):                           # pages for tokens to come
        free = [p for p in range(c["kp"].shape[0]) if p not in c["table"].flatten().tolist()]
        row = c["table"][i]
        k = int((row >= 0).sum())
        row[k:k + 3] = torch.tensor(free[:3], dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(c, ro)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            got = step(c, ro)
    for extra in (0, 1, 20):
        c["lens"] += extra
        c["q"].normal_()
        c["k"].normal_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g.replay()
        x = P.make(torch, [60], [90], seed=extra)
        out, lse = attend(x)                     # another call while the graph runs
        torch.cuda.synchronize()
        P.check_attend(x, out, lse, 128 ** -0.5)
        P.check_attend(dict(c, q=got[0]), got[1], got[2], 128 ** -0.5)
        P.check_mass(dict(c, q=got[0]), got[3], got[2], 128 ** -0.5)


def test_two_streams_at_once(cuda):
    torch = cuda
    cs = [P.make(torch, [1] * 6, [3000 + 100 * k, 5, 900, 1, 77, 2000], hq=8, hk=2, seed=k) for k in range(2)]
    want = [attend(c) for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for c, s in zip(cs, streams):
            with torch.cuda.stream(s):
                got.append(attend(c))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_offsets_past_32_bits(cuda):
    """Pages more than 2^32 elements apart."""
    torch = cuda
    d, hk, block = 128, 8, 64
    pages = 2 ** 33 // (block * hk * d * 2) + 40  # 8.6 G bytes each of k and v, 4.3 G elements
    kp = torch.zeros(pages, block, hk, d, dtype=torch.bfloat16, device="cuda")
    vp = torch.zeros_like(kp)
    new, held = [1, 130], [200, 64]
    c = P.make(torch, new, held, hq=16, hk=hk, d=d, block=block, seed=2)
    src = c["table"].clone()
    used = sorted(set(src[src >= 0].tolist()))
    far = {p: pages - 1 - k for k, p in enumerate(used)}
    for p, f in far.items():
        kp[f], vp[f] = c["kp"][p], c["vp"][p]
        c["table"][src == p] = f
    c["kp"], c["vp"] = kp, vp
    out, lse = attend(c)
    P.check_attend(c, out, lse, d ** -0.5)
    mass = kv(c).block_mass(c["q"], lse, c["table"], c["lens"], c["starts"])
    P.check_mass(c, mass, lse, d ** -0.5)
    c["k"][:, :, :] = 1.5
    kv(c).append(c["k"], c["v"], c["table"], c["lens"], c["starts"])
    assert (kp[int(c["table"][0, 200 // block]), 200 % block] == 1.5).all()


# ---- refusals --------------------------------------------------------------------

def test_refusals(cuda):
    """Arguments that do not fit raise before anything is launched."""
    torch = cuda
    from orchkv_b200 import paged
    c = P.make(torch, [2, 1], [5, 30], hq=4, hk=2)
    x = kv(c)
    a = (c["table"], c["lens"], c["starts"])
    cpu, bad = c["q"].cpu(), torch.zeros(3, 5, 128, dtype=c["dt"], device="cuda")
    lse = torch.zeros(3, 4, device="cuda")
    calls = [
        (lambda: x.attend(c["q"].float(), *a), "dtype"),
        (lambda: x.attend(c["q"][:, :, :64], *a), "must be"),
        (lambda: x.attend(c["q"][0], *a), "must be"),
        (lambda: x.attend(bad, *a), "share"),
        (lambda: x.attend(cpu, *a), "device"),
        (lambda: x.attend(c["q"].transpose(1, 2).contiguous().transpose(1, 2), *a), "contiguous"),
        (lambda: x.attend(torch.zeros(3, 4, 132, dtype=c["dt"], device="cuda")[:, :, :128], *a), "16 bytes"),
        (lambda: x.attend(c["q"], c["table"].long(), *a[1:]), "int32"),
        (lambda: x.attend(c["q"], c["table"][0], *a[1:]), "table must be"),
        (lambda: x.attend(c["q"], c["table"][:, :0], *a[1:]), "no blocks"),
        (lambda: x.attend(c["q"], c["table"].t().contiguous().t(), *a[1:]), "contiguous"),
        (lambda: x.attend(c["q"], c["table"].cpu(), *a[1:]), "device"),
        (lambda: x.attend(c["q"], c["table"], c["lens"][:1], c["starts"]), "entries"),
        (lambda: x.attend(c["q"], c["table"], c["lens"], c["lens"]), "entries"),
        (lambda: x.attend(c["q"], *a, window=-1), "window"),
        (lambda: x.attend(c["q"], *a, max_new=-1), "max_new"),
        (lambda: x.attend(c["q"], *a, out=c["q"][:2]), "out must be"),
        (lambda: x.attend(c["q"], *a, out=c["q"]), "overlap"),
        (lambda: x.attend(c["q"].float().requires_grad_().to(c["dt"]), *a), "gradient"),
        (lambda: x.append(c["k"][:2], c["v"], *a), "v must be"),
        (lambda: x.append(c["q"], c["v"], *a), "k must be"),
        (lambda: x.append(c["k"], c["v"], *a, q_norm=c["k"][0, 0]), "go with q"),
        (lambda: x.append(c["k"], c["v"], *a, k_norm=c["k"][0]), "k_norm"),
        (lambda: x.append(c["k"], c["v"], *a, k_norm=c["k"][0, 0].float()), "k_norm"),
        (lambda: x.append(c["k"], c["v"], *a, positions=torch.zeros(2, device="cuda", dtype=torch.int32)),
         "positions"),
        (lambda: x.append(c["k"], c["v"], *a, positions=torch.zeros(3, device="cuda")), "positions"),
        (lambda: x.append(c["k"], c["v"], *a, rotary=paged.Rotary(256)), "wider"),
        (lambda: x.append(c["k"], c["v"], *a, rotary=paged.Rotary(128, device="cpu")), "wider|device"),
        (lambda: x.block_mass(c["q"], lse[:, :2], *a), "lse"),
        (lambda: x.block_mass(c["q"], lse.double(), *a), "lse"),
        (lambda: x.block_mass(c["q"], lse, *a, out=lse), "out must be"),
    ]
    for fn, msg in calls:
        with pytest.raises(ValueError, match=msg):
            fn()
    with pytest.raises(TypeError):
        x.attend(None, *a)
    from orchkv_b200 import lib
    assert lib().orchkv_paged_status() == 0


def test_nothing_to_do(cuda):
    torch = cuda
    c = P.make(torch, [0, 0], [5, 30], hq=4, hk=2)
    out, lse = attend(c)
    assert out.shape == (0, 4, 128) and lse.shape == (0, 4)
    assert kv(c).append(c["k"], c["v"], c["table"], c["lens"], c["starts"]) is None
    mass = kv(c).block_mass(c["q"], lse, c["table"], c["lens"], c["starts"])
    assert (mass == 0).all()
    none = [t[:0].contiguous() for t in (c["table"], c["lens"])] + [c["starts"][:1].contiguous()]
    assert kv(c).attend(c["q"], *none).shape == (0, 4, 128)
    assert kv(c).block_mass(c["q"], lse, *none).shape == (0, 2, c["table"].shape[1])


@pytest.mark.parametrize("scale", [0.0, -0.3])
@pytest.mark.parametrize("new", [1, 90])
def test_scales_that_turn_or_drop_the_order(cuda, scale, new):
    torch = cuda
    c = P.make(torch, [new, 3], [200, 10], hq=8, hk=2, seed=new)
    out, lse = attend(c, scale=scale)
    P.check_attend(c, out, lse, scale)
    mass = kv(c).block_mass(c["q"], lse, c["table"], c["lens"], c["starts"], scale=scale)
    P.check_mass(c, mass, lse, scale)


@pytest.mark.parametrize("hq,hk,block", [(28, 4, 16), (14, 2, 256), (12, 1, 8), (40, 1, 64), (3, 3, 32)])
@pytest.mark.parametrize("window", [0, 200])
def test_chunks_over_many_units(cuda, hq, hk, block, window):
    """Chunks long enough that units are cut and joined, groups that do not
    divide a tile, one head a KV head; masses of the same calls."""
    torch = cuda
    c = P.make(torch, [700, 1, 90], [900, 3000, 0], hq=hq, hk=hk, d=64, block=block, seed=hq)
    out, lse = attend(c, window=window)
    P.check_attend(c, out, lse, 64 ** -0.5, window)
    mass = kv(c).block_mass(c["q"], lse, c["table"], c["lens"], c["starts"], window=window)
    P.check_mass(c, mass, lse, 64 ** -0.5, window)
    again = kv(c).block_mass(c["q"], lse, c["table"], c["lens"], c["starts"], window=window)
    assert torch.equal(mass, again)
