"""The paged operators on the data plane's own pool: blocks allocated by the
data plane, written, attended over and weighed by the operators, reported,
selected and evicted by the scheduler, and attended over again without the
evicted ones -- the step a decode loop makes."""
import ctypes as C

import pytest

from oracle import paged_model as M
from tests import paged_cases as P

pytestmark = pytest.mark.gpu

L, HQ, HK, D, TPB = 2, 8, 2, 128, 16
SLAB = TPB * D * 2 * 2
N_SLABS = 512


@pytest.fixture
def dp(cuda):
    import orchkv_b200 as o
    cfg = o.make_config(gpu_pool_bytes=N_SLABS * SLAB, dram_pool_bytes=256 * SLAB, tokens_per_block=TPB,
                        d_head=D, dtype=1, max_blocks_per_head=64)
    ext = o.OrchkvConfigExt()
    ext.max_blocks = 1024
    lib = o.lib()
    assert lib.orchkv_init_ext(C.byref(cfg), C.byref(ext)) == 0
    m = o.Manager(tracker_cap=1024, max_blocks=1 << 12)
    assert lib.orchkv_attach_scheduler(m.ref) == 0
    yield o, lib, m
    assert lib.orchkv_shutdown() == 0
    m.close()


class _Raw:
    def __init__(self, ptr, shape):
        self.__cuda_array_interface__ = dict(shape=shape, typestr="<i2", data=(ptr, False), version=3)


def pool_tensors(torch, lib):
    """The pool as tensors [slab, token, d] of K and V."""
    t = torch.as_tensor(_Raw(lib.orchkv_gpu_pool_base(), (N_SLABS, 2, TPB, D)), device="cuda")
    t = t.view(torch.bfloat16)
    return t[:, 0], t[:, 1]


def test_decode_step_on_the_pool(cuda, dp):
    torch = cuda
    o, lib, m = dp
    from orchkv_b200 import paged
    core = o.core()
    core.set_stream(torch.cuda.current_stream().cuda_stream)
    new = [100, 37, 1]
    reqs = [core.request_create(10 + i, L, HK) for i in range(len(new))]
    kv = paged.PagedKV.over_pool()
    assert kv.page_tokens == TPB and kv.head_dim == D and kv.dtype == torch.bfloat16
    ro = paged.Rotary(D)
    kp, vp = pool_tensors(torch, lib)
    g = torch.Generator(device="cuda").manual_seed(0)
    freq = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)

    def rows(T):
        return [torch.randn(T, h, D, generator=g, device="cuda").to(torch.bfloat16) for h in (HQ, HK, HK)]

    def layer_step(l, new):
        T = sum(new)
        starts = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
        table, lens = paged.pool_table(reqs, l, 160, HK)
        q, k, v = rows(T)
        before = kp.clone(), vp.clone()
        want = M.append(*before, "slab", table, lens, starts, k, v, q, freq)
        qr = kv.append(k, v, table, lens, starts, q=q, rotary=ro)
        assert torch.equal(vp.double(), want[1])
        assert ((kp.double() - want[0]).abs() <= 2.0 ** -8 * want[0].abs() * 1.01 + 1e-4).all()
        out, lse = kv.attend(qr, table, lens, starts, max_new=max(new), return_lse=True)
        c = dict(kp=kp, vp=vp, layout="slab", table=table, lens=lens, starts=starts, q=qr, d=D,
                 dt=torch.bfloat16)
        P.check_attend(c, out, lse, D ** -0.5)
        mass = kv.block_mass(qr, lse, table, lens, starts, max_new=max(new))
        P.check_mass(c, mass, lse, D ** -0.5)
        return table, lens, mass

    # prefill, layer by layer: the data plane allocates, the operators write
    for l in range(L):
        for r, n in zip(reqs, new):
            assert core.prefill(r, l, 0, 0, n) == 0
        table, lens, _ = layer_step(l, new)
        assert lens.tolist() == new
    # a decode step: one token a request in every layer
    assert core.append_token_batch(reqs, 0, 0) == 0
    ids = torch.empty(len(reqs) * L, HK, 10, dtype=torch.int32, device="cuda")
    assert core.block_id_table(reqs, 160, ids.data_ptr()) == 0
    ids = ids.view(len(reqs), L, HK, 10)
    for l in range(L):
        table, lens, mass = layer_step(l, [1, 1, 1])
        assert lens.tolist() == [n + 1 for n in new]
        live = ids[:, l].contiguous()
        rc = lib.tm_report_attn_batch_dev(m.ref, live.data_ptr(), mass.data_ptr(), live.numel())
        assert rc == 0
    assert lib.tm_step_and_classify(m.ref) == 0
    # the coldest blocks leave; the next attention is over what is there
    out_ids = torch.zeros(20, dtype=torch.int32, device="cuda")
    count = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert lib.tm_select_victims(m.ref, 20, out_ids.data_ptr(), count.data_ptr()) == 0
    assert core.evict_batch_to_dram(out_ids.data_ptr(), count.data_ptr(), 20) == 0
    assert core.append_token_batch(reqs, 0, 0) in (0, -8)   # -8: a last block was among them
    gone = 0
    for l in range(L):
        table, lens = paged.pool_table(reqs, l, 160, HK)
        need = [-(-int(x) // TPB) for x in lens]
        gone += sum(int((table[i, :, :n] < 0).sum()) for i, n in enumerate(need))
        q = rows(3)[0]
        starts = torch.arange(4, dtype=torch.int32, device="cuda")
        out, lse = kv.attend(q, table, lens, starts, max_new=1, return_lse=True)
        P.check_attend(dict(kp=kp, vp=vp, layout="slab", table=table, lens=lens, starts=starts, q=q, d=D,
                            dt=torch.bfloat16), out, lse, D ** -0.5)
    assert gone == int(count.item()) == 20
    assert lib.orchkv_paged_status() == 0
    for r in reqs:
        core.request_destroy(r)


def test_pool_refusals(cuda, dp):
    torch = cuda
    o, lib, m = dp
    from orchkv_b200 import paged
    r = o.core().request_create(1, L, HK)
    with pytest.raises(RuntimeError, match="-2"):
        paged.pool_table([r], 0, 16, HK + 1)
    with pytest.raises(RuntimeError, match="-2"):
        paged.pool_table([r], L, 16, HK)
    with pytest.raises(ValueError):
        paged.pool_table([], 0, 16, HK)
    assert lib.orchkv_pool_pages(0, C.byref(o._lib.Pages())) == -2
    o.core().request_destroy(r)


def test_pool_needs_the_data_plane(cuda):
    from orchkv_b200 import paged
    with pytest.raises(RuntimeError, match="-9"):
        paged.PagedKV.over_pool()
    with pytest.raises(RuntimeError, match="-9"):
        paged.pool_table([1], 0, 16, 2)
