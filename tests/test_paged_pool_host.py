"""paged.pool_table without a GPU, over a stand-in for the data plane."""
import ctypes as C

import torch

from orchkv_b200 import paged


class Plane:
    """A data plane on device 3 whose pages hold 16 tokens."""

    def __init__(self):
        self.tier = (C.c_int * 4)(3, 0, 0, 0)

    def orchkv_pool_pages(self, heads, pages):
        C.cast(pages, C.POINTER(paged.Pages))[0].page_tokens = 16
        return 0

    def orchkv_gpu_tier(self):
        return C.addressof(self.tier)

    def slab_table(self, requests, layer, heads, row_len, table, lens):
        self.asked = (requests, layer, heads, row_len)
        return 0


def test_pool_tables_lie_on_the_pools_device(monkeypatch):
    plane, made = Plane(), []

    def empty(*shape, dtype, device):
        made.append(torch.device(device))
        return torch.zeros(*shape, dtype=dtype)

    monkeypatch.setattr(paged, "lib", lambda: plane)
    monkeypatch.setattr(paged, "core", lambda: plane)
    monkeypatch.setattr(torch, "empty", empty)
    table, lens = paged.pool_table((7, 9), 1, 33, 2)
    assert made == [torch.device("cuda", 3)] * 2
    assert table.shape == (2, 2, 3) and lens.shape == (2,) and plane.asked == ([7, 9], 1, 2, 33)
