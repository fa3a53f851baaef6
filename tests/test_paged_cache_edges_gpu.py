"""8-bit cache pages at the edges of their index types: very many rows."""
import pytest
import torch

from agent_factory_3_b200.ops import paged


def pool(device, pages=4, page=16, hkv=1, d=8):
    k, ks = paged.empty_fp8_pages(pages, page, hkv, d, device)
    v, vs = paged.empty_fp8_pages(pages, page, hkv, d, device)
    return k, v, ks, vs


@pytest.mark.gpu
def test_more_than_2_27_rows():
    n = 2 ** 27 + 100
    k, v, ks, vs = pool("cuda")
    x = torch.zeros(n, 8, device="cuda", dtype=torch.bfloat16)
    x[0], x[2 ** 27], x[n - 1] = 1.0, 2.0, 3.0
    slots = torch.full((n,), -1, device="cuda", dtype=torch.int32)
    slots[0], slots[2 ** 27], slots[n - 1] = 1, 2, 3
    paged.kv_store_fp8(x, 0, 0, slots, k, v, ks, vs)
    x.zero_()
    paged.kv_gather_fp8(x, 0, 0, slots, k, v, ks, vs)
    assert [float(x[i, 0]) for i in (0, 1, 2 ** 27, n - 1)] == [1.0, 0.0, 2.0, 3.0]
