"""8-bit cache pages at the edges of their index types: very many rows, slot ids in 64 bits."""
import pytest
import torch

from agent_factory_3_b200.ops import paged


def pool(device, pages=4, page=16, hkv=1, d=8):
    k, ks = paged.empty_fp8_pages(pages, page, hkv, d, device)
    v, vs = paged.empty_fp8_pages(pages, page, hkv, d, device)
    return k, v, ks, vs


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_slots_in_64_bits(device):
    """A slot outside the pool is skipped, whatever its low 32 bits say."""
    k, v, ks, vs = pool(device)
    x = torch.arange(1, 7, device=device).float()[:, None].expand(6, 16).bfloat16().contiguous()
    slots = torch.tensor([3, 2 ** 32 + 5, -2 ** 32 + 6, 64, -1, 7], device=device)
    paged.kv_store_fp8(x, 0, 8, slots, k, v, ks, vs)
    got = paged.dequantize_rows_reference(k.view(torch.uint8).view(paged.FP8), ks.transpose(1, 2))
    want = torch.zeros(64, device=device)
    want[3], want[7] = 1, 6
    assert torch.equal(got.reshape(64, 8), want[:, None].expand(64, 8))
    back = torch.full_like(x, 9.0)
    paged.kv_gather_fp8(back, 0, 8, slots, k, v, ks, vs)
    assert back[:, 0].tolist() == [1, 9, 9, 9, 9, 6]


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


@pytest.mark.gpu
def test_no_silent_loss_of_a_gradient():
    """The kernels have no backward pass: a q that asks for a gradient is refused."""
    k, v = (torch.zeros(2, 16, 1, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    args = (k, v, torch.zeros(1, 1, device="cuda", dtype=torch.int32),
            torch.tensor([3], device="cuda", dtype=torch.int32),
            torch.tensor([0, 1], device="cuda", dtype=torch.int32), None, 4, 1)
    q = torch.randn(1, 256, device="cuda").bfloat16().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        paged.paged_attention(q, *args)
    with torch.no_grad():
        assert (paged.paged_attention(q, *args) == 0).all()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_rows_of_no_sequence_are_not_written(device):
    k, v = (torch.randn(2, 16, 1, 64, device=device).bfloat16() for _ in range(2))
    q = torch.randn(6, 256, device=device).bfloat16()
    out = torch.full((6, 256), 7.0, device=device, dtype=torch.bfloat16)
    got = paged.paged_attention(q, k, v, torch.tensor([[0], [1]], device=device, dtype=torch.int32),
                                torch.tensor([3, 9], device=device, dtype=torch.int32),
                                torch.tensor([1, 2, 4], device=device, dtype=torch.int32), None, 4, 1,
                                out=out)
    assert got is out and (out[[0, 4, 5]] == 7).all() and (out[1:4] != 7).any(1).all()
