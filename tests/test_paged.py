"""8-bit KV cache pages and attention over pages on the CPU: the rounding rule from its
definition, the round trip, the reference against a key-by-key softmax, refusals."""
import math

import pytest
import torch

from agent_factory_3_b200.ops import paged


def test_quantisation_rule():
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(400, 64, generator=g) * torch.exp2(
        torch.randint(-120, 120, (400, 1), generator=g).float())).bfloat16()
    x[0] = 0
    x[1] = 448.0
    x[2] = 450.0
    x[3] = 3.3895e38
    x[4, 3], x[5, 4], x[6, 5] = math.nan, math.inf, -math.inf
    codes, scales = paged.quantize_rows_reference(x)
    grid = torch.arange(127, dtype=torch.uint8).view(paged.FP8).double()     # codes 0 .. 448
    e = scales.double() - 127
    xd = x.double()
    fin = torch.isfinite(xd)
    a = torch.where(fin, xd.abs(), torch.zeros_like(xd)).amax(-1)
    assert e[0] == -127 and e[1] == 0 and e[2] == 1 and e[3] == 120
    assert ((a <= 448 * 2.0 ** e) | (e == 120)).all()
    assert ((a > 448 * 2.0 ** (e - 1)) | (e == -127)).all()
    y = xd.abs() / 2.0 ** e[:, None]
    y = torch.where((e == 120)[:, None], y.clamp(max=240), y)
    near = (y[..., None] - grid).abs().amin(-1)
    got = codes.double()
    assert torch.equal(torch.isnan(got), ~fin)
    off = (got.abs() - y).abs()
    assert (off[fin] <= near[fin]).all() and (got.sign()[fin & (got != 0)] == xd.sign()[fin & (got != 0)]).all()
    back = paged.dequantize_rows_reference(codes, scales)
    assert torch.equal(back.bfloat16().float()[fin], back[fin]) and torch.isfinite(back[fin]).all()
    big = fin & (xd.abs() >= a[:, None] * 2.0 ** -14) & ((e > -127) & (e < 120))[:, None]
    assert ((back.double() - xd).abs()[big] <= 2.0 ** -4 * xd.abs()[big]).all()


def test_store_gather_round_trip():
    n, hkv, d, page = 37, 3, 32, 5
    k, ks = paged.empty_fp8_pages(10, page, hkv, d, "cpu")
    v, vs = paged.empty_fp8_pages(10, page, hkv, d, "cpu")
    x = torch.randn(n, 2 * hkv * d).bfloat16()
    slots = torch.randperm(50)[:n].to(torch.int32)
    slots[3], slots[4] = -1, 50
    paged.kv_store_fp8(x, 0, hkv * d, slots, k, v, ks, vs)
    back = torch.zeros_like(x)
    paged.kv_gather_fp8(back, 0, hkv * d, slots, k, v, ks, vs)
    keep = [i for i in range(n) if i not in (3, 4)]
    assert (back[[3, 4]] == 0).all()
    assert ((back[keep] - x[keep]).abs() <= 2.0 ** -4 * x[keep].abs() + 2.0 ** -9).all()
    again = torch.zeros_like(x)                      # values of the cache are stored as they are
    paged.kv_store_fp8(back, 0, hkv * d, slots, k, v, ks, vs)
    paged.kv_gather_fp8(again, 0, hkv * d, slots, k, v, ks, vs)
    assert torch.equal(again, back)


@pytest.mark.parametrize("window", [0, 3])
@pytest.mark.parametrize("fp8", [False, True])
def test_reference_against_single_rows(fp8, window):
    hq, hkv, d, page = 4, 2, 16, 4
    if fp8:
        k, ks = paged.empty_fp8_pages(8, page, hkv, d, "cpu")
        v, vs = paged.empty_fp8_pages(8, page, hkv, d, "cpu")
        paged.kv_store_fp8(torch.randn(32, 2 * hkv * d).bfloat16(), 0, hkv * d,
                           torch.arange(32, dtype=torch.int32), k, v, ks, vs)
        kd = paged.dequantize_rows_reference(k, ks.transpose(1, 2))
        vd = paged.dequantize_rows_reference(v, vs.transpose(1, 2))
    else:
        k, v = torch.randn(8, page, hkv, d).bfloat16(), torch.randn(8, page, hkv, d).bfloat16()
        ks = vs = None
        kd, vd = k, v
    lens, qn = [11, 3, 0, 2], [3, 1, 0, 4]
    table = torch.tensor([[5, 0, -1], [2, 9, 9], [0, 0, 0], [7, 1, 1]], dtype=torch.int32)
    cu = torch.tensor([0, 3, 4, 4, 8], dtype=torch.int32)
    q = torch.randn(8, hq * d).bfloat16()
    sinks = torch.randn(hq)
    out = paged.paged_attention_reference(q, k, v, table, torch.tensor(lens), cu, sinks, hq, hkv,
                                          window, k_scales=ks, v_scales=vs, dtype=torch.float64)
    for b in range(4):
        for i in range(qn[b]):
            pos = lens[b] - qn[b] + i
            for h in range(hq):
                num, den = torch.zeros(d, dtype=torch.float64), math.exp(float(sinks[h]))
                row = q[int(cu[b]) + i].view(hq, d)[h].double()
                for j in range(pos + 1):
                    pg = int(table[b, j // page])
                    if (window and pos - j >= window) or not 0 <= pg < 8:
                        continue
                    w = math.exp(float(row @ kd[pg, j % page, h // 2].double()) / 4.0)
                    num += w * vd[pg, j % page, h // 2].double()
                    den += w
                torch.testing.assert_close(out[int(cu[b]) + i].view(hq, d)[h], num / den,
                                           rtol=1e-6, atol=1e-9)


def test_refusals():
    k, ks = paged.empty_fp8_pages(4, 8, 2, 16, "cpu")
    args = dict(q=torch.randn(1, 64).bfloat16(), k_pages=k, v_pages=k,
                page_table=torch.zeros(1, 2, dtype=torch.int32),
                seq_lens=torch.tensor([3], dtype=torch.int32),
                cu_q=torch.tensor([0, 1], dtype=torch.int32), sinks=None, hq=4, hkv=2)
    paged.paged_attention(**args, k_scales=ks, v_scales=ks)
    for bad in (dict(), dict(k_scales=ks.float(), v_scales=ks), dict(k_scales=ks[:1], v_scales=ks[:1]),
                dict(k_scales=ks, v_scales=ks, hkv=3), dict(k_scales=ks, v_scales=ks, window=-1),
                dict(k_scales=ks, v_scales=ks, cu_q=torch.tensor([0])),
                dict(k_scales=ks, v_scales=ks, q=torch.randn(1, 60)),
                dict(k_pages=k.float(), v_pages=k.float(), k_scales=ks, v_scales=ks)):
        with pytest.raises(RuntimeError):
            paged.paged_attention(**{**args, **bad})
    with pytest.raises(RuntimeError):
        paged.kv_store_fp8(torch.randn(1, 64).bfloat16(), 0, 32, torch.zeros(1, dtype=torch.int32),
                           k.float(), k.float(), None, None)
