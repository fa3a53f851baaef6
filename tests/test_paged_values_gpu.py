"""Attention over cache pages where values differ in magnitude or are not finite, on the GPU
against 64 bits.  Tolerance: that of test_paged_gpu.check, a bf16 rounding of the output and
2^-12 of A, the same attention over |V|."""
import math

import pytest
import torch

from test_paged_gpu import check, make

from agent_factory_3_b200.ops import paged

pytestmark = pytest.mark.gpu


def slots_of(a, page):
    """Slots of the keys of sequence 0, in order."""
    n = int(a["seq_lens"][0])
    t = a["page_table"][0].long()
    j = torch.arange(n, device=t.device)
    return t[j // page] * page + j % page


def put(a, page, keys, k=None, v=None):
    """Writes rows [len(keys), Hkv, 64] into the pages at these keys of sequence 0."""
    at = slots_of(a, page)[torch.as_tensor(keys, device=a["q"].device)]
    hkv = a["hkv"]
    old = [paged.dequantize_rows_reference(
        p.view(torch.uint8)[at // page, at % page].view(paged.FP8), s[at // page, :, at % page])
        if s is not None else p[at // page, at % page].float()
        for p, s in ((a["k_pages"], a["k_scales"]), (a["v_pages"], a["v_scales"]))]
    k, v = (old[i] if x is None else x.float().expand(at.numel(), hkv, 64) for i, x in ((0, k), (1, v)))
    if a["k_scales"] is None:
        a["k_pages"][at // page, at % page] = k.bfloat16()
        a["v_pages"][at // page, at % page] = v.bfloat16()
    else:
        rows = torch.cat([k.reshape(-1, hkv * 64), v.reshape(-1, hkv * 64)], 1).bfloat16()
        paged.kv_store_fp8(rows, 0, hkv * 64, at.to(torch.int32), a["k_pages"], a["v_pages"],
                           a["k_scales"], a["v_scales"])


# ------------------------------------------------------------- values that are not finite
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("q,start,hq,hkv,window,key", [
    (256, 0, 2, 2, 0, 5),          # one head a KV head: rows 128 .. 255 see all of block 0
    (32, 112, 16, 2, 0, 5),        # tokens 16 .. 31 see all of block 0, tokens 0 .. 15 do not
    (32, 112, 16, 2, 0, 120),
    (40, 230, 64, 8, 0, 255),
    (2, 300, 128, 1, 200, 101),    # block 0 is whole for the first token only
    (2, 300, 128, 1, 200, 150),
    (64, 600, 16, 2, 300, 500),
])
def test_broken_value_that_whole_tiles_see(dev, fp8, q, start, hq, hkv, window, key):
    page = 16
    a = make(dev, [q], [start + q], hq, hkv, page, fp8)
    at = int(slots_of(a, page)[key])
    if fp8:
        a["v_pages"].view(torch.uint8)[at // page, at % page, :, 7] = 0x7F
    else:
        a["v_pages"][at // page, at % page, :, 7] = math.nan
    out = check(a, window)
    pos = start + torch.arange(q, device=dev)
    sees = (pos >= key) & ((pos - key < window) if window else (pos >= 0))
    assert torch.equal(torch.isnan(out.view(q, hq, 64)[..., 7]).all(1), sees)


@pytest.mark.parametrize("q", [1, 3, 60, 300])
@pytest.mark.parametrize("key", [5, 130, 399])
def test_scale_byte_that_is_no_number(dev, q, key):
    """A scale byte of 255 is no power of two (kv_store_fp8 never writes it): rows that see such a
    value are not finite, the others are as they were."""
    a = make(dev, [q], [400], 8, 1, 16, True)
    want = check(a)
    at = int(slots_of(a, 16)[key])
    a["v_scales"][at // 16, :, at % 16] = 255
    out = paged.paged_attention(**a, max_q_len=q, max_seq_len=400)
    sees = 400 - q + torch.arange(q, device=dev) >= key
    assert not torch.isfinite(out[sees]).any()
    assert ((out[~sees] - want[~sees]).abs() <= 2.0 ** -7 * want[~sees].abs() + 1e-3).all()


def test_scale_byte_that_is_no_number_in_k(dev):
    """The same key by key, for few rows and in the kernel of long chunks."""
    a = make(dev, [6], [400], 8, 1, 16, True)
    at = int(slots_of(a, 16)[200])
    a["k_scales"][at // 16, :, at % 16] = 255
    few = paged.paged_attention(**a, max_q_len=5, max_seq_len=400)       # 40 rows
    chunk = paged.paged_attention(**a, max_q_len=6, max_seq_len=400)     # 48 rows
    assert torch.isnan(few).any() and torch.isfinite(few).any()      # scores of +inf and of -inf
    assert torch.equal(torch.isnan(few), torch.isnan(chunk))
    assert ((few - chunk).abs() <= 2.0 ** -7 * few.abs() + 1e-3)[torch.isfinite(few)].all()


# ------------------------------------------------------------- magnitudes
@pytest.mark.parametrize("span", [16, 28, 40, 60])
@pytest.mark.parametrize("q,ctx,hq,hkv", [(1, 40, 16, 2), (1, 300, 8, 1), (1, 5000, 64, 8), (1, 700, 32, 1),
                                          (3, 400, 8, 1), (60, 500, 16, 2)])
def test_large_value_without_weight(dev, q, ctx, hq, hkv, span):
    """e4m3: a token whose value is 2^span times the others' and whose weight is e^-100."""
    page = 16
    a = make(dev, [q], [ctx], hq, hkv, page, True)
    u = torch.randn(64, device=dev).bfloat16()
    a["q"] = u.repeat(q, hq).contiguous()
    keys = torch.arange(ctx)
    k = 0.05 * torch.randn(ctx, hkv, 64, device=dev)
    v = torch.randn(ctx, hkv, 64, device=dev)
    for at in (1, ctx // 2):
        k[at] = -800.0 * u.float() / u.float().square().sum()      # scores of -100
        v[at] *= 2.0 ** span
    put(a, page, keys, k, v)
    check(a)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("span", [20, 45])
@pytest.mark.parametrize("q,ctx", [(1, 300), (1, 3000), (3, 400), (60, 500), (200, 1000)])
@pytest.mark.parametrize("first", [False, True])
def test_large_value_of_little_weight(dev, q, ctx, span, first, fp8):
    """A token of weight 2^-span of the largest and a value 2^span times the others' counts as much
    as they do, whether it is met before them or after them."""
    page, hq, hkv = 16, 8, 1
    a = make(dev, [q], [ctx], hq, hkv, page, fp8)
    a["sinks"] = torch.full((hq,), -20.0, device=dev)
    u = torch.randn(64, device=dev).bfloat16()
    a["q"] = u.repeat(q, hq).contiguous()
    k = torch.zeros(ctx, hkv, 64, device=dev)
    v = torch.randn(ctx, hkv, 64, device=dev)
    at = 2 if first else ctx - q
    k[at] = -8.0 * math.log(2.0 ** span) * u.float() / u.float().square().sum()
    v[at] *= 2.0 ** span * ctx
    put(a, page, torch.arange(ctx), k, v)
    check(a)


@pytest.mark.parametrize("q,ctx", [(1, 700), (3, 300), (60, 500), (300, 1000), (64, 6000)])
@pytest.mark.parametrize("power", [-20, -32, -60, 30])
def test_channel_of_another_magnitude(dev, q, ctx, power):
    """bf16 pages keep V's 8 bits at every magnitude, also in one channel among larger ones."""
    a = make(dev, [q], [ctx], 16, 2, 16, False)
    a["v_pages"][..., 5] *= 2.0 ** power
    check(a)
    check(a, window=100)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("q,ctx,window", [(1, 3000, 0), (5, 700, 0), (60, 500, 0), (60, 500, 400), (300, 1000, 0)])
def test_large_values_in_all_later_blocks(dev, q, ctx, window, fp8):
    """From key 384 on values are 2^45 times the earlier ones' at 2^-45 of their weight."""
    page, hq, hkv = 16, 8, 1
    a = make(dev, [q], [ctx], hq, hkv, page, fp8)
    a["sinks"] = torch.full((hq,), -20.0, device=dev)
    u = torch.randn(64, device=dev).bfloat16()
    a["q"] = u.repeat(q, hq).contiguous()
    k = torch.zeros(ctx, hkv, 64, device=dev)
    v = torch.randn(ctx, hkv, 64, device=dev)
    k[384:] = -8.0 * math.log(2.0 ** 45) * u.float() / u.float().square().sum()
    v[384:] *= 2.0 ** 45
    put(a, page, torch.arange(ctx), k, v)
    check(a, window)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("q,ctx,gap", [(q, ctx, gap) for q, ctx in ((6, 200), (60, 500), (300, 400))
                                       for gap in (12, 18, 26, 60)]
                         + [(q, ctx, gap) for q, ctx in ((1, 40), (1, 300), (1, 3000), (2, 2500), (3, 400))
                            for gap in (12, 18)])      # few rows, e4m3: f16 holds 2^-29 of the largest weight
def test_channel_that_the_dominant_key_lacks(dev, q, ctx, gap, fp8):
    """One key has all but e^-gap of a row's weight and zeros in some channels: there the row is what the
    other keys give it."""
    page, hq, hkv = 16, 8, 1
    a = make(dev, [q], [ctx], hq, hkv, page, fp8)
    a["sinks"] = None
    u = torch.randn(64, device=dev).bfloat16()
    a["q"] = u.repeat(q, hq).contiguous()
    k = 0.05 * torch.randn(ctx, hkv, 64, device=dev)
    k[7] = 8.0 * gap * u.float() / u.float().square().sum()
    v = torch.randn(ctx, hkv, 64, device=dev)
    v[7, :, ::5] = 0
    put(a, page, torch.arange(ctx), k, v)
    check(a)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("q,ctx", [(1, 40), (1, 3000), (3, 400), (60, 500)])
def test_keys_of_the_smallest_scale(dev, q, ctx, fp8):
    """Keys of some 2^-121 (scale byte 0) meet queries of 2^120."""
    page = 16
    a = make(dev, [q], [ctx], 16, 2, page, fp8)
    a["q"] = (torch.randn(q, 16 * 64, device=dev) * 2.0 ** 120).bfloat16()
    put(a, page, torch.arange(ctx), torch.randn(ctx, 2, 64, device=dev) * 2.0 ** -121)
    if fp8:
        at = slots_of(a, page)
        assert int(a["k_scales"][at // page, :, at % page].max()) == 0
    check(a)
