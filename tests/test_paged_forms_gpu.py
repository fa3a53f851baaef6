"""Attention over cache pages on the GPU: the forms of the kernels (tile widths, short and long parts,
one page or several to a block, several tokens), values of a wide range, and the precision of P.

Tolerance of the forms: that of test_paged_gpu.check.  Tolerance of test_precision_of_p: the output is
rounded to bf16 (2^-8 of |ref| at most), each probability is held in 11 bits at least (2^-11 of A, the same
attention over |V|), and fp32 sums, ex2.approx and scores of a few dozen add less than 2^-13 of A."""
import math

import pytest
import torch

from test_paged_gpu import check, magnitude, make
from test_paged_values_gpu import put, slots_of

from agent_factory_3_b200.ops import paged

FORMS = [
    # new tokens, context, hq, hkv, page
    ([5], [2600], 64, 8, 64),                 # long parts, several tokens: 16 rows and the rest
    ([2, 3, 1], [2200, 5000, 2500], 16, 2, 48),
    ([5], [3001], 8, 1, 5),                   # pages inside a block
    ([1, 1], [4097, 2049], 64, 8, 16),
    ([1, 1], [3000, 2500], 8, 1, 7),
    ([1], [2100], 4, 4, 32),                  # one row a tile
    ([4] * 8, [700, 300, 650, 4, 699, 257, 256, 512], 64, 8, 16),   # long parts by the number of items
    ([4] * 8, [700, 300, 650, 4, 699, 257, 256, 512], 64, 8, 64),
    ([1], [3000], 20, 1, 64),                 # groups of 17 to 32: tiles of 32 rows
    ([1], [3000], 32, 1, 48),
    ([1, 1], [100, 33], 64, 2, 16),
    ([1, 1], [100, 257], 24, 1, 64),
    ([1, 1, 1], [90, 5, 2500], 34, 2, 8),
    ([6, 7], [3000, 900], 8, 1, 48),          # 48 and 56 rows: the kernel of many rows
    ([9, 2], [4000, 4100], 64, 8, 64),
    ([129], [6000], 24, 1, 16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("window", [0, 100, 2300])
@pytest.mark.parametrize("shape", FORMS)
def test_forms(dev, shape, window, fp8):
    check(make(dev, *shape, fp8), window)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("page", [64, 48])
@pytest.mark.parametrize("q,window", [(1, 0), (1, 2400), (3, 0), (3, 2400), (5, 2400)])
def test_masked_and_broken_values_in_long_parts(dev, q, window, page, fp8):
    """Parts of more than 2048 keys: what a row does not see leaves it as it was, a value that is not
    finite reaches the rows that see it."""
    L = 3001
    a = make(dev, [q], [L], 16, 2, page, fp8)
    want = check(a, window)
    at = slots_of(a, page)
    hidden = torch.ones(a["k_pages"].shape[0] * page, dtype=torch.bool, device=dev)
    hidden[at[(max(0, L - q - window + 1) if window else 0):]] = False
    bad = hidden.nonzero().squeeze(-1)
    for pages in (a["k_pages"], a["v_pages"]):
        if fp8:
            pages.view(torch.uint8)[bad // page, bad % page] = 0x7F
        else:
            pages[bad // page, bad % page] = math.nan
    assert torch.equal(want, check(a, window))
    for key in (L - 1, L - 2400 + 1):         # the last token; with the window, seen by some rows only
        b = int(at[key])
        if fp8:
            a["v_pages"].view(torch.uint8)[b // page, b % page, :, 3] = 0x7F
        else:
            a["v_pages"][b // page, b % page, :, 3] = math.nan
        check(a, window)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("bits", [13, 16, 24, 60])
@pytest.mark.parametrize("shape", [([1], [300], 16, 2, 16), ([1], [3000], 8, 1, 64), ([3], [400], 8, 1, 16),
                                   ([1], [300], 32, 1, 16), ([60], [500], 16, 2, 16), ([300], [400], 8, 1, 48)])
def test_tokens_of_a_wide_range(dev, shape, bits, fp8):
    """Token magnitudes spread over 2^bits, of V and, less, of K."""
    q_lens, lens, hq, hkv, page = shape
    a = make(dev, *shape, fp8)
    n = lens[0]
    g = torch.Generator(device=dev).manual_seed(bits)

    def rows(b, top):
        e = torch.rand(n, 1, 1, device=dev, generator=g) * b
        return torch.randn(n, hkv, 64, device=dev, generator=g) * torch.exp2(top - e)
    put(a, page, torch.arange(n), rows(min(bits, 24), 0), rows(bits, bits / 2))
    check(a)
    check(a, window=130)


# --------------------------------------------------------------------- precision of P
def near_pairs(dev, q, ctx, hq, hkv, fp8):
    """Values that nearly cancel: each key of odd number has the negative of the value before it and
    nearly its weight; one pair carries half of the weight."""
    page = 16
    a = make(dev, [q], [ctx], hq, hkv, page, fp8)
    a["sinks"] = None
    g = torch.Generator(device=dev).manual_seed(q + ctx)
    u = torch.randn(64, device=dev, generator=g)
    u *= 8 / u.norm()
    spread = 1 + 0.05 * torch.randn(q, hq, 1, device=dev, generator=g)
    a["q"] = (u * spread + 0.3 * torch.randn(q, hq, 64, device=dev, generator=g)).bfloat16().view(q, -1)
    k = 0.1 * torch.randn(ctx, hkv, 64, device=dev, generator=g)
    k[:2] += u * (math.log(ctx) / 8)              # scores of log(ctx)
    v = torch.randn((ctx + 1) // 2, hkv, 64, device=dev, generator=g)
    v = torch.stack([v, -v], 1).reshape(-1, hkv, 64)[:ctx]
    put(a, page, torch.arange(ctx), k, v)
    return a


def close(out, ref, mag):
    return (out.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + (2.0 ** -11 + 2.0 ** -13) * mag


PAIRS = [(1, 2, 64, 8), (1, 40, 64, 8), (1, 3000, 64, 8), (1, 40, 32, 1), (5, 60, 64, 8), (5, 3000, 8, 1),
         (40, 60, 16, 2), (200, 300, 64, 8), (40, 5000, 8, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("q,ctx,hq,hkv", PAIRS)
def test_precision_of_p(dev, q, ctx, hq, hkv, fp8):
    a = near_pairs(dev, q, ctx, hq, hkv, fp8)
    out = paged.paged_attention(**a, max_q_len=q, max_seq_len=ctx)
    ref = paged.paged_attention_reference(dtype=torch.float64, **a)
    mag = paged.paged_attention_reference(dtype=torch.float64, **{**a, "v_pages": magnitude(a["v_pages"])})
    assert close(out, ref, mag).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("q,ctx,hq,hkv", PAIRS[:2] + PAIRS[4:5])
def test_that_one_bf16_p_would_be_seen(q, ctx, hq, hkv, fp8):
    """The same bound refuses probabilities rounded to one bf16 (computed key by key on the CPU)."""
    a = near_pairs("cpu", q, ctx, hq, hkv, fp8)
    ref = paged.paged_attention_reference(dtype=torch.float64, **a)
    mag = paged.paged_attention_reference(dtype=torch.float64, **{**a, "v_pages": magnitude(a["v_pages"])})
    at = slots_of(a, 16)
    k, v = (paged.dequantize_rows_reference(p.view(torch.uint8)[at // 16, at % 16].view(paged.FP8), s[at // 16, :, at % 16])
            if s is not None else p[at // 16, at % 16].float()
            for p, s in ((a["k_pages"], a["k_scales"]), (a["v_pages"], a["v_scales"])))
    s = torch.einsum("thd,khd->thk", a["q"].view(q, hq, 64).float(), k.repeat_interleave(hq // hkv, 1)) / 8
    seen = torch.arange(ctx)[None, :] <= ctx - q + torch.arange(q)[:, None]
    s = s.masked_fill(~seen[:, None, :], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))

    def result(p16):
        o = torch.einsum("thk,khd->thd", p16, v.repeat_interleave(hq // hkv, 1)) / p.sum(-1, keepdim=True)
        return o.reshape(q, -1).bfloat16()
    assert close(result(p.half().float()), ref, mag).all()
    assert not close(result(p.bfloat16().float()), ref, mag).all()
