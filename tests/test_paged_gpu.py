"""8-bit KV cache pages and attention over pages on the GPU against 64-bit references.

Tolerance of the attention: the output is rounded to bf16 (2^-9 of |o|) and the probabilities are
rounded to bf16 at worst before they meet V (2^-9 of A = sum_j p_j |v_j| / den, the same attention
over |V|); |o| <= A.  fp32 sums, ex2.approx (2^-22) and scores up to a few dozen add less than
2^-12 of A.  So |o - ref| <= (2^-8 + 2^-12) A."""
import math

import pytest
import torch

from agent_factory_3_b200.ops import paged

pytestmark = pytest.mark.gpu
TOL = 2.0 ** -8 + 2.0 ** -12


def make(dev, q_lens, lens, hq, hkv, page, fp8, seed=0, layout="head", spare=3):
    g = torch.Generator(device=dev).manual_seed(seed)
    per = [(n + page - 1) // page for n in lens]
    total = sum(per) + spare
    if fp8:
        if layout == "head":
            k, ks = paged.empty_fp8_pages(total, page, hkv, 64, dev)
            v, vs = paged.empty_fp8_pages(total, page, hkv, 64, dev)
        else:   # token rows, scale bytes token by token
            k, v = (torch.zeros(total, page, hkv, 64, device=dev, dtype=torch.uint8).view(paged.FP8)
                    for _ in range(2))
            ks, vs = (torch.zeros(total, page, hkv, device=dev, dtype=torch.uint8).transpose(1, 2)
                      for _ in range(2))
        rows = torch.randn(total * page, 2 * hkv * 64, device=dev, generator=g)
        rows *= torch.exp(torch.randn(total * page, 1, device=dev, generator=g))
        paged.kv_store_fp8(rows.bfloat16(), 0, hkv * 64,
                           torch.arange(total * page, device=dev, dtype=torch.int32), k, v, ks, vs)
    else:
        shape = (total, page, hkv, 64) if layout == "token" else (total, hkv, page, 64)
        k, v = (torch.randn(shape, device=dev, generator=g).bfloat16() for _ in range(2))
        if layout == "head":
            k, v = k.transpose(1, 2), v.transpose(1, 2)
        ks = vs = None
    table = torch.full((len(lens), max(per + [1]) + 1), -1, dtype=torch.int32)
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = perm[at:at + n]
        at += n
    cu = torch.tensor([0] + list(torch.tensor(q_lens).cumsum(0)), dtype=torch.int32)
    T = int(cu[-1])
    qkv = torch.randn(T, (hq + 2 * hkv) * 64, device=dev, generator=g).bfloat16()
    return dict(q=qkv[:, :hq * 64], k_pages=k, v_pages=v, page_table=table.to(dev),
                seq_lens=torch.tensor(lens, dtype=torch.int32, device=dev), cu_q=cu.to(dev),
                sinks=torch.randn(hq, device=dev, generator=g), hq=hq, hkv=hkv, k_scales=ks,
                v_scales=vs)


def magnitude(v_pages):
    if v_pages.dtype == paged.FP8:
        return (v_pages.view(torch.uint8) & 0x7F).view(paged.FP8)
    return v_pages.abs()


def check(a, window=0, hints=True, **kw):
    if hints:
        n = (a["cu_q"][1:] - a["cu_q"][:-1]).tolist()
        kw.setdefault("max_q_len", max(n + [1]))
        kw.setdefault("max_seq_len", max(a["seq_lens"].tolist() + [1]))
    out = paged.paged_attention(window=window, **a, **kw)
    ref = paged.paged_attention_reference(window=window, dtype=torch.float64, **a)
    mag = paged.paged_attention_reference(window=window, dtype=torch.float64,
                                          **{**a, "v_pages": magnitude(a["v_pages"])})
    assert torch.equal(torch.isnan(out), torch.isnan(ref))
    err = (out.double() - ref).abs()
    bad = (err > TOL * mag) & ~torch.isnan(ref)
    assert not bad.any(), (float((err / mag.clamp(min=1e-300))[bad].max()), bad.nonzero()[:5])
    return out


SHAPES = [
    # new tokens, context, hq, hkv, page
    ([1], [1], 8, 1, 16),
    ([1, 1, 1, 1, 1], [1, 17, 100, 300, 513], 16, 2, 16),
    ([1] * 3, [64, 65, 4097], 64, 8, 64),
    ([1, 1], [31, 2000], 4, 4, 8),            # one query head per KV head
    ([1, 1], [33, 700], 32, 2, 32),           # 16
    ([1, 1], [33, 700], 40, 1, 32),           # 40
    ([1, 1], [129, 257], 6, 2, 5),            # groups of 3, pages of 5
    ([2, 3, 1, 4], [2, 50, 1, 777], 8, 1, 16),
    ([9, 9, 5], [9, 300, 1030], 64, 8, 64),
    ([0, 3, 0, 1], [10, 3, 0, 5], 8, 2, 16),  # sequences without new tokens
    ([17, 130, 1], [17, 400, 50], 16, 2, 64),
    ([300], [300], 8, 1, 48),                 # pages that do not divide a tile
    ([257, 40], [1000, 41], 12, 4, 7),
    ([100, 33], [100, 2049], 10, 2, 128),     # groups of 5
    ([64], [6000], 64, 8, 64),                # few rows, long context
    ([33], [5000], 128, 1, 64),               # the largest group
]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("window", [0, 1, 48, 128])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention(dev, shape, window, fp8):
    check(make(dev, *shape, fp8), window)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("q", [1, 5, 70])
def test_layouts_hints_and_no_sink(dev, q, fp8):
    a = make(dev, [q, q], [q + 40, 1500], 16, 2, 16, fp8, layout="token")
    first = check(a)
    assert torch.equal(first, check(a, hints=False))
    # a hint that is too small changes the split at most
    check(a, max_q_len=1, max_seq_len=1)
    check({**a, "sinks": None})
    # rows of q and out inside wider buffers, 3-d q
    wide = torch.full((2 * q, 16 * 64 + 64), 7.0, device=dev, dtype=torch.bfloat16)
    out = paged.paged_attention(**{**a, "q": a["q"].reshape(2 * q, 16, 64)}, out=wide[:, :16 * 64],
                                max_q_len=q, max_seq_len=1500)
    assert torch.equal(out, first) and (wide[:, 16 * 64:] == 7).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("q", [1, 3, 40])
def test_pages_that_are_not_held(dev, q, fp8):
    """Entries of -1 and past the pool hide their keys; so does a table that ends early."""
    a = make(dev, [q, q], [400, 900], 16, 2, 16, fp8)
    a["page_table"][0, :5] = -1
    a["page_table"][1, 3] = 10 ** 6
    a["page_table"][1, 20:24] = -7
    check(a)
    check(a, window=100)
    check({**a, "page_table": a["page_table"][:, :40].contiguous()})
    a["page_table"][:] = -1
    out = check(a)
    assert (out == 0).all()
    assert (paged.paged_attention(**{**a, "sinks": None}, max_q_len=q, max_seq_len=900) == 0).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("q,window", [(1, 0), (1, 40), (4, 0), (4, 40), (60, 0), (60, 40), (300, 100)])
def test_rows_before_the_first_key(dev, q, window, fp8):
    """More new tokens than the length says: the first rows stand before key 0 and see nothing."""
    a = make(dev, [q, q], [max(1, q - 2), 0], 8, 1, 16, fp8)
    out = check(a, window)
    assert (out[q:] == 0).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("q", [1, 4, 60, 200])
def test_nan_and_inf_in_masked_places(dev, q, fp8):
    """Whatever stands where a row does not look -- the rest of the last page, other pages, keys
    before the window, later tokens of the chunk -- leaves the row's result as it was."""
    L, window, page = 700, 90, 16
    a = make(dev, [q], [L], 16, 2, page, fp8)
    want = check(a, window)
    used = a["page_table"][0, :(L + page - 1) // page].long()
    slot = (used[:, None] * page + torch.arange(page, device=dev)).reshape(-1)
    hidden = torch.ones(a["k_pages"].shape[0] * page, dtype=torch.bool, device=dev)
    hidden[slot[max(0, L - q - window + 1):L]] = False
    at = hidden.nonzero().squeeze(-1)

    def poison(at, value):
        p, o = at // page, at % page
        for pages in (a["k_pages"], a["v_pages"]):
            if fp8:
                pages.view(torch.uint8)[p, o] = 0x7F
            else:
                pages[p, o] = value
        if fp8:
            a["k_scales"][p, :, o] = 255
            a["v_scales"][p, :, o] = 254
    poison(at, math.inf)
    assert torch.equal(want, check(a, window))
    poison(at, math.nan)
    assert torch.equal(want, check(a, window))
    if q > 1:      # the last token is broken: rows before it do not see it
        poison(slot[L - 1:L], math.nan)
        out = check(a, window)
        assert torch.equal(out[:-1], want[:-1]) and torch.isnan(out[-1]).all()


@pytest.mark.parametrize("q", [1, 3, 60])
def test_infinite_value_of_a_visible_key(dev, q):
    a = make(dev, [q], [200], 8, 1, 16, False)
    page, off = int(a["page_table"][0, 199 // 16]), 199 % 16
    a["v_pages"][page, off, 0, 5] = math.inf
    out = paged.paged_attention(**a, max_q_len=q, max_seq_len=200).view(q, 8, 64)
    assert torch.isinf(out[-1, :, 5]).all()
    assert torch.isfinite(out[:-1]).all()
    keep = [d for d in range(64) if d != 5]
    assert torch.isfinite(out[-1][:, keep]).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("q", [1, 3, 60])
def test_large_and_uneven_scores(dev, q, fp8):
    """Scores in the hundreds, rows dominated by the sink, token magnitudes over 2^12 apart."""
    a = make(dev, [q], [1200], 16, 2, 16, fp8)
    check({**a, "q": a["q"] * 40})
    check({**a, "sinks": a["sinks"] + 60})
    check({**a, "q": torch.zeros_like(a["q"])})
    n = a["k_pages"].shape[0] * 16
    mag = torch.exp2(torch.randint(-6, 7, (n, 1), device=dev).float())
    rows = (torch.randn(n, 2 * 2 * 64, device=dev) * mag).bfloat16()
    slots = torch.arange(n, device=dev, dtype=torch.int32)
    if fp8:
        paged.kv_store_fp8(rows, 0, 128, slots, a["k_pages"], a["v_pages"], a["k_scales"], a["v_scales"])
    else:
        a["v_pages"][:] = rows[:, 128:].view(-1, 16, 2, 64)
    check(a)
    check({**a, "q": a["q"] * 1e-3})


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("q", [1, 4, 150])
def test_offsets_past_32_bits(dev, q, fp8):
    """Pages beyond 4 GiB of a pool."""
    hkv, page = 8, 64
    a = make(dev, [q], [300], 64, hkv, page, fp8)
    n = a["k_pages"].shape[0]
    big = 5 * 2 ** 30 // (page * hkv * 64 * (1 if fp8 else 2))
    for name in ("k_pages", "v_pages"):
        small = a[name]
        if fp8:
            pool = torch.empty(big, hkv, page, 64, device=dev, dtype=torch.uint8)
            pool[big - n:] = small.view(torch.uint8).permute(0, 2, 1, 3)
            a[name] = pool.view(paged.FP8).permute(0, 2, 1, 3)
        else:
            pool = torch.empty(big, page, hkv, 64, device=dev, dtype=torch.bfloat16)
            pool[big - n:] = small
            a[name] = pool
    if fp8:
        for name in ("k_scales", "v_scales"):
            pool = torch.zeros(big, hkv, page, device=dev, dtype=torch.uint8)
            pool[big - n:] = a[name]
            a[name] = pool
    a["page_table"] = torch.where(a["page_table"] >= 0, a["page_table"] + (big - n), a["page_table"])
    check(a)


@pytest.mark.parametrize("fp8", [False, True])
def test_other_stream_and_repeat(dev, fp8):
    a = make(dev, [1, 1, 20], [900, 33, 700], 16, 2, 16, fp8)
    want = paged.paged_attention(**a, max_q_len=20, max_seq_len=900)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = paged.paged_attention(**a, max_q_len=20, max_seq_len=900)
    s.synchronize()
    assert torch.equal(want, got)      # same bits: every sum has a fixed order


def test_capture(dev):
    """Lengths and tables are read on the device: a captured call follows them."""
    a = make(dev, [1, 1], [500, 90], 16, 2, 16, True)
    out = torch.empty(2, 16 * 64, device=dev, dtype=torch.bfloat16)
    paged.paged_attention(**a, max_q_len=1, max_seq_len=512, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        paged.paged_attention(**a, max_q_len=1, max_seq_len=512, out=out)
    a["seq_lens"].copy_(torch.tensor([77, 91], device=dev))
    g.replay()
    want = paged.paged_attention(**a, max_q_len=1, max_seq_len=512)
    assert torch.equal(out, want)


def test_empty_calls(dev):
    a = make(dev, [1], [5], 8, 1, 16, True)
    out = paged.paged_attention(**{**a, "q": a["q"][:0], "page_table": a["page_table"][:0],
                                   "seq_lens": a["seq_lens"][:0], "cu_q": a["cu_q"][:1]})
    assert out.shape == (0, 512)
    none = torch.empty(0, dtype=torch.int32, device=dev)
    paged.kv_store_fp8(a["q"][:0], 0, 64, none, a["k_pages"], a["v_pages"], a["k_scales"], a["v_scales"])
    paged.kv_gather_fp8(a["q"][:0], 0, 64, none, a["k_pages"], a["v_pages"], a["k_scales"], a["v_scales"])


# --------------------------------------------------------------------- store and gather
@pytest.mark.parametrize("layout", ["head", "token"])
@pytest.mark.parametrize("n,hkv,d,page", [(1, 1, 64, 16), (8, 8, 64, 64), (1003, 3, 64, 5),
                                          (300, 2, 128, 16), (77, 5, 32, 8), (33, 1, 256, 4),
                                          (19, 7, 8, 16)])
def test_store_and_gather(dev, n, hkv, d, page, layout):
    g = torch.Generator().manual_seed(n)
    pages = n // page + 3
    x = torch.randn(n, (2 + 2 * hkv) * d, generator=g) * torch.exp2(
        torch.randint(-30, 30, (n, 1), generator=g).float())
    x = x.bfloat16()
    x[0] = 0
    x[n // 2, ::3] = math.nan
    x[n // 3, 1::5] = -math.inf
    x[n - 1] *= 2.0 ** 100
    if n > 8:
        x[4] = 3.3895e38          # near the largest bf16: code 240 at the largest exponent
        x[5] = 1e-40              # denormals
        x[6] = 448 * 2.0 ** 5     # exactly at a step of the exponent
        x[7] = 449 * 2.0 ** 5
    slots = torch.randperm(pages * page, generator=g)[:n].to(torch.int32)
    slots[n // 2:n // 2 + 1] = -1 if n > 8 else slots[n // 2]
    slots[n // 4:n // 4 + 1] = pages * page if n > 8 else slots[n // 4]

    def mk(where):
        if layout == "head":
            return (*paged.empty_fp8_pages(pages, page, hkv, d, where),
                    *paged.empty_fp8_pages(pages, page, hkv, d, where))
        codes = [torch.zeros(pages, page, hkv, d, dtype=torch.uint8, device=where).view(paged.FP8)
                 for _ in range(2)]
        scales = [torch.zeros(pages, page, hkv, dtype=torch.uint8, device=where).transpose(1, 2)
                  for _ in range(2)]
        return codes[0], scales[0], codes[1], scales[1]
    ck, cks, cv, cvs = mk("cpu")
    gk, gks, gv, gvs = mk(dev)
    off = 2 * d
    paged.kv_store_fp8(x, off, off + hkv * d, slots, ck, cv, cks, cvs)
    paged.kv_store_fp8(x.to(dev), off, off + hkv * d, slots.to(dev), gk, gv, gks, gvs)
    for c, gpu in ((ck, gk), (cv, gv)):
        a, b = c.float(), gpu.cpu().float()
        assert torch.equal(torch.isnan(a), torch.isnan(b))
        assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))
    assert torch.equal(cks, gks.cpu()) and torch.equal(cvs, gvs.cpu())
    back_c = torch.full_like(x, 3.0)
    back_g = back_c.to(dev)
    paged.kv_gather_fp8(back_c, off, off + hkv * d, slots, ck, cv, cks, cvs)
    paged.kv_gather_fp8(back_g, off, off + hkv * d, slots.to(dev), gk, gv, gks, gvs)
    a, b = back_c.float(), back_g.cpu().float()
    assert torch.equal(torch.isnan(a), torch.isnan(b))
    assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))
    assert (back_g[:, :off] == 3).all()


def test_refusals(dev):
    a = make(dev, [1, 1], [40, 50], 16, 2, 16, True)
    b = make(dev, [1, 1], [40, 50], 16, 2, 16, False)

    def no(match, base=a, **kw):
        with pytest.raises(RuntimeError, match=match):
            paged.paged_attention(**{**base, **kw}, max_q_len=1, max_seq_len=50)
    no("scales", k_scales=None)
    no("scales", base=b, k_scales=a["k_scales"], v_scales=a["v_scales"])
    no("scales must be", k_scales=a["k_scales"].float(), v_scales=a["v_scales"])
    no("scales must be", k_scales=a["k_scales"][:, :1], v_scales=a["v_scales"][:, :1])
    no("Hkv", hkv=3)
    no("q must be", q=a["q"][:, :64])
    no("bfloat16", q=a["q"].float())
    no("seq_lens must be", cu_q=a["cu_q"][:2])
    no("int32", seq_lens=a["seq_lens"].long())
    no("int32", page_table=a["page_table"].cpu())
    no("page_table must be", page_table=a["page_table"][:1])
    no("sinks", sinks=a["sinks"][:3].contiguous())
    no("window", window=-1)
    no("one type", base=b, v_pages=b["v_pages"].half())
    no("bfloat16 or float8", base=b, k_pages=b["k_pages"].half(), v_pages=b["v_pages"].half())
    no("same strides", base=b, v_pages=b["v_pages"].contiguous(), k_pages=b["k_pages"])
    no("aligned", q=torch.empty(2, 16 * 64 + 1, device=dev, dtype=torch.bfloat16)[:, 1:])
    no("out must be", out=torch.empty(1, 1024, device=dev, dtype=torch.bfloat16))
    wide = make(dev, [1], [40], 129, 1, 16, True)
    no("128 query heads", base=wide)
    d128 = {**b, "k_pages": torch.zeros(4, 16, 2, 128, device=dev, dtype=torch.bfloat16),
            "v_pages": torch.zeros(4, 16, 2, 128, device=dev, dtype=torch.bfloat16)}
    no("head_dim 64", base=d128, q=torch.zeros(2, 16 * 128, device=dev, dtype=torch.bfloat16))
    slots = torch.zeros(2, device=dev, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="float8_e4m3fn"):
        paged.kv_store_fp8(a["q"], 0, 128, slots, b["k_pages"], b["v_pages"], None, None)
    with pytest.raises(RuntimeError, match="past the row"):
        paged.kv_store_fp8(a["q"], 0, 1000, slots, a["k_pages"], a["v_pages"], a["k_scales"], a["v_scales"])
    with pytest.raises(RuntimeError, match="more slots"):
        paged.kv_gather_fp8(a["q"].clone(), 0, 128, torch.zeros(3, device=dev, dtype=torch.int32),
                            a["k_pages"], a["v_pages"], a["k_scales"], a["v_scales"])
    with pytest.raises(RuntimeError, match="aligned"):
        paged.kv_store_fp8(a["q"], 4, 128, slots, a["k_pages"], a["v_pages"], a["k_scales"], a["v_scales"])
