"""Measured cases of the 8-bit KV cache operators and of the attention over cache pages.

Three operators of the rollout engine: writing new keys and values into e4m3 pages
(``store``), reading cached rows back (``gather``), and attention of each sequence's new
tokens over its pages (``attention``: one token in decoding, a few in a speculative verify,
thousands in a prefill chunk; pages in bf16 or in e4m3 with one power-of-two scale per token
and KV head).  Head dim 64 and 8 query heads per KV head are gpt-oss; the other head layouts
are its tensor-parallel slices and the small models of the tests.
"""
import math

import torch

own = False

D = 64


def listed():
    attn = dict(op="attention", hq=64, hkv=8, page=64, window=0)
    return [
        # decode step of 8 requests: a handful of rows, launch latency
        dict(name="store 8 tokens", op="store", n=8, hq=64, hkv=8, page=64, pages=64),
        # odd number of rows, KV heads of one tensor-parallel rank of two
        dict(name="store 1003 tokens", op="store", n=1003, hq=32, hkv=4, page=16, pages=256),
        # the engine's largest prefill step
        dict(name="store 16384 tokens", op="store", n=16384, hq=64, hkv=8, page=64, pages=1024),
        # a cached prefix read back for a short prompt
        dict(name="gather 777 rows", op="gather", n=777, hq=64, hkv=8, page=64, pages=64),
        # the model's longest context read back
        dict(name="gather 131072 rows", op="gather", n=131072, hq=64, hkv=8, page=64, pages=2304),
        # one request decoding on its own: latency
        dict(attn, name="decode 1 x 1025", batch=1, q=1, context=1025, ragged=False, fp8=True),
        # the steady decode window of 128 trajectories around 7k tokens
        dict(attn, name="decode 128 x 7k e4m3", batch=128, q=1, context=14000, ragged=True, fp8=True),
        # a sliding-window layer of the same step, bf16 pages
        dict(attn, name="decode 128 window bf16", batch=128, q=1, context=14000, ragged=True,
             fp8=False, window=128),
        # two requests at the longest context, bf16 pages: work split over a long axis
        dict(attn, name="decode 2 x 131072 bf16", batch=2, q=1, context=131072, ragged=False,
             fp8=False),
        # speculative verify: the last token and 8 drafts of 64 requests
        dict(attn, name="verify 64 x 9 e4m3", batch=64, q=9, context=4200, ragged=True, fp8=True),
        # ragged prefill chunks on cached prefixes, bf16 pages
        dict(attn, name="chunk 5 x 1000 bf16", batch=5, q=1000, context=5003, ragged=True,
             fp8=False),
        # one long chunk on a long cached prefix
        dict(attn, name="chunk 4096 on 12288 e4m3", batch=1, q=4096, context=16384, ragged=False,
             fp8=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "gather", "attention", "attention", "attention", "attention"])
    hq, hkv = rng.choice([(64, 8), (64, 8), (32, 4), (16, 2), (8, 1), (8, 2), (4, 2)])
    page = rng.choice([8, 16, 32, 64, 64, 128])
    if op in ("store", "gather"):
        n = _log_int(rng, 1, 16384 if op == "store" else 131072)
        return dict(op=op, n=n, hq=hq, hkv=hkv, page=page, pages=-(-n // page) + rng.randrange(1, 64))
    kind = rng.choice(["decode", "decode", "verify", "chunk", "chunk"])
    if kind == "decode":
        q, batch, context = 1, _log_int(rng, 1, 256), _log_int(rng, 1, 65536)
        context = max(1, min(context, 2_000_000 * 8 // (batch * hkv)))
    elif kind == "verify":
        q, batch, context = rng.randrange(2, 18), _log_int(rng, 1, 128), _log_int(rng, 32, 16384)
        context = max(q, min(context, 300_000 * 64 * 17 // (batch * hq * q)))
    else:
        q, batch, context = _log_int(rng, 18, 4096), rng.randrange(1, 9), _log_int(rng, 32, 32768)
        context = max(q, min(context, 4096 * 16384 * 64 // (batch * hq * q)))
        q = min(q, context)
    return dict(op="attention", hq=hq, hkv=hkv, page=page, batch=batch, q=q, context=context,
                ragged=rng.random() < 0.7, fp8=rng.random() < 0.6,
                window=rng.choice([0, 0, 128, rng.randrange(1, 700)]))


def _lengths(case):
    """(new tokens, context) of each sequence, the same for every seed.  Ragged: spread evenly
    up to the longest, which comes first."""
    batch, q, context = case["batch"], case["q"], case["context"]
    if not case["ragged"]:
        return torch.full((batch,), q), torch.full((batch,), context)
    gen = torch.Generator()
    gen.manual_seed(batch * 1009 + context)
    q_lens = (1 + (q - 1) * torch.rand(batch, generator=gen)).long().clamp(1, q)
    lens = (context * (0.05 + 0.95 * torch.rand(batch, generator=gen))).long()
    q_lens[0], lens[0] = q, context
    return q_lens, torch.maximum(lens, q_lens)


def _tokens(n, heads, gen, spread):
    """bf16 rows [n, heads, D] as projections give them: the magnitude varies from token to
    token (by ``spread``, in natural log) and a few channels are larger."""
    x = torch.randn(n, heads, D, device="cuda", generator=gen)
    x *= torch.exp(spread * torch.randn(n, 1, 1, device="cuda", generator=gen))
    x[:, :, ::23] *= 2.5
    return x.to(torch.bfloat16)


def _quantise(x):
    """(e4m3 codes, e8m0 scale bytes) of rows [..., D]: 2^e is the smallest power of two that
    brings the largest finite magnitude to 448 or below."""
    f = x.float()
    finite = torch.isfinite(f)
    amax = torch.where(finite, f.abs(), torch.zeros_like(f)).amax(-1, keepdim=True)
    frac, exp = torch.frexp(amax)
    e = torch.where(amax > 0, exp - 9 + (frac > 0.875).int(), torch.full_like(exp, -127))
    e = e.clamp(-127, 120)
    inv = ((127 - e) << 23).view(torch.float32)
    limit = torch.where(e == 120, 240.0, 448.0)
    y = torch.where(finite, torch.minimum(torch.maximum(f * inv, -limit), limit),
                    torch.full_like(f, math.nan))
    return y.to(torch.float8_e4m3fn), (e + 127).to(torch.uint8).squeeze(-1)


def _values(codes, scales):
    """fp32 values of e4m3 rows [..., D] (as bytes) with e8m0 scale bytes [...]."""
    return torch.ldexp(codes.view(torch.float8_e4m3fn).float(), scales.int().unsqueeze(-1) - 127)


def _pool(case, pages, gen, fp8, spread):
    """One layer's pages (and scale bytes) full of tokens: e4m3 pages keep each KV head's rows
    together in memory, bf16 pages each token's heads."""
    page, hkv = case["page"], case["hkv"]
    x = _tokens(pages * page, hkv, gen, spread).view(pages, page, hkv, D)
    if not fp8:
        return x, None
    codes, scales = _quantise(x)
    codes = codes.view(torch.uint8).permute(0, 2, 1, 3).contiguous().view(torch.float8_e4m3fn)
    return codes.permute(0, 2, 1, 3), scales.permute(0, 2, 1).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    hq, hkv, page = case["hq"], case["hkv"], case["page"]
    width = (hq + 2 * hkv) * D
    s = {"op": case["op"], "hq": hq, "hkv": hkv, "k_off": hq * D, "v_off": (hq + hkv) * D}
    if case["op"] in ("store", "gather"):
        n, pages = case["n"], case["pages"]
        s["k"], s["ks"] = _pool(case, pages, gen, True, 0.5)
        s["v"], s["vs"] = _pool(case, pages, gen, True, 0.7)
        s["slots"] = torch.randperm(pages * page, device="cuda", generator=gen)[:n].to(torch.int32)
        s["qkv"] = _tokens(n, hq + 2 * hkv, gen, 0.5).view(n, width)
        return s
    q_lens, lens = _lengths(case)
    batch = case["batch"]
    per_seq = (lens + page - 1) // page
    total = int(per_seq.sum())
    s["k"], s["ks"] = _pool(case, total + 3, gen, case["fp8"], 0.25)
    s["v"], s["vs"] = _pool(case, total + 3, gen, case["fp8"], 0.5)
    perm = torch.randperm(total + 3, device="cuda", generator=gen)[:total].to(torch.int32)
    table = torch.zeros(batch, int(per_seq.max()), dtype=torch.int32, device="cuda")
    held = torch.arange(table.shape[1])[None, :] < per_seq[:, None]
    table[held.cuda()] = perm
    cu = torch.zeros(batch + 1, dtype=torch.int32)
    cu[1:] = q_lens.cumsum(0)
    rows = _tokens(int(cu[-1]), hq + 2 * hkv, gen, 0.25).view(int(cu[-1]), width)
    s.update(q=rows[:, :hq * D], table=table, lens=lens.to(torch.int32).cuda(), cu=cu.cuda(),
             sinks=torch.randn(hq, device="cuda", generator=gen), window=case["window"],
             max_q=int(q_lens.max()), max_len=int(lens.max()))
    return s


def _plain_store(s):
    for_k, for_v = s["k"].view(torch.uint8), s["v"].view(torch.uint8)
    page, hkv = s["k"].shape[1], s["hkv"]
    slots = s["slots"].long()
    n = slots.numel()
    at, off = slots // page, slots % page
    codes, scales = _quantise(s["qkv"][:, s["k_off"]:s["k_off"] + hkv * D].reshape(n, hkv, D))
    for_k[at, off] = codes.view(torch.uint8)
    s["ks"][at, :, off] = scales
    codes, scales = _quantise(s["qkv"][:, s["v_off"]:s["v_off"] + hkv * D].reshape(n, hkv, D))
    for_v[at, off] = codes.view(torch.uint8)
    s["vs"][at, :, off] = scales


def _plain_gather(s):
    page, hkv = s["k"].shape[1], s["hkv"]
    slots = s["slots"].long()
    at, off = slots // page, slots % page
    k = _values(s["k"].view(torch.uint8)[at, off], s["ks"][at, :, off])
    v = _values(s["v"].view(torch.uint8)[at, off], s["vs"][at, :, off])
    s["qkv"][:, s["k_off"]:s["k_off"] + hkv * D] = k.reshape(-1, hkv * D).to(torch.bfloat16)
    s["qkv"][:, s["v_off"]:s["v_off"] + hkv * D] = v.reshape(-1, hkv * D).to(torch.bfloat16)


def _plain_attention(s):
    hq, hkv = s["hq"], s["hkv"]
    group = hq // hkv
    page = s["k"].shape[1]
    cu, lens = s["cu"].long(), s["lens"].long()
    batch, max_q, max_len = lens.numel(), s["max_q"], s["max_len"]
    dev = lens.device
    j = torch.arange(max_len, device=dev)
    at, off = s["table"][:, j // page].long(), (j % page)[None, :]
    if s["ks"] is None:
        k, v = s["k"][at, off].float(), s["v"][at, off].float()
    else:
        k = _values(s["k"].view(torch.uint8)[at, off], s["ks"][at, :, off])
        v = _values(s["v"].view(torch.uint8)[at, off], s["vs"][at, :, off])
    k, v = k.permute(0, 2, 3, 1), v.transpose(1, 2)             # [B, Hkv, D, L], [B, Hkv, L, D]
    i = torch.arange(max_q, device=dev)
    q_lens = cu[1:] - cu[:-1]
    row = (cu[:-1, None] + i[None, :]).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[row].view(batch, max_q, hkv, group, D)
    q = q.permute(0, 2, 1, 3, 4).reshape(batch, hkv, max_q * group, D)
    pos = (lens - q_lens)[:, None] + i[None, :]                  # [B, max_q]
    seen = j[None, None, :] <= pos[:, :, None]
    if s["window"]:
        seen &= pos[:, :, None] - j[None, None, :] < s["window"]
    sc = (q @ k).view(batch, hkv, max_q, group, max_len)
    sc *= 1.0 / math.sqrt(D)
    sc.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    sink = s["sinks"].view(1, hkv, 1, group, 1)
    top = torch.maximum(sc.amax(-1, keepdim=True), sink)
    sc -= top
    sc.exp_()
    den = sc.sum(-1, keepdim=True) + torch.exp(sink - top)
    o = (sc.view(batch, hkv, max_q * group, max_len) @ v).view(batch, hkv, max_q, group, D) / den
    o = o.permute(0, 2, 1, 3, 4).reshape(batch, max_q, hq * D)
    return o[i[None, :] < q_lens[:, None]].to(torch.bfloat16)


def run(s):
    if own:
        from agent_factory_3_b200.ops import paged
    if s["op"] == "store":
        if own:
            paged.kv_store_fp8(s["qkv"], s["k_off"], s["v_off"], s["slots"], s["k"], s["v"],
                               s["ks"], s["vs"])
        else:
            _plain_store(s)
        return {"k": s["k"], "v": s["v"], "k_scales": s["ks"], "v_scales": s["vs"]}
    if s["op"] == "gather":
        if own:
            paged.kv_gather_fp8(s["qkv"], s["k_off"], s["v_off"], s["slots"], s["k"], s["v"],
                                s["ks"], s["vs"])
        else:
            _plain_gather(s)
        return s["qkv"]
    if own:
        return paged.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], s["cu"],
                                     s["sinks"], s["hq"], s["hkv"], s["window"], k_scales=s["ks"],
                                     v_scales=s["vs"], max_q_len=s["max_q"],
                                     max_seq_len=s["max_len"])
    return _plain_attention(s)


def work(case):
    hq, hkv = case["hq"], case["hkv"]
    if case["op"] in ("store", "gather"):
        # a bf16 row of K and V on one side, codes and scale bytes on the other, the slot ids
        return {"bytes": case["n"] * (2 * hkv * (2 * D + D + 1) + 4), "flops": 0}
    q_lens, lens = (x.double() for x in _lengths(case))
    first = lens - q_lens                                    # position of the first row
    if case["window"]:
        w = float(case["window"])
        short = torch.minimum((w - 1 - first).clamp(min=0), q_lens)   # rows that see fewer keys
        pairs = short * (2 * first + 1 + short) / 2 + (q_lens - short) * w
        keys = torch.minimum(lens, q_lens + w - 1)
    else:
        pairs = q_lens * (first + 1 + lens) / 2
        keys = lens
    per_key = hkv * (2 * (D + 1) if case["fp8"] else 4 * D)
    return {"bytes": float(keys.sum()) * per_key + 4 * float(q_lens.sum()) * hq * D,
            "flops": 4.0 * D * hq * float(pairs.sum())}


def exact(case, seed):
    s = prepare(case, seed)
    hq, hkv, page = case["hq"], case["hkv"], case["page"]

    def power(e):                                            # 2^e exactly, e >= -1022
        return ((e.long() + 1023) << 52).view(torch.float64)

    def values(codes, scales, at, off):
        c = codes.view(torch.uint8)[at, off].to(torch.int32)                  # [n, Hkv, D]
        e, m = (c >> 3) & 15, (c & 7).double()
        mag = torch.where(e > 0, (8 + m) * power(e - 10), m * 2.0 ** -9)
        mag = torch.where((c & 127) == 127, torch.full_like(mag, math.nan), mag)
        sign = 1.0 - 2.0 * (c >> 7).double()
        return sign * mag * power(scales[at, :, off].int() - 127).unsqueeze(-1)

    if case["op"] == "store":
        slots = s["slots"].long()
        out = {}
        for name, byte, col in (("k", "ks", s["k_off"]), ("v", "vs", s["v_off"])):
            x = s["qkv"][:, col:col + hkv * D].reshape(-1, hkv, D).double()
            a = x.abs().amax(-1)
            e = torch.full_like(a, -127.0)
            for p in range(-126, 121):                       # smallest e with a <= 448 * 2^e
                e = torch.where(a > 448.0 * 2.0 ** (p - 1), torch.full_like(e, float(p)), e)
            y = x * power(-e).unsqueeze(-1)
            y = torch.where((e == 120).unsqueeze(-1), y.clamp(-240, 240), y.clamp(-448, 448))
            # e4m3: steps of 2^(floor(log2 |y|) - 3), 2^-9 at the least; ties to the even step
            step = power(torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4)
            y = torch.round(y / step) * step
            pages = s[name].double()
            pages[slots // page, slots % page] = y
            scales = s[byte].clone()
            scales[slots // page, :, slots % page] = (e + 127).to(torch.uint8)
            out[name], out[name + "_scales"] = pages, scales
        return out
    if case["op"] == "gather":
        slots = s["slots"].long()
        out = s["qkv"].double()
        for name, byte, col in (("k", "ks", s["k_off"]), ("v", "vs", s["v_off"])):
            x = values(s[name], s[byte], slots // page, slots % page)
            out[:, col:col + hkv * D] = x.reshape(-1, hkv * D)
        return out
    group = hq // hkv
    cu, lens = s["cu"].tolist(), s["lens"].tolist()
    out = torch.empty(cu[-1], hq, D, dtype=torch.float64, device="cuda")
    for b in range(len(lens)):
        n, first = lens[b], lens[b] - (cu[b + 1] - cu[b])
        j = torch.arange(n, device="cuda")
        at, off = s["table"][b, j // page].long(), j % page
        if s["ks"] is None:
            k, v = s["k"][at, off].double(), s["v"][at, off].double()
        else:
            k, v = values(s["k"], s["ks"], at, off), values(s["v"], s["vs"], at, off)
        for r0 in range(cu[b], cu[b + 1], 512):
            r1 = min(r0 + 512, cu[b + 1])
            pos = first + torch.arange(r0 - cu[b], r1 - cu[b], device="cuda")
            seen = j[None, :] <= pos[:, None]
            if s["window"]:
                seen &= j[None, :] > pos[:, None] - s["window"]
            q = s["q"][r0:r1].double().view(r1 - r0, hkv, group, D)
            for g in range(hkv):
                z = torch.einsum("rhd,kd->rhk", q[:, g], k[:, g]) / 8.0
                z = torch.where(seen[:, None, :], z, torch.full_like(z, -math.inf))
                sink = s["sinks"][g * group:(g + 1) * group].double().view(1, group, 1)
                z = torch.softmax(torch.cat([z, sink.expand(r1 - r0, group, 1)], -1), -1)
                out[r0:r1, g * group:(g + 1) * group] = torch.einsum("rhk,kd->rhd", z[..., :-1], v[:, g])
    return out.view(-1, hq * D)
