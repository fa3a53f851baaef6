"""KV cache pages in 8 bits and attention over pages (rollout engine).

``kv_store_fp8`` writes new keys and values into e4m3 pages with one power-of-two scale per
(token, KV head), ``kv_gather_fp8`` reads rows back as bf16, and ``paged_attention`` computes
the attention of each sequence's new tokens -- one in decoding, a few in a speculative verify,
thousands in a prefill chunk -- over its pages in place, bf16 or e4m3.

e4m3 pools: codes [pages, page_size, Hkv, D] (``empty_fp8_pages`` keeps each KV head's rows of a
page together in memory) and scale bytes [pages, Hkv, page_size] uint8, e8m0: a row's values are
code * 2^(byte - 127), which bf16 holds exactly.  With a = the row's largest finite magnitude the
exponent is the smallest e in [-127, 120] with a <= 448 * 2^e; codes are rounded to nearest even
(and end at 240 for e = 120, so that values stay finite in bf16); entries that are not finite
become NaN.

CUDA kernels: csrc/paged_cache.cu and csrc/paged_attention.cu; the PyTorch references below run
on CPU tensors.
"""
from __future__ import annotations

import math

import torch

from ._ext import ext, use_cuda_kernels

FP8 = torch.float8_e4m3fn


def empty_fp8_pages(num_pages: int, page_size: int, hkv: int, head_dim: int, device):
    """(codes [pages, page_size, Hkv, D] e4m3, scale bytes [pages, Hkv, page_size] uint8), zeroed."""
    codes = torch.zeros(num_pages, hkv, page_size, head_dim, dtype=torch.uint8, device=device)
    scales = torch.zeros(num_pages, hkv, page_size, dtype=torch.uint8, device=device)
    return codes.view(FP8).permute(0, 2, 1, 3), scales


def quantize_rows_reference(x: torch.Tensor):
    """e4m3 codes and e8m0 scale bytes of rows [..., D]."""
    f = x.float()
    finite = torch.isfinite(f)
    amax = torch.where(finite, f.abs(), torch.zeros_like(f)).amax(-1, keepdim=True)
    frac, exp = torch.frexp(amax)               # amax = frac * 2^exp, frac in [0.5, 1)
    e = torch.where(amax > 0, exp - 9 + (frac > 0.875).to(exp.dtype), torch.full_like(exp, -127))
    e = e.clamp(-127, 120)
    inv = ((127 - e).to(torch.int32) << 23).view(torch.float32)
    limit = torch.where(e == 120, 240.0, 448.0)
    y = torch.minimum(torch.maximum(f * inv, -limit), limit)
    y = torch.where(finite, y, torch.full_like(y, math.nan))
    return y.to(FP8), (e + 127).to(torch.uint8).squeeze(-1)


def dequantize_rows_reference(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """fp32 values of e4m3 rows [..., D] with scale bytes [...]."""
    return torch.ldexp(codes.float(), scales.to(torch.int32).unsqueeze(-1) - 127)


def _check(ok: bool, msg: str) -> None:
    if not ok:
        raise RuntimeError(f"af3: {msg}")


def _check_pages(k_pages, v_pages, k_scales, v_scales) -> None:
    _check(k_pages.dim() == 4 and k_pages.shape == v_pages.shape,
           "pages must be [pages, page_size, Hkv, D], K and V alike")
    _check(k_pages.dtype == v_pages.dtype, "K and V pages must have one type")
    if k_pages.dtype == FP8:
        _check(k_scales is not None and v_scales is not None,
               "float8_e4m3fn pages need k_scales and v_scales")
        want = (k_pages.shape[0], k_pages.shape[2], k_pages.shape[1])
        _check(k_scales.dtype == v_scales.dtype == torch.uint8, "scales must be uint8 (e8m0)")
        _check(tuple(k_scales.shape) == tuple(v_scales.shape) == want,
               "scales must be [pages, Hkv, page_size], K and V alike")
    else:
        _check(k_scales is None and v_scales is None, "bfloat16 pages take no scales")


def _slots(slots, k_pages):
    ok = (slots >= 0) & (slots < k_pages.shape[0] * k_pages.shape[1])
    s = slots[ok].long()
    return ok, s // k_pages.shape[1], s % k_pages.shape[1]


def _slots32(slots, k_pages):
    """Slot ids as the kernels take them; ids of other types that are outside the pool become -1
    before they are narrowed."""
    if slots.dtype != torch.int32:
        n = min(k_pages.shape[0] * k_pages.shape[1], 2 ** 31 - 1)
        slots = slots.long()
        slots = torch.where((slots >= 0) & (slots < n), slots, -1).to(torch.int32)
    return slots.contiguous()


def kv_store_fp8_reference(qkv, k_off, v_off, slots, k_pages, v_pages, k_scales, v_scales):
    _check_pages(k_pages, v_pages, k_scales, v_scales)
    _check(k_pages.dtype == FP8, "kv_store_fp8 needs float8_e4m3fn pages")
    hkv, d = k_pages.shape[2:]
    ok, page, off = _slots(slots, k_pages)
    for col, pages, scales in ((k_off, k_pages, k_scales), (v_off, v_pages, v_scales)):
        x = qkv[: slots.numel()][ok, col:col + hkv * d].reshape(-1, hkv, d)
        codes, sc = quantize_rows_reference(x)
        pages.view(torch.uint8)[page, off] = codes.view(torch.uint8)
        scales[page, :, off] = sc


def kv_gather_fp8_reference(qkv, k_off, v_off, slots, k_pages, v_pages, k_scales, v_scales):
    _check_pages(k_pages, v_pages, k_scales, v_scales)
    _check(k_pages.dtype == FP8, "kv_gather_fp8 needs float8_e4m3fn pages")
    hkv, d = k_pages.shape[2:]
    ok, page, off = _slots(slots, k_pages)
    rows = ok.nonzero().squeeze(-1)
    for col, pages, scales in ((k_off, k_pages, k_scales), (v_off, v_pages, v_scales)):
        x = dequantize_rows_reference(pages.view(torch.uint8)[page, off].view(FP8),
                                      scales[page, :, off])
        qkv[rows, col:col + hkv * d] = x.reshape(-1, hkv * d).to(qkv.dtype)


def kv_store_fp8(qkv, k_off, v_off, slots, k_pages, v_pages, k_scales, v_scales) -> None:
    """K/V of row i of qkv [n, width] (Hkv * D values from columns k_off and v_off) -> page slot
    slots[i] (slot = page * page_size + offset) as e4m3 codes and scale bytes.  A slot outside the
    pool (e.g. -1) is skipped; the others must be distinct."""
    if not use_cuda_kernels(qkv):
        return kv_store_fp8_reference(qkv, k_off, v_off, slots, k_pages, v_pages, k_scales, v_scales)
    if slots.dtype != torch.int32 or not slots.is_contiguous():
        slots = _slots32(slots, k_pages)
    ext().kv_store_fp8(qkv, k_off, v_off, slots, k_pages, v_pages, k_scales, v_scales)


def kv_gather_fp8(qkv, k_off, v_off, slots, k_pages, v_pages, k_scales, v_scales) -> None:
    """The inverse of ``kv_store_fp8``: cached rows -> K/V columns of qkv in bf16, without rounding.
    Rows of slots outside the pool keep what they hold."""
    if not use_cuda_kernels(qkv):
        return kv_gather_fp8_reference(qkv, k_off, v_off, slots, k_pages, v_pages, k_scales, v_scales)
    if slots.dtype != torch.int32 or not slots.is_contiguous():
        slots = _slots32(slots, k_pages)
    ext().kv_gather_fp8(qkv, k_off, v_off, slots, k_pages, v_pages, k_scales, v_scales)


def paged_attention_reference(q, k_pages, v_pages, page_table, seq_lens, cu_q, sinks, hq, hkv,
                              window=0, scale=None, k_scales=None, v_scales=None,
                              dtype=torch.float32):
    """Dense reference, sequence by sequence, in ``dtype``.  Returns [T, Hq*D] of that type."""
    _check_pages(k_pages, v_pages, k_scales, v_scales)
    _check(hkv > 0 and hq % hkv == 0 and k_pages.shape[2] == hkv,
           "k_pages must be [pages, page_size, Hkv, D] with Hkv dividing Hq")
    P, D = k_pages.shape[1], k_pages.shape[3]
    _check(q.reshape(q.shape[0], -1).shape[1] == hq * D, "q must be [T, Hq * D]")
    _check(cu_q.numel() == seq_lens.numel() + 1 and page_table.shape[0] == seq_lens.numel(),
           "seq_lens must be [B], cu_q [B + 1] and page_table [B, max_pages]")
    _check(window >= 0, "window must not be negative")
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    T = q.shape[0]
    qv = q.reshape(T, hq, D)
    out = torch.zeros(T, hq, D, dtype=dtype, device=q.device)
    cu = cu_q.tolist()
    for b, L in enumerate(seq_lens.tolist()):
        t0, t1 = cu[b], cu[b + 1]
        n = min(L, page_table.shape[1] * P)
        if t1 <= t0 or n <= 0:
            continue
        j = torch.arange(n, device=q.device)
        page = page_table[b][j // P].long()
        there = (page >= 0) & (page < k_pages.shape[0])
        page = torch.where(there, page, torch.zeros_like(page))
        if k_scales is None:
            k, v = k_pages[page, j % P].to(dtype), v_pages[page, j % P].to(dtype)
        else:
            k, v = (torch.ldexp(c.view(torch.uint8)[page, j % P].view(FP8).to(dtype),
                                s[page, :, j % P].to(torch.int32).unsqueeze(-1) - 127)
                    for c, s in ((k_pages, k_scales), (v_pages, v_scales)))
        pos = L - (t1 - t0) + torch.arange(t1 - t0, device=q.device)
        seen = (j[None, :] <= pos[:, None]) & there[None, :]
        if window:
            seen &= pos[:, None] - j[None, :] < window
        k = k.repeat_interleave(hq // hkv, 1).transpose(0, 1)          # [Hq, n, D]
        v = v.repeat_interleave(hq // hkv, 1).transpose(0, 1)
        s = qv[t0:t1].to(dtype).transpose(0, 1) @ k.transpose(1, 2) * scale
        s = s.masked_fill(~seen[None], float("-inf"))
        top = s.amax(-1, keepdim=True)
        if sinks is not None:
            top = torch.maximum(top, sinks.to(dtype).view(hq, 1, 1))
        top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
        p = torch.exp(s - top)
        den = p.sum(-1, keepdim=True)
        if sinks is not None:
            den = den + torch.exp(sinks.to(dtype).view(hq, 1, 1) - top)
        # a key that a row does not see is left out of its sum, whatever its value
        finite = torch.isfinite(v).all(-1).all(0)
        o = p[..., finite] @ v[:, finite]
        for x in (~finite).nonzero().squeeze(-1).tolist():
            o = torch.where(seen[None, :, x, None], o + p[..., x, None] * v[:, x, None, :], o)
        o = torch.where(den > 0, o / den, torch.where(torch.isnan(den), den, torch.zeros_like(o)))
        out[t0:t1] = o.transpose(0, 1)
    return out.reshape(T, hq * D)


def paged_attention(q, k_pages, v_pages, page_table, seq_lens, cu_q, sinks, hq, hkv, window=0,
                    scale=None, k_scales=None, v_scales=None, max_q_len=None, max_seq_len=None,
                    out=None):
    """Attention of the new tokens of B sequences over their cache pages.

    q [T, Hq*D]: the new tokens' queries, sequence after sequence (rows may be strided);
    cu_q int32 [B+1]: their row ranges; seq_lens int32 [B]: tokens of each sequence, its new ones
    (already stored) included; page_table int32 [B, max_pages].  Row i of sequence b has position
    p = seq_lens[b] - (cu_q[b+1] - cu_q[b]) + i and sees keys j <= p, with ``window`` only those
    with p - j < window.  A page id outside [0, pages) marks a page that is not held (any more):
    its keys are not visible.  ``sinks`` [Hq] joins the denominator (None: no sink).  A row that
    sees nothing gets zeros; rows outside cu_q's ranges are not written.  There is no backward pass on
    CUDA tensors: a q that asks for a gradient is refused.

    max_q_len / max_seq_len: the longest of each, if the caller knows them (otherwise they are
    read back from the device).  They choose the kernel variant and its split of the work; the
    result does not depend on them being exact.
    """
    if not use_cuda_kernels(q):
        r = paged_attention_reference(q, k_pages, v_pages, page_table, seq_lens, cu_q, sinks, hq,
                                      hkv, window, scale, k_scales, v_scales).to(q.dtype)
        if out is None:
            return r
        cu = cu_q.tolist()
        for t0, t1 in zip(cu, cu[1:]):      # rows of no sequence are left as they are
            out[t0:t1] = r[t0:t1]
        return out
    if q.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("af3: paged_attention has no backward pass: call it under torch.no_grad()")
    if q.dim() == 3:
        q = q.reshape(q.shape[0], -1)
    if scale is None:
        scale = 1.0 / math.sqrt(k_pages.shape[-1])
    if out is None:
        out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    if max_q_len is None:
        max_q_len = int((cu_q[1:] - cu_q[:-1]).max()) if seq_lens.numel() else 1
    if max_seq_len is None:
        max_seq_len = int(seq_lens.max()) if seq_lens.numel() else 1
    if sinks is not None and (sinks.dtype != torch.float32 or not sinks.is_contiguous()):
        sinks = sinks.float().contiguous()
    ext().paged_attention(q, k_pages, v_pages, k_scales, v_scales, page_table, seq_lens, cu_q, sinks,
                          out, hq, hkv, window, scale, max_q_len, max_seq_len)
    return out
