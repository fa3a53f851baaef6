"""Attention over cache pages against the other paths of the rollout engine, and the kernel for few
rows against the one for many: median times in us, L2 flushed before each call.

    python perf/paged_paths.py

64 query heads on 8 KV heads, head dim 64, pages of 64, sinks; the inputs of perf/operators.py.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from agent_factory_3_b200.ops import decode, paged  # noqa: E402
from agent_factory_3_b200.ops._ext import ext  # noqa: E402
from perf.operators import prepare  # noqa: E402

BASE = dict(op="attention", hq=64, hkv=8, page=64, window=0, ragged=False)


def median_us(f, flush, n=15):
    for _ in range(3):
        f()
    ts = []
    for _ in range(n):
        flush.zero_()
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        torch.cuda.synchronize()
        ts.append(a.elapsed_time(b) * 1e3)
    return sorted(ts)[n // 2]


def in_place(s, max_q=None):
    return lambda: paged.paged_attention(
        s["q"], s["k"], s["v"], s["table"], s["lens"], s["cu"], s["sinks"], s["hq"], s["hkv"], s["window"],
        k_scales=s["ks"], v_scales=s["vs"], max_q_len=max_q or s["max_q"], max_seq_len=s["max_len"])


def row_by_row(s, q):
    """decode_attention with one row a token."""
    table = s["table"].repeat_interleave(q, 0).contiguous()
    lens = (s["lens"][:, None] - (q - 1) + torch.arange(q, device="cuda")).reshape(-1).int().contiguous()
    return lambda: decode.decode_attention(s["q"], s["k"], s["v"], table, lens, s["sinks"], s["hq"], s["hkv"],
                                           s["window"], None, s["max_len"])


def gathered(s, q, ctx):
    """One sequence's context gathered into a packed buffer, then the packed attention."""
    hq, hkv = s["hq"], s["hkv"]
    width, cols = (hq + 2 * hkv) * 64, hq * 64
    j = torch.arange(ctx, device="cuda")
    slots = (s["table"][0].long()[j // 64] * 64 + j % 64).int()
    new = torch.zeros(q, width, device="cuda", dtype=torch.bfloat16)
    new[:, :cols] = s["q"]
    at = torch.arange(ctx - q, ctx, device="cuda")
    tiles = torch.tensor([(0, x, min(x + 256, ctx)) for x in range(ctx - q, ctx, 256)][::-1], dtype=torch.int32,
                         device="cuda")
    cu = torch.tensor([0, ctx], dtype=torch.int32, device="cuda")

    def run():
        c = torch.zeros(ctx, width, device="cuda", dtype=torch.bfloat16)
        if s["ks"] is None:
            decode.kv_gather(c, cols, cols + hkv * 64, slots, s["k"], s["v"])
            c.index_copy_(0, at, new)
        else:
            paged.kv_gather_fp8(c, cols, cols + hkv * 64, slots, s["k"], s["v"], s["ks"], s["vs"])
            c[:, :cols].index_copy_(0, at, new[:, :cols])
        o = torch.empty(ctx, cols, device="cuda", dtype=torch.bfloat16)
        lse = torch.empty(hq, ctx, device="cuda")
        ext().attn_fwd(c, s["sinks"], tiles, cu, o, lse, hq, hkv, 64, s["window"], 0.125)
        return o.index_select(0, at)
    return run


def main():
    flush = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")

    def t(f):
        return median_us(f, flush)

    def both(**kw):
        return [prepare({**BASE, **kw, "fp8": fp8}, 1) for fp8 in (False, True)]

    for window in (0, 128):
        b, f = both(batch=128, q=1, context=4096, window=window)
        print("decode 128 x 4096, window %d: decode_attention %.1f, in place bf16 %.1f, e4m3 %.1f"
              % (window, t(row_by_row(b, 1)), t(in_place(b)), t(in_place(f))), flush=True)
    b, f = both(batch=64, q=9, context=4096)
    print("verify 64 x 9 on 4096: row by row %.1f, in place bf16 %.1f, e4m3 %.1f"
          % (t(row_by_row(b, 9)), t(in_place(b)), t(in_place(f))), flush=True)
    for q, ctx, window in ((4096, 16384, 0), (4096, 16384, 128), (1024, 32768, 0), (256, 8192, 0)):
        b, f = both(batch=1, q=q, context=ctx, window=window)
        print("chunk %d of %d, window %d: gathered + packed bf16 %.1f, e4m3 %.1f; in place bf16 %.1f, e4m3 %.1f"
              % (q, ctx, window, t(gathered(b, q, ctx)), t(gathered(f, q, ctx)), t(in_place(b)), t(in_place(f))),
              flush=True)
    # the longest q chooses the kernel: 5 tokens (40 rows a KV head) or fewer the one for few rows
    for batch, q, ragged in ((64, 4, False), (64, 5, False), (64, 5, True), (8, 5, False)):
        for name, s in zip(("bf16", "e4m3"), both(batch=batch, q=q, context=4200, ragged=ragged)):
            print("%d sequences of %s%d tokens on %s4200, %s: few rows %.1f, many rows %.1f"
                  % (batch, "1 to " * ragged, q, "210 to " * ragged, name, t(in_place(s, q)), t(in_place(s, 6))),
                  flush=True)


if __name__ == "__main__":
    main()
