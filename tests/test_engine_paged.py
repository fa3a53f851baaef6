"""Rollout engine with attention over the cache pages in place and with an e4m3 cache (CPU
references): the same logits as the gathering path, chunked prefill and verify blocks, reading
the cache back, prefix hits, memory accounting, launch flags."""
import threading

import pytest
import torch

from agent_factory_3_b200.engine.kv_cache import PagedKVCache
from agent_factory_3_b200.engine.model_runner import ModelRunner, StepItem
from agent_factory_3_b200.engine.scheduler import Engine, Request
from agent_factory_3_b200.models.gpt_oss import GptOssConfig, GptOssForCausalLM


@pytest.fixture(scope="module")
def model():
    return GptOssForCausalLM(GptOssConfig.tiny(), device="cpu", dtype=torch.float32).init_random(0).eval()


def runner(model, quant=None, paged=False):
    c = model.cfg
    kv = PagedKVCache(c.num_hidden_layers, 16, 8, c.num_key_value_heads, c.head_dim,
                      c.num_experts_per_tok, "cpu", torch.float32, kv_quant=quant)
    return ModelRunner(model, kv, lora_active=False, paged=paged)


def steps(prompts, whole):
    """A prefill (whole or in two chunks), a mixed step and a verify block of two sequences."""
    a, b = prompts
    pa, pb = [3, 0, 5], [2, 7]
    if whole:
        yield [StepItem(a, 0, pa)]
    else:
        yield [StepItem(a[:9], 0, pa, want_logits=False)]
        yield [StepItem(a[9:], 9, pa)]
    yield [StepItem([5], len(a), pa), StepItem(b, 0, pb)]
    yield [StepItem([6], len(a) + 1, pa), StepItem([7, 8, 9], len(b), pb, all_logits=True)]


PROMPTS = (list(range(20, 37)), list(range(40, 47)))


def logits(r, whole=True):
    return torch.cat([r.forward(s).logits for s in steps(PROMPTS, whole)])


def test_paged_equals_gathered(model):
    want = logits(runner(model))
    for whole in (True, False):
        torch.testing.assert_close(logits(runner(model, paged=True), whole), want, rtol=1e-3, atol=1e-3)


def test_quantised_cache(model):
    a, b, plain = runner(model, "e4m3"), runner(model, "e4m3"), runner(model)
    assert a.paged
    # new tokens see the stored values: how a prompt is cut does not matter
    torch.testing.assert_close(logits(a, True), logits(b, False), rtol=1e-3, atol=1e-3)
    logits(plain)
    slots = torch.tensor([3 * 8 + i for i in range(8)] + [1, 2 * 8 + 4])
    k, v = a.kv.read(0, slots)
    pk, pv = plain.kv.read(0, slots)
    assert k.shape == (10, model.cfg.num_key_value_heads, model.cfg.head_dim)
    for x, y in ((k.float(), pk), (v.float(), pv)):        # layer 0 sees the same input
        top = y.abs().amax(-1, keepdim=True)
        # half a step of e4m3 (2^-4 of the value), 2^-10 of the scale below its normal range,
        # where the scale is at most top / 224; then bf16 exactly
        assert ((x - y).abs() <= 2.0 ** -4 * y.abs() + 2.0 ** -10 * top / 224 + 1e-12).all()


@pytest.mark.parametrize("kw", [dict(kv_quant="e4m3"), dict(paged_attention=True)])
def test_engine_generates(model, kw):
    eng = Engine(model, num_pages=64, page_size=8, max_prefill_tokens=16, **kw).start()
    try:
        outs = []
        for _ in range(2):
            done = threading.Event()
            r = Request(input_ids=list(range(7, 47)), max_new_tokens=6, temperature=0.0,
                        on_output=lambda o: done.set() if o["finished"] else None)
            eng.submit(r)
            assert done.wait(60)
            outs.append((list(r.output_ids), r.cached_tokens))
    finally:
        eng.stop()
    assert len(outs[0][0]) == 6 and outs[0][0] == outs[1][0]
    assert outs[0][1] == 0 and outs[1][1] >= 32            # the second run hits the prefix cache


def test_memory_accounting():
    page = PagedKVCache.bytes_per_page(36, 64, 8, 64, 4, kv_quant="e4m3")
    assert page == 36 * 64 * (2 * 8 * 65 + 4)
    kv = PagedKVCache(2, 4, 8, 2, 16, 2, "cpu", kv_quant="e4m3")
    held = sum(t.numel() for pool in (kv.k, kv.v, kv.k_scale, kv.v_scale) for t in pool)
    assert kv.bytes_per_token * 4 * 8 == held
    with pytest.raises(ValueError, match="kv_quant"):
        PagedKVCache(1, 1, 8, 2, 16, 2, "cpu", kv_quant="int4")


def test_launch_flags():
    from agent_factory_3_b200.engine.server import build_arg_parser, resolve_args
    a = build_arg_parser().parse_args(["--kv-quant", "e4m3", "--kv-cache-dtype", "fp8_e4m3"])
    assert a.kv_quant == "e4m3" and not any("stays bf16" in n for n in resolve_args(a, world=1))
    a = build_arg_parser().parse_args(["--paged-attention"])
    assert a.paged_attention and a.kv_quant == "none" and resolve_args(a, world=1) == []
