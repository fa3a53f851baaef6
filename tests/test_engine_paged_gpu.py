"""Rollout engine over cache pages in place and with an e4m3 cache, on the GPU kernels."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    from agent_factory_3_b200.models.gpt_oss import GptOssConfig, GptOssForCausalLM
    cfg = GptOssConfig.preset("gpt-oss-20b")
    cfg.num_hidden_layers = 2
    cfg.layer_types = cfg.layer_types[:2]
    return GptOssForCausalLM(cfg, device="cuda").init_random(0).eval()


def runner(model, quant=None, paged=False):
    from agent_factory_3_b200.engine.kv_cache import PagedKVCache
    from agent_factory_3_b200.engine.model_runner import ModelRunner
    c = model.cfg
    kv = PagedKVCache(2, 48, 64, c.num_key_value_heads, c.head_dim, c.num_experts_per_tok, "cuda",
                      torch.bfloat16, kv_quant=quant)
    return ModelRunner(model, kv, lora_active=False, paged=paged)


def attention(r, items, li, seed):
    """Output of one layer's attention for the items, with the layer's own input."""
    a = r.model.layers[li].self_attn
    n = sum(len(it.ids) for it in items)
    g = torch.Generator(device="cuda").manual_seed(seed)
    xn = torch.randn(n, r.cfg.hidden_size, device="cuda", generator=g).bfloat16()
    with torch.inference_mode():
        return r._attention(li, r._meta(items), xn, a.qkv_weight, a.qkv_bias, None, None, 1.0,
                            a.sinks, a.window, r.cfg.num_attention_heads,
                            r.cfg.num_key_value_heads, r.model.rope(r.device))


@pytest.mark.parametrize("li", [0, 1])      # sliding-window and full-attention layer
def test_attention_of_a_step(model, li):
    from agent_factory_3_b200.engine.model_runner import StepItem
    ids = list(range(1000))
    first = [StepItem(ids[:300], 0, [0, 1, 2, 3, 4, 5]), StepItem(ids[:77], 0, [6, 7])]
    mixed = [StepItem([1], 77, [6, 7]), StepItem(ids[:60], 300, [0, 1, 2, 3, 4, 5]),
             StepItem(ids[:9], 0, [9], all_logits=True)]
    verify = [StepItem(ids[:9], 78, [6, 7], all_logits=True), StepItem(ids[:9], 9, [9], all_logits=True)]
    plain, paged, quant = runner(model), runner(model, paged=True), runner(model, "e4m3")
    for seed, items in enumerate((first, mixed, verify)):
        want = attention(plain, items, li, seed).float()
        top = want.abs().max()
        # both round probabilities and output to bf16 at worst
        assert (attention(paged, items, li, seed).float() - want).abs().max() <= 2.0 ** -6 * top
        # keys and values rounded to 4 bits: a half step is 2^-4
        err = (attention(quant, items, li, seed).float() - want).norm() / want.norm()
        assert err < 2.0 ** -4


@pytest.mark.parametrize("quant", [None, "e4m3"])
def test_graph_decode_matches_eager(model, quant):
    from agent_factory_3_b200.engine.cuda_graph import DecodeGraphs
    from agent_factory_3_b200.engine.model_runner import StepItem
    eager, graphed = runner(model, quant, True), runner(model, quant, True)
    graphed.graphs = DecodeGraphs(graphed)
    prompts = [list(range(70)), list(range(200, 330))]
    pages = [[0, 1], [2, 3, 4]]
    for r in (eager, graphed):
        r.forward([StepItem(p, 0, pg) for p, pg in zip(prompts, pages)])
    for step in range(3):
        items = [StepItem([7 + step], 70 + step, pages[0]), StepItem([9 + step], 130 + step, pages[1])]
        want, got = eager.forward(items).logits, graphed.forward(items).logits
        assert torch.isfinite(got).all()
        assert (got - want).norm() <= 0.05 * want.norm()
    assert graphed.graphs.replays == 3
