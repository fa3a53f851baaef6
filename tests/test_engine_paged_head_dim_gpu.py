"""Rollout engine over cache pages with a head dimension that the attention kernels do not have."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    from agent_factory_3_b200.models.gpt_oss import GptOssConfig, GptOssForCausalLM
    cfg = GptOssConfig.preset("gpt-oss-20b")
    cfg.num_hidden_layers = 2
    cfg.layer_types = cfg.layer_types[:2]
    cfg.head_dim = 32
    return GptOssForCausalLM(cfg, device="cuda").init_random(0).eval()


def runner(model, quant=None, paged=False):
    from agent_factory_3_b200.engine.kv_cache import PagedKVCache
    from agent_factory_3_b200.engine.model_runner import ModelRunner
    c = model.cfg
    kv = PagedKVCache(2, 16, 16, c.num_key_value_heads, c.head_dim, c.num_experts_per_tok, "cuda",
                      torch.bfloat16, kv_quant=quant)
    return ModelRunner(model, kv, lora_active=False, paged=paged)


def attention(r, items, li, xn):
    a = r.model.layers[li].self_attn
    with torch.inference_mode():
        return r._attention(li, r._meta(items), xn, a.qkv_weight, a.qkv_bias, None, None, 1.0,
                            a.sinks, a.window, r.cfg.num_attention_heads,
                            r.cfg.num_key_value_heads, r.model.rope(r.device)).float()


@pytest.mark.parametrize("li", [0, 1])      # sliding-window and full-attention layer
def test_steps_equal_one_prefill(model, li):
    """A prompt cut into chunk, decode row, verify block and a mixed step against one prefill."""
    from agent_factory_3_b200.engine.model_runner import StepItem
    g = torch.Generator(device="cuda").manual_seed(li)
    x, y = (torch.randn(n, model.cfg.hidden_size, device="cuda", generator=g).bfloat16() for n in (60, 9))
    ids, px, py = list(range(60)), [0, 3, 1, 2], [5]
    plain = runner(model)
    want = attention(plain, [StepItem(ids, 0, px)], li, x)
    want_y = attention(plain, [StepItem(ids[:9], 0, py)], li, y)
    for r, tol in ((runner(model, paged=True), 2.0 ** -6), (runner(model, "e4m3"), 2.0 ** -3)):
        got = [attention(r, [StepItem(ids[:50], 0, px)], li, x[:50]),
               attention(r, [StepItem(ids[50:51], 50, px)], li, x[50:51]),
               attention(r, [StepItem(ids[51:59], 51, px, all_logits=True)], li, x[51:59])]
        last = attention(r, [StepItem(ids[59:], 59, px), StepItem(ids[:9], 0, py)], li,
                         torch.cat([x[59:], y]))
        got = torch.cat(got + [last[:1]])
        # bf16 pages: P and the output rounded to bf16 at worst; e4m3: K and V rounded to 4 bits
        for a, b in ((got, want), (last[1:], want_y)):
            assert (a - b).abs().max() <= 2 * tol * b.abs().max()
            assert (a - b).norm() <= tol * b.norm()


@pytest.mark.parametrize("quant", [None, "e4m3"])
def test_decode_steps_with_graphs(model, quant):
    """Whole steps: graphs leave such decode steps to the gathering path."""
    from agent_factory_3_b200.engine.cuda_graph import DecodeGraphs
    from agent_factory_3_b200.engine.model_runner import StepItem
    r = runner(model, quant, True)
    r.graphs = DecodeGraphs(r)
    prompt, pages = list(range(40)), [0, 1, 2]
    r.forward([StepItem(prompt, 0, pages)])
    got = r.forward([StepItem([7], 40, pages)]).logits
    whole = runner(model, quant, True).forward([StepItem(prompt + [7], 0, pages)]).logits
    assert r.graphs.replays == 0 and got.shape == whole.shape
    assert (got - whole).norm() <= 0.05 * whole.norm()
