"""Serving with a key / value cache in 8 bits: prompts, portions, single tokens and captured steps through the engine."""
import pytest
import torch

from zml_b200 import ops
from zml_b200.models import dopurax, lfm2, qwen3_5, qwen3_moe
from zml_b200.models.llama import PRESETS, LlamaConfig, LlamaModel
from zml_b200.serving import Engine

gpu = pytest.mark.gpu
KINDS = pytest.mark.parametrize("kind", ["fp8", "int8"])
FAMILIES = {
    "llama": (LlamaConfig, LlamaModel, PRESETS["tiny-llama-test"]),
    "qwen3_moe": (qwen3_moe.Qwen3MoeConfig, qwen3_moe.Qwen3MoeModel, qwen3_moe.PRESETS["tiny-moe-test"]),
    "qwen3_5": (qwen3_5.Qwen35Config, qwen3_5.Qwen35Model, qwen3_5.PRESETS["tiny-qwen35-test"]),
    "lfm2": (lfm2.Lfm2Config, lfm2.Lfm2Model, lfm2.PRESETS["tiny-lfm2-test"]),
}


def model(family="llama", device="cpu", dtype=torch.bfloat16):
    config, cls, preset = FAMILIES[family]
    return cls(config.from_hf(dict(preset)), device=device, dtype=dtype).init_random(seed=3, std=0.05)


def engine(m, kind, page=16, **kw):
    return Engine(m, num_pages=64, page_size=page, max_batch=4, max_seq_len=512, kv_dtype=kind, **kw)


def tokens(n, seed=0):
    return torch.randint(0, 1000, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def fed(m, kind, prompt, portions, page=16, **kw):
    """Logits behind every portion's last token."""
    e = engine(m, kind, page, **kw)
    r, out, at = e.open_request(), [], 0
    for n in portions:
        out.append(e.step([(r, prompt[at:at + n])], [[n - 1]])[0].float().cpu())
        at += n
    return torch.stack(out)


def off(a, b):
    return float((a - b).norm() / b.norm())


@KINDS
def test_portions_and_single_tokens_agree_with_one_prompt(kind):
    """What is cached is the same however the tokens come, and attention over prompts and of single tokens read the same values.  What is left is
    bf16: activations rounded at 2^-8 through two layers, and codes that such a rounding moves by a step of 2^-4 (one in eight of a row's numbers, then
    averaged over the keys)."""
    m, prompt = model(), tokens(80)
    whole = fed(m, kind, prompt, [80])
    assert off(fed(m, kind, prompt, [33, 30, 17])[-1], whole[0]) < 0.03
    assert off(fed(m, kind, prompt, [77, 1, 1, 1])[-1], whole[0]) < 0.03


@KINDS
def test_logits_are_near_those_of_the_bf16_cache(kind):
    """e4m3 keeps four bits of a number: each key and value is within 2^-4, 0.036 of its size on average, int8 within half a unit of 63 to 127.  The
    differences are independent from key to key; they add up to at most that share of attention's part of the residual stream."""
    m, prompt = model(), tokens(80)
    assert off(fed(m, kind, prompt, [80])[0], fed(m, None, prompt, [80])[0]) < 0.1


def test_what_takes_no_such_cache():
    m = model()
    for bad in ("fp16", "e4m3", ""):
        with pytest.raises(ValueError):
            engine(m, bad)
    with pytest.raises(ValueError):
        engine(m, "fp8", page=24)
    with pytest.raises(ValueError):
        engine(model(dtype=torch.float32), "fp8")
    other = dopurax.DopuraxModel(dopurax.DopuraxConfig.from_hf(dict(dopurax.PRESETS[next(k for k in dopurax.PRESETS if "tiny" in k)])), device="cpu")
    with pytest.raises(ValueError):
        engine(other, "fp8")
    m.set_attention_backend("vanilla")
    e = engine(m, "fp8")
    with pytest.raises(ValueError):
        e.step([(e.open_request(), [1, 2, 3])])


def test_memory():
    m = model()
    a, b = engine(m, None).kv_cache, engine(m, "int8").kv_cache
    assert b.nbytes() * 64 == a.numel() * 65             # 65 bytes for a head of 64 numbers


@pytest.mark.parametrize("family", ["qwen3_moe", "qwen3_5", "lfm2"])
def test_other_families_cpu(family):
    m, prompt = model(family), tokens(40)
    whole = fed(m, "fp8", prompt, [40])
    assert off(fed(m, "fp8", prompt, [38, 1, 1])[-1], whole[0]) < 0.05


# ------------------------------------------------------------------ on the device
@gpu
@KINDS
@pytest.mark.parametrize("page", [64, 16])
def test_engine_matches_the_cpu(kind, page):
    """The same weights through the kernels and through the restatements; both round activations to bf16, in another order."""
    g = model(device="cuda")
    c = LlamaModel(g.config, device="cpu")
    c.embed, c.final_norm, c.lm_head = g.embed.cpu(), g.final_norm.cpu(), g.lm_head.cpu()
    for lw in g.layers:
        to = type(lw)()
        for name in lw.__slots__:
            t = getattr(lw, name)
            setattr(to, name, t.cpu() if isinstance(t, torch.Tensor) else t)
        c.layers.append(to)
    prompt, portions = tokens(200, 1), [150, 40, 1, 1, 7, 1]
    want = fed(c, kind, prompt, portions, page)
    got = fed(g, kind, prompt, portions, page)
    for a, b in zip(got, want):
        assert off(a, b) < 0.03
    ops.raise_on_status()


@gpu
@KINDS
@pytest.mark.parametrize("family", sorted(FAMILIES))
def test_captured_steps_are_eager_ones(family, kind):
    m = model(family, "cuda")
    prompts = [tokens(n, n) for n in (30, 5, 64, 129)]
    eager = engine(m, kind, 64, use_graphs=False).generate(prompts, max_new_tokens=24)[0]
    captured = engine(m, kind, 64).generate(prompts, max_new_tokens=24)[0]
    assert eager == captured
    ops.raise_on_status()


@gpu
@KINDS
def test_serving_many_requests(kind):
    m = model(device="cuda")
    prompts = [tokens(n, n) for n in (30, 5, 64, 129, 17, 90, 1, 200)]
    alone = [engine(m, kind, 64).generate([p], max_new_tokens=12)[0][0] for p in prompts]
    served = engine(m, kind, 64).serve(prompts, 12)[0]
    # greedy tokens of a random model may part where two logits are equal to bf16; most do not
    same = sum(a == b for x, y in zip(alone, served) for a, b in zip(x, y))
    assert all(len(x) == 12 for x in served) and same >= 0.75 * 12 * len(prompts)
    ops.raise_on_status()


@gpu
def test_graphs_of_short_and_long_sequences_are_apart():
    """A step that was captured for short sequences is not replayed for long ones: their launches are planned by the longest sequence."""
    m = model(device="cuda")
    prompts = [tokens(10), tokens(3000, 4)]

    def run(**kw):
        e = Engine(m, num_pages=80, page_size=64, max_batch=4, max_seq_len=4096, kv_dtype="fp8", **kw)
        return e, [e.generate([p], max_new_tokens=6)[0][0] for p in prompts]
    e, captured = run()
    plans = [e._plan_splits(1, n) for n in (16, 3006)]
    assert plans[0] != plans[1] and {key[3] for key in e._graphs} == set(plans)
    assert captured == run(use_graphs=False)[1]
    ops.raise_on_status()
