"""What an engine with shared pages takes, it can answer, with a GPU and without."""
import pytest
import torch

from zml_b200 import ops
from zml_b200.models.llama import PRESETS, LlamaConfig, LlamaModel
from zml_b200.serving import Engine

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _model(device, **more):
    cfg = LlamaConfig.from_hf(dict(PRESETS["tiny-llama-test"], **more))
    return LlamaModel(cfg, device=device, dtype=torch.float32 if device == "cpu" else torch.bfloat16).init_random(seed=1, std=0.08)


@pytest.mark.parametrize("device", DEVICES)
def test_sizes_are_refused_when_the_engine_is_made(device):
    fits = _model(device)
    for kw in ({"page_size": 8}, {"page_size": 48}, {"max_batch": ops.shared.MAX_BATCH + 1}):
        with pytest.raises(ValueError, match="shared pages are for"):
            Engine(fits, 16, share_prefixes=True, **kw)
    with pytest.raises(ValueError, match="shared pages are for heads"):
        Engine(_model(device, head_dim=32), 16, share_prefixes=True)
    wide = _model(device)
    wide.hq, wide.hkv = 129, 1
    with pytest.raises(ValueError, match="129 to 1"):
        Engine(wide, 16, share_prefixes=True)
    eng = Engine(fits, 64, page_size=64, max_batch=4, max_seq_len=256, share_prefixes=True)
    eng.SHARE_BYTES = 0
    a = list(range(70))
    got, _ = eng.generate([a + [1], a + [2]], 3)
    assert [len(t) for t in got] == [3, 3]
    if device == "cpu":                                          # (in bf16 two orders of a sum may choose two tokens)
        assert got == Engine(fits, 64, page_size=64, max_batch=4, max_seq_len=256).generate([a + [1], a + [2]], 3)[0]
    assert eng.pool.num_free == 63
