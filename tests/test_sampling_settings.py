"""Who draws what a sampling strategy asks for: the tagged API, the models, the engine and the server."""
import pytest
import torch

from zml_b200 import nn, ops
from zml_b200.models.common import SamplingStrategy
from zml_b200.tensor import Rng, Tensor

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]


def _draws(x, tags, opts, n=40, device="cpu"):
    rng, out = Rng(5, device), []
    for _ in range(n):
        tok, rng = nn.sample_tokens(Tensor(x, None, tags), opts, rng)
        out.append(tok.data)
    assert tok.shape().tags == tuple(t for t in tags if t != "voc") and tok.data.dtype is torch.int32
    return torch.stack(out)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_tagged_draws_follow_top_p_and_min_p(device, dtype):
    x = torch.randn((3, 4, 300), generator=torch.Generator().manual_seed(0), dtype=torch.float64).to(dtype).to(device)
    best = x.float().argmax(-1).int()
    for tags, y in ((("b", "s", "voc"), x), (("b", "voc", "s"), x.transpose(1, 2)), (("voc", "b", "s"), x.movedim(-1, 0))):
        for one in (SamplingStrategy(50, 1.0, 1e-4), SamplingStrategy(0, 1.0, 1.0, 1.0), SamplingStrategy(-1, 1e-4), SamplingStrategy(1, 1.0, 0.5), SamplingStrategy()):
            assert bool((_draws(y, tags, one, 3, device) == best).all())
        for opts in (SamplingStrategy(0, 1.0, 0.9), SamplingStrategy(-1), SamplingStrategy(40, 1.3, 0.8, 0.05), SamplingStrategy(300, 0.8, 0.7)):
            got = _draws(y, tags, opts, 40, device)
            assert all(len(set(got[:, i, j].tolist())) > 3 for i in range(3) for j in range(4))       # flat rows: every one draws
            p = torch.softmax(x.double() / opts.temperature, -1)
            order = p.sort(-1, descending=True)
            place = torch.zeros_like(order.indices).scatter_(-1, order.indices, torch.arange(300, device=device).expand_as(order.indices))
            place = place.gather(-1, got.movedim(0, -1).long())
            if opts.topk > 0:
                assert int(place.max()) < opts.topk
            if opts.top_p < 1 and opts.topk <= 0:       # no token behind the smallest set that reaches top_p
                most = (order.values.cumsum(-1) - order.values < opts.top_p + 1e-3).sum(-1, keepdim=True)
                assert bool((place < most).all())
            if opts.min_p > 0:
                w = p.gather(-1, got.movedim(0, -1).long()) / p.amax(-1, keepdim=True)
                assert bool((w >= opts.min_p * (1 - 1e-2)).all())
    flat = Tensor(x[0, 0], None, ("voc",))
    assert int(nn.sample_tokens(flat, SamplingStrategy(0, 1.0, 1e-3), Rng(1, device))[0].data) == int(best[0, 0])


@pytest.mark.parametrize("device", DEVICES)
def test_tagged_draws_are_those_of_the_operator(device):
    x = torch.randn((6, 500), generator=torch.Generator().manual_seed(2)).to(device)
    bits = torch.randint(0, 2 ** 53, (6,), generator=Rng(9, device).gen, device=device)
    want = ops.sample(x, bits.double() * 2.0 ** -53, 0.7, 100, 0.95, 0.01)
    got, _ = nn.sample_tokens(Tensor(x, None, ("b", "voc")), SamplingStrategy(100, 0.7, 0.95, 0.01), Rng(9, device))
    assert torch.equal(got.data, want)


@pytest.mark.parametrize("device", DEVICES)
def test_a_wide_top_k_alone_stays_with_gumbel_noise(device):
    x = torch.randn((6, 500), generator=torch.Generator().manual_seed(2)).to(device)
    vals, idx = torch.topk(x, 200, -1)
    noise = Rng(9, device).gumbel(Tensor(vals, None, ("b", "topk")).shape()).data
    want = idx.gather(1, (vals * (1 / 0.7) + noise).argmax(-1, keepdim=True))[:, 0].int()
    got, _ = nn.sample_tokens(Tensor(x, None, ("b", "voc")), SamplingStrategy(200, 0.7), Rng(9, device))
    assert torch.equal(got.data, want)


class _Engine:
    max_pages, page_size, comm = 8, 16, None


class _Tok:
    def decode(self, ids, *a):
        return "x" * len(ids)


def test_settings_next_to_their_ends_still_cut_at_the_server():
    from zml_b200.serving.server import Server
    greedy = Server(_Engine(), _Tok())
    for given, top_p, min_p in (({"top_p": 0.9996}, 0.999, 0.0), ({"top_p": 0.99999999}, 0.999, 0.0), ({"top_p": 1e-9}, 0.001, 0.0), ({"top_p": 0.9994}, 0.999, 0.0),
                                ({"min_p": 0.0004}, 1.0, 0.001), ({"min_p": 1e-9}, 1.0, 0.001), ({"min_p": 0.9999}, 1.0, 0.999), ({"top_p": 0}, 0.0, 0.0),
                                ({"min_p": 1}, 1.0, 1.0), ({"top_p": 0.9996, "min_p": 0.0004}, 0.999, 0.001)):
        assert greedy._sampling(given) == (0, 1.0, 0, top_p, min_p)
        assert greedy._sampling({**given, "top_k": 500}) == (500, 1.0, 0, top_p, min_p)
    for none in ({"top_p": 1}, {"min_p": 0}, {"top_p": 1.0, "min_p": 0.0}):
        assert greedy._sampling(none) == (1, 1.0, 0)


def test_a_server_without_a_top_k_cut_keeps_it_so():
    from zml_b200.serving.server import Server
    every = Server(_Engine(), _Tok(), strategy=SamplingStrategy(-1, 0.9))
    assert every._sampling({}) == (-1, 0.9, 0)
    assert every._sampling({"temperature": 0.5}) == (-1, 0.5, 0)
    assert every._sampling({"top_p": 1.0, "seed": 3}) == (-1, 0.9, 3)
    assert every._sampling({"temperature": 0.5, "top_p": 0.8}) == (0, 0.5, 0, 0.8, 0.0)
    assert every._sampling({"temperature": 0.5, "top_k": 7}) == (7, 0.5, 0)
    assert every._sampling({"temperature": 0}) == (1, 1.0, 0)


def test_settings_that_cut_nothing_do_not_ask_for_a_draw():
    from zml_b200.serving.server import Server
    greedy = Server(_Engine(), _Tok(), strategy=SamplingStrategy(1, 1.0, 0.9))      # greedy, with a nucleus for requests that draw
    for none in ({}, {"min_p": 0}, {"top_p": 1}, {"min_p": 0.0, "top_p": 1.0}):
        assert greedy._sampling(none) == (1, 1.0, 0)
    assert greedy._sampling({"temperature": 0.5, "min_p": 0}) == (0, 0.5, 0, 0.9, 0.0)
    assert greedy._sampling({"min_p": 0.1}) == (0, 1.0, 0, 0.9, 0.1)
    assert greedy._sampling({"top_p": 0.5}) == (0, 1.0, 0, 0.5, 0.0)
    nucleus = Server(_Engine(), _Tok(), strategy=SamplingStrategy(0, 0.7, 0.8))
    assert nucleus._sampling({"min_p": 0}) == (0, 0.7, 0, 0.8, 0.0) and nucleus._sampling({"top_p": 1}) == (128, 0.7, 0)
    assert Server(_Engine(), _Tok(), strategy=SamplingStrategy(40, 0.7))._sampling({"top_p": 1}) == (40, 0.7, 0)
    assert Server(_Engine(), _Tok(), strategy=SamplingStrategy(0))._sampling({}) == (0, 1.0, 0)


@pytest.mark.parametrize("device,vocab", [("cpu", 1000), ("cpu", 100), pytest.param("cuda", 100, marks=gpu)])
def test_a_top_k_that_gumbel_noise_takes_keeps_it(device, vocab):
    from zml_b200.models.decoder import DecoderModel
    from zml_b200.parallel.comm import Comm
    model = DecoderModel.__new__(DecoderModel)
    model.comm = Comm.single(torch.device(device))
    x = torch.randn((7, vocab), generator=torch.Generator().manual_seed(4)).to(device)
    rng = torch.tensor([11, 3], device=device)
    for k in (5, 128, 129, 200, 5000):
        for given in (None, rng):
            # (a counter on the CPU is the captured steps', which the CPU does not have)
            want = ops.topk_sample(x, k, 0.8, 11, 2, rng=given if device == "cuda" else None)
            assert torch.equal(model.sample(x, SamplingStrategy(k, 0.8), 11, 2, given), want)
    assert torch.equal(model.sample(x, SamplingStrategy(200, 0.8, 0.9), 11, 2, rng), ops.sample(x, None, 0.8, 200, 0.9, rng=rng))


@gpu
def test_a_wide_top_k_of_a_model_on_the_gpu():
    from zml_b200.models.decoder import DecoderModel
    from zml_b200.parallel.comm import Comm
    model = DecoderModel.__new__(DecoderModel)
    model.comm = Comm.single(torch.device("cuda"))
    x = torch.randn((7, 1000), generator=torch.Generator().manual_seed(4)).cuda()
    rng = torch.tensor([11, 3], device="cuda")
    for k in (129, 500, -1):
        assert torch.equal(model.sample(x, SamplingStrategy(k, 0.8), 11, 2, rng), ops.sample(x, None, 0.8, max(k, 0), rng=rng))
