"""Prompts that begin with the same pages, and nucleus sampling, through the engine and its server."""
import pytest
import torch

from zml_b200 import ops
from zml_b200.models.common import SamplingStrategy
from zml_b200.models.llama import PRESETS, AttnMeta, LlamaConfig, LlamaModel
from zml_b200.serving import Engine
from zml_b200.serving.engine import OutOfPages
from zml_b200.serving.server import Server

PAGE = 16
NUCLEUS = SamplingStrategy(topk=0, temperature=0.8, top_p=0.9)


def _model(device="cpu", dtype=torch.float32, **more):
    cfg = LlamaConfig.from_hf(dict(PRESETS["tiny-llama-test"], **more))
    return LlamaModel(cfg, device=device, dtype=dtype).init_random(seed=1, std=0.08)


def _engine(model, share, pages=64, **more):
    more = dict(dict(page_size=PAGE, max_batch=8, max_seq_len=256, max_prefill_tokens=48), **more)
    eng = Engine(model, num_pages=pages, share_prefixes=share, **more)
    eng.SHARE_BYTES = 0                  # small models share keys of a few kilobytes
    return eng


def _prompts(vocab, prefixes=(40, 33), seed=0):
    """Two families behind their own beginnings, one prompt twice, one that is its family's beginning, and one by itself."""
    g = torch.Generator().manual_seed(seed)
    draw = lambda n: torch.randint(0, vocab, (n,), generator=g).tolist()
    a, b = draw(prefixes[0]), draw(prefixes[1])
    return [a + draw(3), b + draw(20), a + draw(9), draw(37), a, b + draw(1), a + draw(3)] + [a]


def _count_groups(eng):
    """Records whether each decode step of the engine reads its keys in groups."""
    seen, shared = [], eng._shared
    eng._shared = lambda b: seen.append(shared(b)) or seen[-1]
    return seen


def test_generate_and_serve_give_the_answers_of_the_plain_engine():
    model = _model()
    prompts = _prompts(model.config.vocab_size)
    # The random numbers go by the number of forward calls, and pages that are there need fewer portions of 48 tokens: with draws both
    # engines take their prompts in one call.
    for strategy, portion in ((None, 48), (SamplingStrategy(topk=5, temperature=0.7), 512), (NUCLEUS, 512)):
        want, _ = _engine(model, False, max_prefill_tokens=portion).generate(prompts, 7, strategy, seed=3)
        eng = _engine(model, True, max_prefill_tokens=portion)
        seen = _count_groups(eng)
        got, _ = eng.generate(prompts, 7, strategy, seed=3)
        assert got == want and any(s is not None for s in seen)
        assert eng.pool.num_free == 63 and not eng.pool.more and not eng._prefixes and not eng._prefix_of
    budgets = [3, 9, 1, 6, 8, 2, 7, 5]
    want, _ = _engine(model, False).serve(prompts, budgets, sync_interval=2)
    eng = _engine(model, True, max_batch=3)                      # rows that change their sequences, families that come and go
    got, _ = eng.serve(prompts, budgets, sync_interval=2)
    assert got == want and eng.pool.num_free == 63 and not eng._prefixes
    got, _ = _engine(model, True).serve(prompts, budgets, sync_interval=1, arrivals=[0, 0, 1, 1, 2, 3, 4, 6])
    assert got == want


def test_nucleus_strategies_follow_their_seed():
    model = _model()
    prompts = _prompts(model.config.vocab_size)[:4]
    a, _ = _engine(model, False).generate(prompts, 6, NUCLEUS, seed=5)
    b, _ = _engine(model, False).generate(prompts, 6, NUCLEUS, seed=5)
    c, _ = _engine(model, False).generate(prompts, 6, NUCLEUS, seed=6)
    assert a == b and a != c
    greedy, _ = _engine(model, False).generate(prompts, 6)
    for narrow in (SamplingStrategy(0, 1.0, 0.0), SamplingStrategy(0, 1.0, 1.0, 1.0), SamplingStrategy(1, 1.0, 0.5)):
        assert _engine(model, False).generate(prompts, 6, narrow, seed=9)[0] == greedy       # one token is left
    assert not SamplingStrategy().cuts and not SamplingStrategy(0).cuts and not SamplingStrategy(128).cuts and not SamplingStrategy(1, 1.0, 0.5).draws
    assert SamplingStrategy(129).cuts and SamplingStrategy(-1).cuts and SamplingStrategy(5).draws and NUCLEUS.draws


def test_pages_are_held_once_and_given_back_by_their_last_holder():
    model = _model()
    eng = _engine(model, True)
    a, tail = list(range(40)), [1, 2, 3]
    first = eng.new_request(a, 8, share=True)                    # 48 tokens: 3 pages
    assert eng.pool.num_free == 60
    second = eng.new_request(a + tail, 5, share=True)            # the same, 2 pages of them shared
    assert second.pages[:2] == first.pages[:2] and second.pages[2] != first.pages[2] and eng.pool.num_free == 59
    assert second.common == 2 and second.computed == 32
    alone = eng.new_request(a, 8)                                # not asked to share
    assert not set(alone.pages) & set(first.pages) and alone.common == 0
    eng.release(first)
    assert eng.pool.num_free == 57                               # its last page only
    third = eng.new_request(a, 8, share=True)
    assert third.pages[:2] == second.pages[:2]
    for r in (second, third, alone):
        eng.release(r)
    assert eng.pool.num_free == 63 and not eng.pool.more and not eng._prefixes and not eng._prefix_of
    # a prompt that ends with a page: its last token has to be computed, so its last page is its own
    r = eng.new_request(a[:32], 4, share=True)
    s = eng.new_request(a[:32], 4, share=True)
    assert s.common == 1 and s.pages[0] == r.pages[0] and s.pages[1] != r.pages[1]
    # the same page behind another one is not the same keys
    t = eng.new_request(a[16:32] + a[16:32] + [5], 4, share=True)
    assert t.common == 0
    short = eng.new_request(a[:16], 4, share=True)
    assert short.common == 0
    for x in (r, s, t, short):
        eng.release(x)
    # one that does not fit leaves no holder behind
    full = _engine(model, True, pages=6)
    x = full.new_request(a, 8, share=True)
    with pytest.raises(OutOfPages):
        full.new_request(a + list(range(60)), 8, share=True)
    assert not full.pool.more and full.pool.num_free == 2
    full.release(x)
    assert full.pool.num_free == 5 and not full._prefixes


def test_an_error_leaves_no_uncomputed_page_to_later_requests(monkeypatch):
    model = _model()
    prompts = _prompts(model.config.vocab_size)
    want, _ = _engine(model, False).generate(prompts, 4)
    for call in ("generate", "serve"):
        eng = _engine(model, True)
        hidden = model.hidden_states
        with monkeypatch.context() as m:
            m.setattr(model, "hidden_states", lambda *a: (_ for _ in ()).throw(RuntimeError("lost")))
            with pytest.raises(RuntimeError, match="lost"):
                getattr(eng, call)(prompts, 4)
        assert not eng._prefixes and not eng._prefix_of
        assert model.hidden_states == hidden
        eng2 = eng if eng.pool.num_free >= 40 else _engine(model, True)
        assert eng2.generate(prompts, 4)[0] == want


def test_groups_of_a_step():
    model = _model()
    eng = _engine(model, True)
    a = list(range(96))
    b = a[:16] + list(range(200, 290))

    def groups(prompts):
        reqs = [eng.new_request(p, 4, share=True) for p in prompts]
        host = eng._share_groups(list(enumerate(reqs)))
        for r in reqs:
            eng.release(r)
        if host is None:
            return None
        members, starts, lens = host.tolist()
        out, g = [], 0
        while starts[g + 1] > starts[g]:
            out.append((sorted(members[starts[g]:starts[g + 1]]), lens[g]))
            g += 1
        assert all(s == starts[g] for s in starts[g:]) and not any(lens[g:])
        return out
    # everybody's beginning is a's first page, but the two pairs have 6 pages each: 6 + 6 are more than 3 x 1
    assert sorted(groups([a + [1], b + [1], a + [2], b + [2]])) == [([0, 2], 96), ([1, 3], 96)]
    # one of them short: the pair spares 6 pages, all three together 2
    assert groups([a + [1], a[:16] + [7] * 20, a + [2]]) == [([0, 2], 96)]
    # five of them short: the pair's 6 pages and theirs, 4 x 2, are more than all seven's, 6 x 2
    assert sorted(groups([a + [1]] + [a[:32] + [i] * 20 for i in range(5)] + [a + [2]])) == [([0, 6], 96), ([1, 2, 3, 4, 5], 32)]
    # five a little shorter: 6 + 4 x 5 are less than 6 x 5
    assert groups([a + [1]] + [a[:80] + [i] * 20 for i in range(5)] + [a + [2]]) == [(list(range(7)), 80)]
    assert groups([a + [1], b + [1] * 3]) == [([0, 1], 16)]
    eng.SHARE_BYTES = 1
    assert groups([a, list(range(300, 340))]) is None
    eng.SHARE_BYTES = 96 * eng._key_bytes()
    assert groups([a + [1], a + [2]]) == [([0, 1], 96)]
    eng.SHARE_BYTES += 1
    assert groups([a + [1], a + [2]]) is None


def test_sharing_is_refused_where_it_does_not_hold():
    model = _model()
    with pytest.raises(ValueError, match="8 bits"):
        Engine(_model(dtype=torch.bfloat16), 16, page_size=64, kv_dtype="fp8", share_prefixes=True)
    windowed = _model()
    windowed.config.sliding_window = 32
    with pytest.raises(ValueError, match="window"):
        Engine(windowed, 16, share_prefixes=True)
    model.attn_backend = "vanilla"
    with pytest.raises(ValueError, match="vanilla"):
        Engine(model, 16, share_prefixes=True)
    model = _model()
    model.SHARED_PREFIX = False                                  # as every model that does not say that its attention takes groups
    with pytest.raises(ValueError, match="does not share"):
        Engine(model, 16, share_prefixes=True)


def test_server_takes_top_p_and_min_p():
    class Recorder:
        max_pages, page_size, comm = 8, 16, None

        def __init__(self):
            self.calls = []

        def serve(self, prompts, budgets, strategy, eos_ids, seed=0, on_tokens=None):
            self.calls.append((len(prompts), strategy, seed))
            return [[1] * b for b in budgets], None

    class Tok:
        def decode(self, ids, *a):
            return "x" * len(ids)
    plain = Server(Recorder(), Tok())
    assert plain._sampling({}) == (1, 1.0, 0)
    assert plain._sampling({"top_p": 1, "min_p": 0}) == (1, 1.0, 0)                      # neither cuts
    assert plain._sampling({"top_p": 0.9}) == (0, 1.0, 0, 0.9, 0.0)
    assert plain._sampling({"min_p": 0.05, "temperature": 0.5, "seed": 7}) == (0, 0.5, 7, 1.0, 0.05)
    assert plain._sampling({"top_p": 0.9, "top_k": 500}) == (500, 1.0, 0, 0.9, 0.0)
    assert plain._sampling({"top_p": 0.9, "top_k": -1}) == (0, 1.0, 0, 0.9, 0.0)
    assert plain._sampling({"top_p": 0.9, "top_k": 1}) == (1, 1.0, 0)
    assert plain._sampling({"top_p": 0.9, "temperature": 0}) == (1, 1.0, 0)
    assert plain._sampling({"top_p": 0.12345}) == (0, 1.0, 0, 0.123, 0.0)
    assert plain._sampling({"top_p": 1.0, "temperature": 0.7}) == (128, 0.7, 0)
    warm = Server(Recorder(), Tok(), strategy=SamplingStrategy(0, 0.7, 0.8))
    assert warm._sampling({}) == (0, 0.7, 0, 0.8, 0.0) and warm._sampling({"min_p": 0.1}) == (0, 0.7, 0, 0.8, 0.1)
    assert warm._sampling({"top_p": 1.0}) == (128, 0.7, 0) and warm._sampling({"temperature": 0}) == (1, 1.0, 0)
    assert Server(Recorder(), Tok(), strategy=SamplingStrategy(40, 0.7, 0.8))._sampling({"top_p": 0.5}) == (40, 0.7, 0, 0.5, 0.0)
    for bad in ({"top_p": -0.1}, {"top_p": 1.5}, {"top_p": "0.9"}, {"min_p": True}, {"min_p": float("nan")}, {"top_p": [0.9]}):
        with pytest.raises(ValueError, match="a number from 0 to 1"):
            plain._sampling(bad)
    rs = [plain.submit({"prompt": [1, 2], "max_tokens": 2, **more}, False) for more in ({"top_p": 0.9, "seed": 4}, {}, {"top_p": 0.9, "seed": 4})]
    while not all(r.done.is_set() for r in rs):
        plain.step()
    assert plain.engine.calls == [(2, SamplingStrategy(0, 1.0, 0.9, 0.0), 4), (1, SamplingStrategy(), 0)]


_TP_WORKER = r"""
import torch
from zml_b200.models.common import SamplingStrategy
from zml_b200.models.llama import PRESETS, LlamaConfig, LlamaModel
from zml_b200.parallel.comm import Comm
from zml_b200.serving import Engine
c = Comm.from_env(backend="gloo")
cfg = LlamaConfig.from_hf(PRESETS["tiny-llama-test"])
outs = []
for comm in (c, Comm.single(torch.device("cpu"))):
    model = LlamaModel(cfg, comm, device="cpu", dtype=torch.float32).init_random(seed=2, std=0.08)
    eng = Engine(model, num_pages=64, page_size=16, max_batch=4, max_seq_len=128, share_prefixes=True)
    eng.SHARE_BYTES = 0
    g = torch.Generator().manual_seed(3)
    a = torch.randint(0, cfg.vocab_size, (35,), generator=g).tolist()
    outs.append(eng.generate([a + [1], a + [2, 3], a], 6, SamplingStrategy(0, 0.8, 0.95), seed=11)[0])
assert outs[0] == outs[1], outs
print("SHARED_TP_OK", c.rank, flush=True)
c.finish(0)
"""


def test_two_tensor_parallel_ranks_draw_the_tokens_of_one(tmp_path):
    import os
    import subprocess
    import sys
    script = tmp_path / "w.py"
    script.write_text(_TP_WORKER)
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node=2", "--master-addr", "127.0.0.1",
                        "--master-port", "29683", str(script)], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, PYTHONPATH=root))
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-3000:]
    assert r.stdout.count("SHARED_TP_OK") == 2


def _logits(model, ids):
    """Logits of every position of one sequence, computed as a prompt."""
    t, dev = len(ids), model.device
    pages = -(-t // PAGE)
    i32 = dict(dtype=torch.int32, device=dev)
    pos = torch.arange(t, **i32)
    kv = torch.zeros(model.kv_cache_shape(pages + 1, PAGE), dtype=model.dtype, device=dev)
    meta = AttnMeta(True, pos, pos + PAGE, torch.arange(1, pages + 1, **i32)[None], torch.tensor([t], **i32), torch.tensor([0, t], **i32),
                    total_q_blocks=-(-t // 64))
    return model.logits(model.hidden_states(torch.tensor(ids, **i32), meta, kv), pos.long()).float()


@pytest.mark.gpu
def test_engine_on_the_gpu_shares_keys_in_captured_and_eager_steps():
    model = _model("cuda", torch.bfloat16)
    prompts = _prompts(model.config.vocab_size, (100, 200))
    budgets = [3, 9, 1, 6, 8, 2, 7, 5]
    outs = {}
    for graphs in (True, False):
        eng = _engine(model, True, pages=128, max_seq_len=512, use_graphs=graphs)
        seen = _count_groups(eng)
        outs[graphs] = [eng.generate(prompts, 9)[0], eng.generate(prompts, 9)[0], eng.serve(prompts, budgets, sync_interval=2)[0],
                        eng.generate(prompts, 9, NUCLEUS, seed=2)[0], eng.generate(prompts, 9, NUCLEUS, seed=2)[0]]
        assert any(s is not None for s in seen) and eng.pool.num_free == 127
    assert outs[True] == outs[False]                             # a replay and an eager step run the same kernels
    assert outs[True][0] == outs[True][1] and outs[True][3] == outs[True][4]
    # A greedy token is the largest logit up to what two orders of computing the hidden state differ by: 5e-2 on either side, as in the
    # other tests of this model's logits against another computation of them.
    for p, o in zip(prompts, outs[True][0]):
        lg = _logits(model, p + o)[len(p) - 1:len(p) + len(o) - 1]
        picked = lg.gather(1, torch.tensor(o, device="cuda")[:, None])[:, 0]
        assert bool((picked >= lg.amax(1) - 0.1).all())
    ops.raise_on_status()
    with pytest.raises(ValueError, match="shared pages are for"):
        Engine(model, 16, page_size=8, share_prefixes=True)


@pytest.mark.gpu
def test_attention_and_draw_captured_together():
    """One decode step's tail as a server runs it: attention behind two shared beginnings, the head, a draw - captured once and replayed with
    other lengths, other groups and other numbers."""
    torch.manual_seed(0)
    b, hq, hkv, hd, page, vocab, pages = 6, 8, 2, 64, 16, 1000, 40
    dev = dict(device="cuda")
    q = torch.randn(b, hq, hd, dtype=torch.bfloat16, **dev)
    kc, vc = (torch.randn(pages, page, hkv, hd, dtype=torch.bfloat16, **dev) for _ in range(2))
    head = torch.randn(vocab, hq * hd, dtype=torch.bfloat16, **dev) * 0.1
    u = torch.rand(b, **dev)
    table = torch.arange(10, **dev).int().repeat(b, 1)
    table[3:] += 10
    table[:, 8:] = 20 + 2 * torch.arange(b, **dev).int()[:, None] + torch.arange(2, **dev).int()
    lens = torch.full((b,), 8 * page + 9, dtype=torch.int32, **dev)
    rows, starts = torch.arange(b, **dev).int(), torch.tensor([0, 3, 6, 6, 6, 6, 6], **dev).int()
    plens = torch.tensor([8 * page, 8 * page, 0, 0, 0, 0], **dev).int()

    def run():
        a = ops.paged_decode(q, kc, vc, table, lens, shared=ops.SharedPrefix(rows, starts, plens))
        lg = ops.gemm(a.reshape(b, hq * hd), head, out_dtype=torch.float32)
        return a, lg, *ops.sample(lg, u, 0.8, 50, 0.9, return_logprobs=True)
    eager = run()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    graph.replay()
    assert all(torch.equal(x, y) for x, y in zip(out, eager))
    lens.sub_(9)                                                 # nothing behind the beginnings
    starts.copy_(torch.tensor([0, 2, 4, 6, 6, 6, 6]))            # rows 2 and 3 do not share a page and one page only: other groups
    table[2:4, :8] = torch.arange(8, **dev).int()
    u.uniform_()
    graph.replay()
    torch.cuda.synchronize()
    again = run()
    assert all(torch.equal(x, y) for x, y in zip(out, again))
    plain = ops.paged_decode(q, kc, vc, table, lens)
    # two roundings to bf16 of sums of values up to 4: half a step each, and the weights' rounding of the same size in both
    assert float((plain.float() - again[0].float()).abs().max()) <= 4 * 4 * 2 ** -8
    ops.raise_on_status()
