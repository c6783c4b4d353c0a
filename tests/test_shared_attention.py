"""Attention of single tokens behind a shared prefix (ops.shared) against softmax attention in 64 bits, sequence after sequence.

A weight is rounded to bf16 once and so is the output: half a step each, 2^-8 relative.  A score's product of hd terms is summed in fp32: hd additions
of at most 2^-23 of the sum of magnitudes (the tensor core cuts where an addition would round), which moves a weight by as much times the scale.
"""
import math
import random

import pytest
import torch

from zml_b200 import ops

gpu = pytest.mark.gpu


def make(groups, alone=(), hq=8, hkv=2, hd=64, page=64, seed=0, device="cpu", nan_behind=True, strided=False):
    """groups: [(keys that are shared, [keys of their own of every member])]; alone: keys of sequences in no group, 0 for none."""
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    seqs = [(i, p, p + n) for i, (p, own) in enumerate(groups) for n in own] + [(-1, 0, n) for n in alone]
    rng.shuffle(seqs)
    b = len(seqs)
    width = max(1, max(-(-n // page) for _, _, n in seqs)) + 1
    need = 2 + sum(p // page for p, _ in groups) + sum(-(-n // page) for _, _, n in seqs)
    order = list(range(need))
    rng.shuffle(order)
    common = [[order.pop() for _ in range(p // page)] for p, _ in groups]
    k = torch.randn((need, page, hkv, hd), generator=g) * torch.exp(0.5 * torch.randn((1, 1, hkv, hd), generator=g))
    v = torch.randn((need, page, hkv, hd), generator=g)
    k, v = k.bfloat16(), v.bfloat16()
    table = torch.full((b, width), order[0], dtype=torch.int32)
    first = {}
    for i, (gr, p, n) in enumerate(seqs):
        pages = list(common[gr]) if gr >= 0 else []
        pages += [order.pop() for _ in range(-(-n // page) - len(pages))]
        table[i, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
        rest = p % page
        if rest and gr >= 0:                          # the page that the prefix fills in part: the same keys in each member's own
            if gr in first:
                for c in (k, v):
                    c[pages[p // page], :rest] = c[first[gr], :rest]
            first.setdefault(gr, pages[p // page])
        if nan_behind and n % page:
            k[pages[-1], n % page:] = math.nan
            v[pages[-1], n % page:] = math.inf
    q = torch.randn((b, hq + 3 if strided else hq, hd), generator=g).bfloat16().to(device)[:, :hq]
    shared = ops.SharedPrefix.of([([i for i, s in enumerate(seqs) if s[0] == j], p) for j, (p, _) in enumerate(groups)], device)
    lens = torch.tensor([n for _, _, n in seqs], dtype=torch.int32)
    return {"q": q, "k": k.to(device), "v": v.to(device), "table": table.to(device), "lens": lens.to(device), "shared": shared}


def oracle(s, scale=None):
    """(out, attention over |v|, largest sum of |q k| scale) in 64 bits."""
    q, k, v, table, lens = (s[n].cpu() for n in ("q", "k", "v", "table", "lens"))
    hkv, hd, page = k.shape[2], k.shape[3], k.shape[1]
    scale = hd ** -0.5 if scale is None else scale
    out, mag, most = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64), 0.0
    for i, n in enumerate(lens.tolist()):
        if n <= 0:
            continue
        at = table[i, :-(-n // page)].long()
        kk, vv = (c[at].flatten(0, 1)[:n].double().permute(1, 0, 2) for c in (k, v))
        qq = q[i].double().unflatten(0, (hkv, -1))
        p = torch.softmax(qq @ kk.mT * scale, -1)
        out[i], mag[i] = (p @ vv).flatten(0, 1), (p @ vv.abs()).flatten(0, 1)
        most = max(most, float((qq.abs() @ kk.abs().mT).max()) * scale)
    return out, mag, most


def check(got, s, scale=None):
    out, mag, most = oracle(s, scale)
    rel = 2.0 ** -8 + 2 * most * s["k"].shape[3] * 2.0 ** -23 + 2.0 ** -16
    err = (got.cpu().double() - out).abs()
    assert bool((err <= rel * mag + 2.0 ** -8 * out.abs() + 1e-30).all()), float((err / mag.clamp_min(1e-30)).max())


def call(s, **more):
    return ops.paged_decode(s["q"], s["k"], s["v"], s["table"], s["lens"], shared=s["shared"], **more)


# ------------------------------------------------------------------ without a GPU
def test_cpu_is_plain_attention():
    s = make([(70, [0, 1, 9]), (128, [5, 64])], alone=(0, 3))
    s["k"], s["v"] = s["k"].nan_to_num(0, 0, 0), s["v"].nan_to_num(0, 0, 0)
    check(call(s), s)
    assert not call(s)[s["lens"] == 0].any()


def test_groups_from_lists():
    p = ops.SharedPrefix.of([([3, 1], 64), ([], 5), ([0], 7)])
    assert p.rows.tolist() == [3, 1, 0] and p.starts.tolist() == [0, 2, 2, 3] and p.lens.tolist() == [64, 5, 7]


def refusals(s):
    q, k, v, table, lens, shared = (s[n] for n in ("q", "k", "v", "table", "lens", "shared"))
    b = q.shape[0]
    go = lambda q=q, k=k, v=v, t=table, n=lens, p=shared, **m: ops.paged_decode(q, k, v, t, n, shared=p, **m)  # noqa: E731
    for error, f in [
            (TypeError, lambda: go(p=(shared.rows, shared.starts, shared.lens))),
            (ValueError, lambda: go(window=5)),
            (ValueError, lambda: go(ext=object())),
            (ValueError, lambda: go(scale=0.0)),
            (ValueError, lambda: go(scale=-1.0)),
            (ValueError, lambda: go(scale=math.nan)),
            (ValueError, lambda: go(scale=math.inf)),
            (ValueError, lambda: go(q=q[:, :7])),
            (ValueError, lambda: go(q=q[..., :32])),
            (ValueError, lambda: go(q=q[:, 0])),
            (ValueError, lambda: go(k=k[:, :48], v=v[:, :48])),
            (ValueError, lambda: go(k=k[:, :8], v=v[:, :8])),
            (ValueError, lambda: go(v=v[:-1])),
            (ValueError, lambda: go(k=k[:0], v=v[:0])),
            (ValueError, lambda: go(k=k.transpose(0, 1).contiguous().transpose(0, 1))),
            (ValueError, lambda: go(t=table.long())),
            (ValueError, lambda: go(t=table[:-1])),
            (ValueError, lambda: go(t=table[:, :0])),
            (ValueError, lambda: go(t=table[:, ::2])),
            (ValueError, lambda: go(n=lens.long())),
            (ValueError, lambda: go(n=lens[:-1])),
            (ValueError, lambda: go(out=torch.empty_like(q, dtype=torch.float32))),
            (ValueError, lambda: go(out=torch.empty_like(q[:-1]))),
            (ValueError, lambda: go(p=ops.SharedPrefix.of([(list(range(b)) + [0], 5)], q.device))),
            (ValueError, lambda: go(p=ops.SharedPrefix.of([([], 5)] * (b + 1), q.device))),
            (ValueError, lambda: ops.SharedPrefix(shared.rows.long(), shared.starts, shared.lens)),
            (ValueError, lambda: ops.SharedPrefix(shared.rows, shared.starts[1:], shared.lens)),
            (ValueError, lambda: ops.SharedPrefix(shared.rows[:, None], shared.starts, shared.lens))]:
        with pytest.raises(error):
            f()


def test_refusals():
    refusals(make([(70, [0, 1, 9])]))


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
def test_refuses_quantised_caches(dtype):
    s = make([(70, [0, 1, 9])])
    c = ops.QuantKV.alloc(s["k"].shape[0], 2, 64, 64, torch.int8 if dtype == "int8" else torch.float8_e4m3fn)
    with pytest.raises(ValueError):
        ops.paged_decode(s["q"], c, c, s["table"], s["lens"], shared=s["shared"])


# ------------------------------------------------------------------ kernels
SIZES = [
    ([(1, [0])], (), 1, 1, 64, 64),
    ([(64, [1, 1])], (), 2, 1, 128, 64),
    ([(63, [0, 1, 2])], (0, 1), 8, 2, 128, 64),
    ([(1000, [0, 5, 64, 700])], (), 32, 8, 128, 64),
    ([(65, [7, 0, 129]), (128, [3]), (500, [200, 1])], (0, 90), 32, 8, 64, 64),
    ([(130, [2] * 5)], (1,), 16, 4, 256, 64),
    ([(777, list(range(0, 200, 20)))], (), 20, 4, 128, 16),
    ([(333, [5, 0, 40])], (17, 0), 12, 1, 64, 32),
    ([(500, [1, 300])], (), 8, 2, 256, 128),
    ([(500, [1, 300])], (), 8, 2, 64, 192),
    ([(260, [3, 4, 0])], (12,), 14, 2, 128, 64),            # groups of seven heads: rows of a tile are 126
    ([(200, [3, 4, 0])], (12,), 128, 1, 64, 64),            # a tile a sequence
    ([(200, [3, 4, 0])], (12,), 66, 1, 128, 16),
    ([(96, [1, 2, 3])] * 9, (), 4, 4, 128, 32),
    ([(5, [1])] * 40, (3,) * 20, 8, 2, 64, 64),
    ([(4000, [i % 7 for i in range(70)])], (), 8, 2, 128, 64),      # several tiles of rows
    ([], (1, 64, 65, 300, 0), 8, 2, 128, 64),               # nothing is shared
    ([(0, [1, 64, 300])], (), 8, 2, 128, 64),
]


@gpu
@pytest.mark.parametrize("case", SIZES, ids=[str(i) for i in range(len(SIZES))])
def test_sizes(case):
    groups, alone, hq, hkv, hd, page = case
    s = make(groups, alone, hq, hkv, hd, page, seed=len(groups) + hq, device="cuda")
    got = call(s)
    ops.raise_on_status()
    check(got, s)
    assert not got[s["lens"] == 0].any()


@gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_many_tiles_for_every_cta(hd):
    s = make([(9000, [10, 800, 0]), (5000, [64, 1, 300, 77])], (2000, 1), 16, 8, hd, 64, device="cuda")
    got = call(s)
    ops.raise_on_status()
    check(got, s)


@gpu
def test_a_thousand_sequences():
    s = make([(64, [i % 5 for i in range(500)])], tuple(i % 3 for i in range(524)), 4, 2, 64, 16, device="cuda")
    got = call(s)
    ops.raise_on_status()
    check(got, s)


@gpu
def test_large_and_small_scores():
    s = make([(700, [0, 100, 300])], (65,), 8, 2, 128, 64, device="cuda")
    s["q"] *= 30.0
    check(call(s), s)
    check(call(s, scale=1e-3), s, 1e-3)
    s["k"][:, ::2] *= 8.0                             # the maximum rises late
    check(call(s), s)
    ops.raise_on_status()


@gpu
def test_strides_outputs_and_streams():
    s = make([(300, [1, 40, 65])], (0,), 8, 2, 128, 64, device="cuda", strided=True)
    assert s["q"].stride(0) == 11 * 128
    want = call(s)
    check(want, s)
    odd = torch.zeros(s["q"].numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view(4, 8, 128)
    assert call(s, out=odd) is odd and torch.equal(odd, want)
    out = torch.empty_like(want)
    assert call(s, out=out) is out and torch.equal(out, want)
    t = torch.zeros(s["q"].numel() + 4, dtype=torch.bfloat16, device="cuda")[4:].view(4, 8, 128)      # rows that start on 8 bytes
    t.copy_(s["q"])
    assert torch.equal(call({**s, "q": t}), want)
    perm = s["q"].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(call({**s, "q": perm}), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = call(s)
    side.synchronize()
    assert torch.equal(again, want)
    ops.raise_on_status()


@gpu
def test_same_as_without_sharing():
    s = make([(700, [10, 100, 300]), (64, [1, 2])], (65,), 32, 8, 128, 64, device="cuda", nan_behind=False)
    plain = ops.paged_decode(s["q"], s["k"], s["v"], s["table"], s["lens"])
    check(call(s), s)
    check(plain, s)


@gpu
def test_a_captured_call_follows_lengths_and_groups():
    s = make([(500, [10, 100, 300]), (130, [1, 2])], (65, 0), 8, 2, 128, 64, device="cuda", nan_behind=False)
    out = torch.empty_like(s["q"])
    call(s, out=out)
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(s, out=out)
    second = torch.empty_like(out)
    with torch.cuda.graph(other):
        call(s, out=second)
    p = s["shared"]
    for rows, starts, lens, seq in [
            (p.rows.tolist(), p.starts.tolist(), p.lens.tolist(), s["lens"].tolist()),
            (p.rows.tolist(), p.starts.tolist(), [448, 128], [max(0, n - 1) for n in s["lens"].tolist()]),
            (p.rows.tolist(), [0, 0, 0], [0, 0], s["lens"].tolist()),
            (p.rows.tolist(), [0, 3, 3], [64, 9], s["lens"].tolist())]:
        p.rows.copy_(torch.tensor(rows)), p.starts.copy_(torch.tensor(starts)), p.lens.copy_(torch.tensor(lens)), s["lens"].copy_(torch.tensor(seq))
        out.fill_(7.0), second.fill_(7.0)
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        check(out, s)
        assert torch.equal(out, second)
    ops.raise_on_status()


@gpu
def test_results_repeat():
    s = make([(3000, [i for i in range(30)])], (), 32, 8, 128, 64, device="cuda")
    first = call(s)
    for _ in range(20):
        assert torch.equal(call(s), first)


@gpu
def test_lists_that_say_nonsense_touch_no_other_memory():
    """Members outside of the batch, offsets out of order, lengths below zero or beyond the table, sequences in two groups: the outputs mean nothing then, but rows of
    sequences that are in no group do."""
    s = make([(130, [3, 4, 5])], (70, 9), 8, 2, 64, 64, device="cuda", nan_behind=False)
    i32 = dict(dtype=torch.int32, device="cuda")
    rows = s["shared"].rows.tolist()
    free = [i for i in range(5) if i not in rows]
    out, _, _ = oracle(s)
    for r, st, n in [([-5, 77, rows[0]], [0, 3], [130]), (rows, [2, -4], [130]), (rows, [0, 900], [10 ** 6]), (rows, [0, 3], [-5]),
                     ([rows[0]] * 3, [0, 3], [130]), (rows, [0, 2, 1, 3], [130, 64, 64]), (rows, [0, 3, 0, 3], [130, 10, 20])]:
        got = call({**s, "shared": ops.SharedPrefix(torch.tensor(r, **i32), torch.tensor(st, **i32), torch.tensor(n, **i32))})
        ops.raise_on_status()
        assert torch.allclose(got[free].cpu().double(), out[free], atol=0.05)
    bad = {**s, "lens": s["lens"].clone()}
    bad["lens"][free[0]] = -3
    bad["lens"][rows[0]] = 10 ** 7                    # as many as the table has
    assert not call(bad)[free[0]].any()
    ops.raise_on_status()


@gpu
def test_refusals_on_the_gpu():
    s = make([(70, [0, 1, 9])], device="cuda")
    refusals(s)
    with pytest.raises(TypeError):
        call({**s, "q": s["q"].float()})
    with pytest.raises(ValueError):
        call({**s, "table": s["table"].cpu()})
    with pytest.raises(ValueError):
        call({**s, "shared": ops.SharedPrefix.of([([0], 5)])})
    flat = torch.zeros(s["k"].numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view(s["k"].shape)
    with pytest.raises(ValueError):
        call({**s, "k": flat})
    empty = call({**s, "q": s["q"][:0], "table": s["table"][:0], "lens": s["lens"][:0], "shared": ops.SharedPrefix.of([], "cuda")})
    assert empty.shape == (0, 8, 64)


@gpu
def test_a_sequence_that_is_listed_twice_is_where_it_is_listed_last():
    s = make([(256, [3, 40, 5, 0, 70, 9])], (70,), 8, 2, 64, 64, device="cuda")
    a = s["shared"].rows.tolist()
    for groups in ([(a[:5], 256), ([a[2], a[4]], 128)], [(a[:2], 64), (a[1:], 256)], [(a[:3] + a[:2], 256)], [([a[0]] * 7, 256)]):
        check(call({**s, "shared": ops.SharedPrefix.of(groups, "cuda")}), s)
    s["lens"][:] = 256                                # nothing of their own
    got = call({**s, "shared": ops.SharedPrefix.of([(a[:4], 192), ([a[3], a[1]], 64)], "cuda")})
    check(got[a], {**s, "q": s["q"][a], "table": s["table"][a], "lens": s["lens"][a]})
    ops.raise_on_status()
