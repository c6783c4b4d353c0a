"""The 8-bit key / value cache where numbers are very large, very small or far apart, and where bounds that a caller gives are wrong.

Oracles are restatements in 64 bits; tolerances are derived beside their tests.  A rounding to a format is off by at most half a step: 2^-8 relative in
bf16, 2^-11 in f16.
"""
import os
import subprocess
import sys
import threading
import time

import pytest
import torch

from test_kv8 import DTYPES, E4M3, INT8, gpu, paged, sequence64, values64
from zml_b200 import ops
from zml_b200.ops import kv8


# ------------------------------------------------------------------ reader
def read_back(cache, rows):
    """The first `rows` rows of page 0 through `ops.paged_read`: [rows, heads, hd]."""
    i32 = dict(dtype=torch.int32, device=cache.device)
    return ops.paged_read(cache, cache, torch.zeros(1, 1, **i32), torch.tensor([rows], **i32))[0][0, :rows]


LARGE_BYTES = [27, 40, 100, 150, 200, 220, 228, 230, 231, 232, 233, 236, 240, 244, 246, 248]


def check_every_code(dtype, device):
    """All 256 codes under scales up to the largest that a row is written with.  Exact, as codes times a power of two are bf16 numbers, where that is below
    2^128 (beyond: infinities, which no row that was written holds)."""
    codes = torch.arange(256, dtype=torch.uint8).view(1, 4, 1, 64).repeat(1, 1, 16, 1).contiguous().view(dtype).to(device)
    exps = torch.tensor(LARGE_BYTES, dtype=torch.uint8).view(1, 1, 16).repeat(1, 4, 1).contiguous().to(device)
    cache = ops.QuantKV(codes, exps)
    want = values64(cache)[0].transpose(0, 1)
    want = torch.where(want.abs() >= 2.0 ** 128, torch.copysign(torch.full_like(want, float("inf")), want), want)
    assert torch.equal(read_back(cache, 16).double().nan_to_num(nan=-1.5, posinf=1e300, neginf=-1e300), want.nan_to_num(nan=-1.5, posinf=1e300, neginf=-1e300))


@DTYPES
def test_every_code_under_large_scales_cpu(dtype):
    check_every_code(dtype, "cpu")


@gpu
@DTYPES
def test_every_code_under_large_scales(dtype):
    check_every_code(dtype, "cuda")
    ops.raise_on_status()


# ------------------------------------------------------------------ attention of single tokens
def shared_out(lens, hq, hkv, hd, bound):
    parts, _ = kv8._plan(0, len(lens), hq, hkv, hd, bound)
    return "chunks" if parts > 0 else "warp" if parts == 0 else "cluster"


# lengths, the bound of them that the launch is planned by: a warp, one CTA, or chunks take the first sequence, tiles in turn among the warps of a CTA
WAYS = pytest.mark.parametrize("kind,lens,bound", [("warp", [200] * 310, 200), ("cluster", [200], 1), ("chunks", [200, 20000, 33, 2500], 20000)],
                               ids=["warp", "cluster", "chunks"])


def sequences(lens, hkv, hd, dtype, device, page=64):
    """A cache in which sequence i holds the pages after those of sequence i - 1, all of it zeros: keys, values, table, lengths, first page of each."""
    held = [-(-n // page) for n in lens]
    first = [sum(held[:i]) for i in range(len(lens))]
    table = torch.zeros(len(lens), max(held), dtype=torch.int32)
    for i, (a, m) in enumerate(zip(first, held)):
        table[i, :m] = torch.arange(a, a + m, dtype=torch.int32)
    k, v = (ops.QuantKV.alloc(sum(held), hkv, page, hd, dtype, device) for _ in range(2))
    k.exponents.fill_(127)
    v.exponents.fill_(127)
    return k, v, table.to(device), torch.tensor(lens, dtype=torch.int32, device=device), first


def put(cache, first, keys, rows):
    """Rows `keys` of the one head of the sequence whose pages begin at `first`."""
    codes, exponents = kv8.quantize(rows.float(), cache.codes.dtype)
    page, at = (first + keys // 64).to(cache.device), (keys % 64).to(cache.device)
    cache.codes.view(torch.uint8)[page, 0, at] = codes.view(torch.uint8).to(cache.device)
    cache.exponents[page, 0, at] = exponents.to(cache.device)


def scale_of_log2(x):
    """A float32 scale whose product with log2(e), in float32, is x."""
    f = torch.tensor(x / 1.4426950408889634, dtype=torch.float32)
    for _ in range(8):
        if float(f * torch.tensor(1.4426950408889634)) == x:
            return float(f)
        f = torch.nextafter(f, torch.tensor(float("inf")) if float(f * torch.tensor(1.4426950408889634)) < x else torch.tensor(0.0))
    raise AssertionError("no such scale")


@gpu
@DTYPES
@pytest.mark.parametrize("hd", [64, 128, 256])
@WAYS
def test_scores_where_fp32_counts_in_sixteens(kind, lens, bound, hd, dtype):
    """Scores of 2^27 + 16 and, later in the same warp, 2^27 + 32, in units of log2: the second key outweighs the first by 2^16, more than f16 holds over the
    slack that weights have.  Both scores are exact: 8 x 64 x 2^14 and one or two, times 16.  What is left of the first key is 2^-16, and the second value is
    rounded as a weight (2^-11) and to bf16 (2^-8)."""
    assert shared_out(lens, 1, 1, hd, bound) == kind
    k, v, table, sl, first = sequences(lens, 1, hd, dtype, "cuda")
    near = torch.zeros(hd)
    near[:8], near[8] = 64.0, 1.0
    far = near.clone()
    far[8] = 2.0
    g = torch.Generator().manual_seed(3)
    va, vb = (kv8._values(*kv8.quantize(torch.randn(hd, generator=g), dtype)) for _ in range(2))
    later = 4 * (16 if hd == 256 else 32) + 7
    put(k, first[0], torch.tensor([5, later]), torch.stack([near, far]))
    put(v, first[0], torch.tensor([5, later]), torch.stack([va, vb]))
    q = torch.zeros(len(lens), 1, hd, dtype=torch.bfloat16, device="cuda")
    q[:, 0, :8], q[:, 0, 8] = 2.0 ** 14, 1.0
    out = ops.paged_decode(q, k, v, table, sl, scale=scale_of_log2(16.0), max_seq_len=bound)[0, 0].double().cpu()
    va, vb = va.double(), vb.double()
    assert bool(((out - vb).abs() <= (2.0 ** -8 + 2.0 ** -11) * vb.abs() + 2.0 ** -15 * (va.abs() + vb.abs())).all()), out
    ops.raise_on_status()


def check_closely(out, q, k, v, table, lens, scale, which, int8, window=0):
    """Rows `which` of a decode call against 64 bits, each key with its own share of the tolerance.

    bf16 rounds the result (2^-8); a weight is rounded to f16 (2^-11), or lies among f16's subnormals (half a step of 2^-24, where the largest p s_v
    of the row is 2^7 or more): 2^-32 of the largest p s_v, times a code.  A score is a sum of hd products in fp32 and three roundings, (hd + 8) 2^-24 of the sum of
    their magnitudes; queries beside int8 keys are rounded to half a unit where the row's largest is 2^14 or more (2^-15), so a score is off by that
    times the sum of the key's magnitudes.  exp2 gives 2^-21; a key's error acts on the sum of values and on the sum of weights.  Weights below 2^-126 of the
    reference, which is up to 2^8 below the largest, may vanish."""
    hd, hkv = q.shape[2], k.codes.shape[1]
    group = q.shape[1] // hkv
    most_code = 128.0 if int8 else 448.0
    for i in which:
        n = int(lens[i])
        ks, vs = sequence64(k, table[i], n), sequence64(v, table[i], n)
        scales = torch.exp2(v.exponents[table[i, :-(-n // v.page_size)].long()].double() - 127.0).transpose(1, 2).reshape(-1, hkv)[:n]
        first = max(0, n - window) if window else 0
        n, ks, vs, scales = n - first, ks[first:], vs[first:], scales[first:]
        for h in range(q.shape[1]):
            kh, vh, qh = ks[:, h // group], vs[:, h // group], q[i, h].double()
            delta = (hd + 8) * 2.0 ** -24 * abs(scale) * (kh.abs() @ qh.abs()) + 2.0 ** -21
            if int8:
                delta = delta + 2.0 ** -15 * float(qh.abs().max()) * abs(scale) * kh.abs().sum(-1)
            p = torch.softmax((kh @ qh) * scale, 0)
            want, mag = p @ vh, p @ vh.abs()
            gone = torch.where(p < 2.0 ** -116 * p.max(), p, 0.0) @ vh.abs()
            tol = (2.0 ** -8 * want.abs() + 2.0 ** -11 * mag + (p * delta) @ vh.abs() + (p @ delta) * mag + gone
                   + n * 2.0 ** -32 * most_code * float((p * scales[:, h // group]).max()) + 2.0 ** -130)
            err = (out[i, h].double() - want).abs()
            assert bool((err <= tol).all()), (i, h, float((err / tol).max()), float((err - tol).max()))


@gpu
@DTYPES
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("up", [26, 40, 100])
@WAYS
def test_large_values_that_nobody_looks_at(kind, lens, bound, up, hd, dtype):
    """One value row is 2^up times as large as the others, and its key's score 60 below theirs or far lower: it must not cost the others their digits (2^100 and
    60 below, it is what the result is made of).  A second query head of the same key head looks at that key and at no other."""
    assert shared_out(lens, 2, 1, hd, bound) == kind
    g = torch.Generator().manual_seed(up + hd)
    n = lens[0]
    for place in (0, 70, n - 1):
        for low in (60.0, 600.0):
            k, v, table, sl, first = sequences(lens, 1, hd, dtype, "cuda")
            ks, vs = torch.randn(n, hd, generator=g) * 0.1, torch.randn(n, hd, generator=g)
            ks[:, 0] = 0.0
            ks[place] = 0.0
            ks[place, 0] = -low                           # a code times a power of two
            vs[place] *= 2.0 ** up
            put(k, first[0], torch.arange(n), ks)
            put(v, first[0], torch.arange(n), vs)
            q = torch.randn(len(lens), 2, hd, generator=g).bfloat16()
            q[:, 0, 0], q[:, 1, 0] = 1.0, -1.0
            q = q.cuda()
            out = ops.paged_decode(q, k, v, table, sl, scale=1.0, max_seq_len=bound)
            check_closely(out, q, k, v, table, sl, 1.0, [0], dtype is INT8)
    ops.raise_on_status()


@gpu
@DTYPES
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("step,down", [(12.0, 5.0), (12.0, 17.0), (12.0, 30.0), (-12.0, -5.0), (-12.0, -30.0), (0.3, 1.0), (0.3, -1.0), (7.0, 0.0)])
@pytest.mark.parametrize("hq", [3, 12])
@WAYS
def test_scores_and_values_that_climb_and_fall(kind, lens, bound, hq, step, down, hd, dtype):
    """Along a sequence scores rise by `step` (in units of log2) every 13 keys while values shrink by 2^down: what the weights are taken from moves with
    nearly every tile, in both directions, and the first or the last keys make the result."""
    assert shared_out(lens, hq, 1, hd, bound) == kind
    g = torch.Generator().manual_seed(hd)
    n = lens[0]
    k, v, table, sl, first = sequences(lens, 1, hd, dtype, "cuda")
    ks, vs = torch.randn(n, hd, generator=g) * 0.05, torch.randn(n, hd, generator=g)
    at = torch.arange(n) // 13
    ks[:, 0] = (step * at.float()).bfloat16().float()
    vs *= torch.exp2(-down * (at.float() - 7.0))[:, None].clamp(2.0 ** -110, 2.0 ** 110)
    put(k, first[0], torch.arange(n), ks)
    put(v, first[0], torch.arange(n), vs)
    q = torch.randn(len(lens), hq, hd, generator=g).bfloat16()
    q[:, :, 0] = torch.tensor([1.0, 0.25, -1.0]).repeat(hq // 3)
    q = q.cuda()
    out = ops.paged_decode(q, k, v, table, sl, scale=0.6931471805599453, max_seq_len=bound)
    check_closely(out, q, k, v, table, sl, 0.6931471805599453, [0], dtype is INT8)
    ops.raise_on_status()


# ------------------------------------------------------------------ writer
TOP = [3.3895313892515355e38, 3.3762e38, 3.36e38, 3.3e38, 3.29e38, 3.2e38, 2.99e38, 2.98e38, 2.9e38, 1.7e38, 1e38]


def check_top(cache, x):
    """Rows x [tokens, heads, hd] of finite numbers up to bf16's largest: they stand for finite numbers, within half a step, or within a whole one where the
    next step would be 2^128."""
    got = values64(cache)[0, :, :x.shape[0]].transpose(0, 1).cpu()
    back = read_back(cache, x.shape[0]).double().cpu()
    assert torch.equal(got, back) and bool((back.abs() < 2.0 ** 128).all())
    s = torch.exp2(cache.exponents[0, :, :x.shape[0]].t().double().cpu() - 127.0)[..., None]
    x = x.double().cpu()
    step = s * torch.ones_like(x)
    if cache.codes.dtype is E4M3:
        step = s * torch.exp2(torch.floor(torch.log2((x.abs() / s).clamp_min(2.0 ** -6)))) / 8
    full = (back.abs() + step) >= 2.0 ** 128
    assert bool(((x - back).abs() <= torch.where(full, step, step / 2)).all())


def top_rows():
    x = torch.randn(2 * len(TOP), 1, 64, generator=torch.Generator().manual_seed(1)) * 1e37
    for i, t in enumerate(TOP):
        x[2 * i, 0, 7 * i % 64], x[2 * i + 1, 0, (11 * i + 3) % 64] = t, -t
    return x.bfloat16()


@DTYPES
def test_rows_up_to_the_largest_number_stay_finite_cpu(dtype):
    x = top_rows()
    cache = ops.QuantKV.alloc(1, 1, 32, 64, dtype)
    codes, exps = kv8.quantize(x[:, 0], dtype)
    cache.codes.view(torch.uint8)[0, 0, :len(x)], cache.exponents[0, 0, :len(x)] = codes.view(torch.uint8), exps
    check_top(cache, x)


@gpu
@DTYPES
@pytest.mark.parametrize("shift", [0, 1])
def test_rows_up_to_the_largest_number_stay_finite(dtype, shift):
    x = top_rows()
    n = len(x)
    buf = torch.zeros(n, 3 * 64 + 8, dtype=torch.bfloat16, device="cuda")
    qkv = buf[:, shift:shift + 3 * 64]
    qkv[:, 64:128], qkv[:, 128:] = x[:, 0].cuda(), x[:, 0].cuda()
    k, v = (ops.QuantKV.alloc(1, 1, 32, 64, dtype, "cuda") for _ in range(2))
    ids = torch.arange(n, dtype=torch.int32, device="cuda")
    ops.rope_kvwrite(qkv, torch.zeros_like(ids), ids, torch.ones(32, device="cuda"), k, v, 1, 1, 64)
    check_top(k, x)                                       # position 0 turns nothing
    check_top(v, x)
    codes, exps = kv8.quantize(x[:, 0], dtype)
    for c in (k, v):
        assert torch.equal(c.codes.view(torch.uint8)[0, 0, :n].cpu(), codes.view(torch.uint8)) and torch.equal(c.exponents[0, 0, :n].cpu(), exps)
    ops.raise_on_status()


# ------------------------------------------------------------------ prompts
@DTYPES
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_a_bound_of_the_lengths_that_is_too_small_changes_nothing(device, dtype):
    """`max_seq_len` chooses the kernel of `ops.paged_prefill`, whatever the cache."""
    k, v, table, sl = paged([300, 70, 500], 2, 64, 128, dtype, 5, device)
    q = torch.randn(30, 4, 128, generator=torch.Generator().manual_seed(4)).bfloat16().to(device)
    starts = torch.tensor([0, 10, 20, 30], dtype=torch.int32, device=device)
    want = ops.paged_prefill(q, k, v, table, sl, starts, impl="mma")
    for bound in (1, 64, 100, 10 ** 6):
        assert torch.equal(ops.paged_prefill(q, k, v, table, sl, starts, max_seq_len=bound, impl="mma"), want)
    if device != "cpu":
        ops.raise_on_status()


@gpu
@pytest.mark.parametrize("page", [16, 64, 128])
def test_sequences_that_the_workspace_has_no_room_for(page):
    """`kv_pages` below what the sequences hold: reported, and those that do not fit have outputs of zero and see nobody else's keys.  The first ones are
    as they were."""
    lens = [130, 70, 500]
    k, v, table, sl = paged(lens, 2, page, 128, E4M3, 5, "cuda")
    q = torch.randn(30, 4, 128, generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
    starts = torch.tensor([0, 10, 20, 30], dtype=torch.int32, device="cuda")
    want = ops.paged_prefill(q, k, v, table, sl, starts)
    ops.raise_on_status()
    for total, whole in ((256, 2), (128, 2), (0, 1)):                            # tokens of the pages; room for 64 more behind each sequence
        got = ops.paged_prefill(q, k, v, table, sl, starts, kv_pages=total // page)
        with pytest.raises(ops.KernelError):
            ops.raise_on_status()
        assert torch.equal(got[:10 * whole], want[:10 * whole]) and not bool(got[10 * whole:].any())


def test_sequences_that_the_workspace_has_no_room_for_cpu():
    k, v, table, sl = paged([130, 70], 2, 64, 64, E4M3, 5)
    q = torch.randn(4, 4, 64).bfloat16()
    with pytest.raises(ValueError):
        ops.paged_prefill(q, k, v, table, sl, torch.tensor([0, 2, 4], dtype=torch.int32), kv_pages=4)


@DTYPES
@pytest.mark.parametrize("group,hd", [(1, 64), (2, 64), (2, 128), (1, 256)])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_prompts_over_a_table_without_columns(device, group, hd, dtype):
    """New tokens of sequences that have no pages at all see nothing: the bf16 kernels are given a table with a column, which they read whatever the lengths are."""
    k, v, _, _ = paged([5, 9], 2, 64, hd, dtype, 5, device)
    i32 = dict(dtype=torch.int32, device=device)
    q = torch.ones(320, 2 * group, hd, dtype=torch.bfloat16, device=device)
    out = ops.paged_prefill(q, k, v, torch.zeros(2, 0, **i32), torch.tensor([0, 3], **i32), torch.tensor([0, 1, 320], **i32))
    assert out.shape == q.shape and not bool(out.any())
    if device != "cpu":
        assert kv8._read(k, v, torch.zeros(2, 0, **i32), torch.tensor([0, 3], **i32), 64, 1, 1)[2].tolist() == [[0], [0]]
        ops.raise_on_status()


# ------------------------------------------------------------------ tickets of captured calls
def test_captures_in_several_threads_draw_different_tickets(monkeypatch):
    """What a captured call takes of the stock is its own, wherever threads take turns: the stock's counter gives way whenever it is written."""
    class Slow(list):
        def __setitem__(self, at, value):
            super().__setitem__(at, value)
            time.sleep(1e-4)

    stock = Slow([torch.zeros(1 << 16, dtype=torch.int32), 0])
    monkeypatch.setattr(kv8, "_CAPTURED", {0: stock})
    monkeypatch.setattr(kv8, "_capturing", lambda: True)
    got, q = [], torch.zeros(1)

    def capture():
        for n in range(1, 40):
            t = kv8._tickets(q, 0, 0, n)
            got.append((t.data_ptr(), t.data_ptr() + 4 * t.numel()))

    threads = [threading.Thread(target=capture) for _ in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    got.sort()
    assert len(got) == 6 * 39 and all(a[1] <= b[0] for a, b in zip(got, got[1:]))
    assert got[0][0] == stock[0].data_ptr() and got[-1][1] <= stock[0].data_ptr() + 4 * (1 << 16)


# ------------------------------------------------------------------ the bounds-checking build
_BOUNDS_WORKER = """
import torch
from zml_b200 import ops
from zml_b200.models.llama import PRESETS, LlamaConfig, LlamaModel
from zml_b200.ops import _lib
from zml_b200.serving import Engine
assert _lib.bounds_check_build()
m = LlamaModel(LlamaConfig.from_hf(dict(PRESETS["tiny-llama-test"])), device="cuda").init_random(seed=3, std=0.05)
for page, pages in ((128, 7), (16, 40), (320, 3), (64, 11)):
    prompts = [[(7 * i + j) % 1000 for i in range(n)] for j, n in enumerate((300, 50, 129) if page != 320 else (500,))]
    e = Engine(m, num_pages=pages, page_size=page, max_batch=4, max_seq_len=640, kv_dtype="fp8", use_graphs=False)
    outs = e.generate(prompts, max_new_tokens=3)[0]
    assert all(len(o) == 3 for o in outs)
    ops.raise_on_status()
print("CLEAN", flush=True)
"""


@gpu
def test_the_bounds_checking_build_knows_the_pages_of_the_copy(tmp_path):
    """Attention over prompts reads a copy in pages of 64 tokens, of which there are more than pages of 128 in the cache: page numbers of the copy are no
    offence."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    so = os.path.join(root, "zml_b200", "_C", "libzb_cuda_bc.so")
    if not os.path.exists(so):
        from zml_b200 import _build
        _build.build_cuda(extra_flags=["-DZB_BOUNDS_CHECK", "-rdc=true"], variant="bc")
    script = tmp_path / "w.py"
    script.write_text(_BOUNDS_WORKER)
    r = subprocess.run([sys.executable, str(script)], capture_output=True, text=True, timeout=600, env={**os.environ, "ZB_CUDA_LIB": so, "PYTHONPATH": root})
    assert r.returncode == 0 and "CLEAN" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]
