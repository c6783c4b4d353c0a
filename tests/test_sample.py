"""The draw of tokens (ops.sample) against a restatement in 64 bits, row after row, that is written from the definition.

The kernel's weights are whole multiples of 2^-44 of the largest: each is off by 2^-45, so sums of n of them are off by n 2^-45 at most.  Where a uniform number lies
nearer than that to a border between tokens (or a nucleus ends nearer than that to top_p), another token is right, too; the oracle says how near it was.  Log-probabilities are
rounded to fp32 once: 2^-24 relative, and 2^-24 of what the weights' own error moves.
"""
import math

import pytest
import torch

from zml_b200 import ops
from zml_b200.ops import sampling

gpu = pytest.mark.gpu


def oracle(x, u, t, k, p, m):
    """One row in 64 bits: (token, log-probability, how near the nearest border was, as a part of the sum)."""
    x = [(-math.inf if math.isnan(v) else v) for v in x]
    top = max(x)
    if top == -math.inf:
        return 0, math.nan, 1.0
    first = x.index(top)
    if not t > 0 or p <= 0 or k == 1:
        return first, 0.0, 1.0
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    w = [1.0 if v == top else (math.exp((v - top) / t) if v > -math.inf and top < math.inf else 0.0) for v in x]
    if 0 < k < len(x):
        order = order[:k]
    near, stay = 1.0, order
    if p < 1:
        total, before, stay = math.fsum(w[i] for i in order), 0.0, []
        for i in order:
            if before >= p * total and stay:
                break
            near = min(near, abs(before - p * total) / total) if before else near
            stay.append(i)
            before += w[i]
        near = min(near, abs(before - p * total) / total)
    if m > 0:
        stay = [i for i in stay if w[i] >= min(m, 1.0)]
    stay = sorted(stay)
    total = math.fsum(w[i] for i in stay)
    u = min(max(u, 0.0), 1.0) if not math.isnan(u) else 0.0
    upto, token = 0.0, None
    for i in stay:
        upto += w[i]
        near = min(near, abs(upto - u * total) / total)
        if token is None and w[i] > 0 and upto > u * total:
            token = i
    if token is None:
        token = max(i for i in stay if w[i] > 0)
    return token, math.log(w[token] / total), near


def check(logits, uniforms, settings, device, dtype=torch.float32, most_near=0):
    """Draws from `logits` (a list of rows, or a tensor) on the device and compares all rows; returns how many were too near to a border to tell."""
    logits = torch.as_tensor(logits, dtype=torch.float32).to(dtype)
    rows, vocab = logits.shape
    uniforms = torch.as_tensor(uniforms, dtype=torch.float64)
    on = {n: (v.to(device) if isinstance(v, torch.Tensor) else v) for n, v in settings.items()}
    token, logprob = ops.sample(logits.to(device), uniforms.to(device), return_logprobs=True, **on)
    assert token.dtype is torch.int32 and token.shape == (rows,) and logprob.dtype is torch.float32
    near = 0
    for r in range(rows):
        one = {n: (v[r].item() if isinstance(v, torch.Tensor) else v) for n, v in settings.items()}
        want, lp, gap = oracle(logits[r].double().tolist(), float(uniforms[r]), one.get("temperature", 1.0), one.get("top_k", 0), one.get("top_p", 1.0),
                               one.get("min_p", 0.0))
        if 0.0 < gap < vocab * 2.0 ** -45:            # (weights that meet a border exactly are few whole numbers, in which nothing is rounded)
            near += 1
            continue
        assert int(token[r]) == want, (r, int(token[r]), want, one, gap)
        if math.isnan(lp):
            assert math.isnan(float(logprob[r]))
        else:
            assert abs(float(logprob[r]) - lp) <= 2.0 ** -23 * abs(lp) + vocab * 2.0 ** -44 + 2.0 ** -40, (r, float(logprob[r]), lp)
    assert near <= most_near
    return near


def spread(rows, vocab, sigma, seed, masked=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, vocab), generator=g) * sigma
    if masked:
        x[torch.rand((rows, vocab), generator=g) < masked] = -math.inf
        x[:, vocab // 2] = 0.0
    return x, torch.rand(rows, generator=g, dtype=torch.float64)


def mixed(rows, seed):
    g = torch.Generator().manual_seed(seed)
    pick = lambda v, d: torch.tensor(v, dtype=d)[torch.randint(0, len(v), (rows,), generator=g)]  # noqa: E731
    return {"temperature": pick([0.0, 0.3, 0.7, 1.0, 1.5, 4.0, -1.0, math.nan], torch.float32), "top_k": pick([0, 1, 2, 5, 40, 300, 5000, -3, 10 ** 6], torch.int32),
            "top_p": pick([1.0, 0.999, 0.9, 0.5, 0.1, 0.0, 2.0, math.nan, 1e-9], torch.float32),
            "min_p": pick([0.0, 0.05, 0.3, 1.0, 1e-6, -1.0, 2.0, math.nan], torch.float32)}


def suite(device, most=60000):
    nan, inf = math.nan, math.inf
    # ---- edges of the settings, ties and infinities, on short rows
    rows = [[1.0, 1.0, 1.0, 1.0], [0.0, 2.0, 2.0, -inf], [nan, 1.0, nan, 0.5], [-inf, -inf, 3.0, -inf], [inf, 1.0, inf, 0.0], [nan, -inf, nan, -inf],
            [-1e30, 1e30, 0.0, 1e30], [-0.0, 0.0, -0.0, 0.0], [1e-40, 0.0, -1e-40, 2e-40], [3e38, -3e38, 3e38, 2.9e38]]
    for settings in ({}, {"top_k": 2}, {"top_k": 3}, {"top_p": 0.5}, {"top_p": 0.25, "min_p": 0.2}, {"min_p": 1.0}, {"min_p": 0.5}, {"temperature": 0.0},
                     {"temperature": 1e-30}, {"temperature": 1e30}, {"temperature": inf}, {"temperature": nan}, {"top_k": 1}, {"top_p": 0.0},
                     {"top_p": -1.0}, {"top_p": 1e-300}, {"min_p": 7.0}, {"top_k": 2, "top_p": 0.6, "min_p": 0.3, "temperature": 0.5}, {"top_k": -1, "top_p": nan, "min_p": nan}):
        for u in (0.0, 0.13, 0.2499, 0.37, 0.62, 0.87, 1.0 - 2.0 ** -53, 1.0, -1.0, 5.0, nan):
            # (1 - 2^-53 and 1e-300 lie nearer to the sum's ends than its rounding)
            check(rows, [u] * len(rows), settings, device, most_near=len(rows) if u == 1.0 - 2.0 ** -53 or settings.get("top_p") == 1e-300 else 0)
    check([[5.0], [nan], [-inf]], [0.3, 0.3, 0.3], {"top_p": 0.5, "top_k": 3}, device)
    # ---- lengths, among them those that end inside a warp's row or a slice
    for vocab in (2, 3, 31, 127, 128, 129, 511, 2047, 2049, 4097, 16385, most):
        x, u = spread(3, vocab, 2.0, vocab)
        check(x, u, {"top_p": 0.9}, device)
        check(x, u, {"top_k": 7, "min_p": 0.01}, device)
    # ---- flat rows and many ties: cuts inside of them
    x = torch.zeros(6, 3001)
    x[:, 1500:] = 1.0
    u = [0.0, 0.1, 0.5, 0.77, 0.9, 0.9999]
    for settings in ({}, {"top_k": 1700}, {"top_k": 1000}, {"top_p": 0.6}, {"top_p": 0.95}, {"top_k": 2000, "top_p": 0.9}, {"min_p": 0.4}, {"min_p": 0.3}, {"top_k": 2500, "top_p": 0.99, "min_p": 0.2}):
        check(x, u, settings, device, most_near=1)
    # ---- everything together
    x, u = spread(64, 5003, 3.0, 5, masked=0.3)
    check(x, u, mixed(64, 6), device)
    x, u = spread(64, 700, 0.3, 7)
    check(x, u, mixed(64, 8), device)
    check(x, u, {**mixed(64, 9), "top_p": 0.8}, device, dtype=torch.bfloat16)
    # top_p is a part of the sum of the top_k, whatever min_p leaves of them
    check(x, u, {"top_k": 300, "top_p": 0.5, "min_p": 0.05, "temperature": 0.3}, device)
    check(x, u, {"top_k": 30, "top_p": 0.5, "min_p": 0.6}, device)
    # nearly the whole, and a tail of tiny weights
    x, u = spread(8, 4000, 6.0, 11)
    check(x, u, {"top_p": 1.0 - 2.0 ** -20}, device, most_near=4)      # the nucleus ends among weights of 1e-9, one in ten of them near
    x[:, 17] = 60.0
    check(x, u, {}, device)


def test_cpu():
    suite("cpu", 20000)


def test_uniforms_of_a_generator():
    x, _ = spread(5, 300, 1.0, 1)
    rng = torch.tensor([7, 3])
    want = ops.sample(x, torch.tensor([sampling.uniform(7, 3, r) for r in range(5)], dtype=torch.float64), top_p=0.9)
    assert torch.equal(ops.sample(x, rng=rng, top_p=0.9), want)
    n = [sampling.uniform(1, d, r) for d in range(100) for r in range(100)]
    assert min(n) >= 0 and max(n) < 1 and len(set(n)) == 10000 and abs(sum(n) / 10000 - 0.5) < 5 * 12 ** -0.5 / 100


def refusals(device):
    x, u = spread(3, 50, 1.0, 0)
    x, u = x.to(device), u.to(device)
    f32, i32 = dict(dtype=torch.float32, device=device), dict(dtype=torch.int32, device=device)
    for error, f in [
            (TypeError, lambda: ops.sample(x.double(), u)),
            (TypeError, lambda: ops.sample(x.half(), u)),
            (TypeError, lambda: ops.sample(x[0], u)),
            (ValueError, lambda: ops.sample(x[:, :0], u)),
            (ValueError, lambda: ops.sample(torch.zeros((1, 8 * 49152 + 1), **f32), u[:1])),
            (ValueError, lambda: ops.sample(x)),
            (ValueError, lambda: ops.sample(x, u, rng=torch.zeros(2, dtype=torch.int64, device=device))),
            (ValueError, lambda: ops.sample(x, u[:2])),
            (ValueError, lambda: ops.sample(x, u.half())),
            (ValueError, lambda: ops.sample(x, u[:, None])),
            (ValueError, lambda: ops.sample(x, rng=torch.zeros(2, **i32))),
            (ValueError, lambda: ops.sample(x, rng=torch.zeros(1, dtype=torch.int64, device=device))),
            (ValueError, lambda: ops.sample(x, u, temperature=torch.ones(2, **f32))),
            (ValueError, lambda: ops.sample(x, u, temperature=torch.ones(3, dtype=torch.float64, device=device))),
            (ValueError, lambda: ops.sample(x, u, top_k=torch.ones(3, **f32))),
            (ValueError, lambda: ops.sample(x, u, top_p=torch.ones(6, **f32)[::2])),
            (ValueError, lambda: ops.sample(x, u, min_p=torch.ones((3, 1), **f32))),
            (ValueError, lambda: ops.sample(x, u, out=torch.zeros(3, dtype=torch.int64, device=device))),
            (ValueError, lambda: ops.sample(x, u, out=torch.zeros(4, **i32)))]:
        with pytest.raises(error):
            f()


def test_refusals():
    refusals("cpu")


# ------------------------------------------------------------------ kernels
@gpu
def test_kernel():
    suite("cuda")
    ops.raise_on_status()


@gpu
@pytest.mark.parametrize("rows,vocab,dtype", [(1, 128256, torch.float32), (3, 151936, torch.bfloat16), (40, 65536, torch.float32), (300, 20000, torch.float32), (2, 248320, torch.float32),
                                              (1, 8 * 49152, torch.float32), (700, 1025, torch.bfloat16)])
def test_large(rows, vocab, dtype):
    """Against the restatement by sorting, which the CPU's tests hold to the definition; its borders are off by 2^-52 a term."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = (torch.randn((rows, vocab), device="cuda", generator=g) * 2.0).to(dtype)
    for settings in ({}, {"temperature": 3.0, "top_p": 0.97}, {"temperature": 0.2, "top_p": 0.5}, {"top_k": 50, "top_p": 0.95}, {"top_k": vocab // 2, "min_p": 1e-4}, {"top_k": 3000, "top_p": 0.9},
                     {"min_p": 0.02}):
        u = torch.rand(rows, device="cuda", generator=g, dtype=torch.float64)
        token, logprob = ops.sample(x, u, return_logprobs=True, **settings)
        want, lp = sampling._sample_cpu(x.cpu(), u.cpu(), *(settings.get(n, d) for n, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))), None)
        assert torch.equal(token.cpu(), want), (settings, (token.cpu() != want).sum())
        assert torch.allclose(logprob.cpu(), lp, rtol=2.0 ** -23, atol=vocab * 2.0 ** -44 + 2.0 ** -40)


@gpu
def test_strides_outputs_streams_and_repeats():
    x, u = spread(9, 5001, 2.0, 3)
    x, u = x.cuda(), u.cuda()
    want = ops.sample(x, u, top_p=0.9)
    wide = torch.full((9, 5004), 100.0, device="cuda")
    wide[:, 1:5002] = x
    assert torch.equal(ops.sample(wide[:, 1:5002], u, top_p=0.9), want)           # rows at any address, and nothing behind their end
    assert torch.equal(ops.sample(x.t().contiguous().t(), u, top_p=0.9), want)
    assert torch.equal(ops.sample(x[4:5].expand(9, -1), u, top_p=0.9)[4:5], want[4:5])
    out = torch.full((9,), -1, dtype=torch.int32, device="cuda")
    assert ops.sample(x, u, top_p=0.9, out=out) is out and torch.equal(out, want)
    assert torch.equal(ops.sample(x, u.float().double(), top_p=0.9), ops.sample(x, u.float(), top_p=0.9))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ops.sample(x, u, top_p=0.9)
    side.synchronize()
    assert torch.equal(again, want)
    for _ in range(20):
        assert torch.equal(ops.sample(x, u, top_p=0.9), want)
    assert ops.sample(x[:0], u[:0]).shape == (0,)


@gpu
def test_captured():
    x, u = spread(9, 5001, 2.0, 3)
    x, u = x.cuda(), u.cuda()
    rng = torch.tensor([5, 0], device="cuda")
    p = torch.full((9,), 0.9, device="cuda")
    ops.sample(x, u, top_p=p), ops.sample(x, rng=rng, top_p=p)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = ops.sample(x, u, top_p=p), ops.sample(x, rng=rng, top_p=p)
    for i, value in enumerate((0.9, 0.2, 1.0)):
        p.fill_(value)
        u.copy_(torch.rand(9, dtype=torch.float64))
        rng[1] = i
        graph.replay()
        assert torch.equal(a, ops.sample(x, u, top_p=value if value in (1.0,) else p))
        n = torch.tensor([sampling.uniform(5, i, r) for r in range(9)], dtype=torch.float64, device="cuda")
        assert torch.equal(b, ops.sample(x, n, top_p=p))


@gpu
def test_frequencies():
    """20000 draws of four tokens: each count within five standard deviations."""
    w = torch.tensor([0.5, 0.25, 0.2, 0.05])
    x = w.log().cuda().expand(20000, 4)
    got = torch.bincount(ops.sample(x, rng=torch.tensor([1, 2], device="cuda")), minlength=4).cpu()
    assert bool(((got - 20000 * w).abs() <= 5 * (20000 * w * (1 - w)).sqrt()).all())


@gpu
def test_refusals_on_the_gpu():
    refusals("cuda")
    x, u = spread(3, 50, 1.0, 0)
    with pytest.raises(ValueError):
        ops.sample(x.cuda(), u)
    with pytest.raises(ValueError):
        ops.sample(x.cuda(), u.cuda(), temperature=torch.ones(3))


def long_cuts(device, dtype=torch.float32):
    """Cuts that leave more than a list holds, or nearly so: of many logits, of few distinct ones, of many that are nearly alike, of such without weight."""
    vocab = 30000
    g = torch.Generator().manual_seed(5)
    alike = 1.0 + torch.randperm(vocab, generator=g).float() * 2.0 ** -22                   # all of one bin, and all different (in 32 bits)
    few = torch.tensor([0.0, 1e-3, 2e-3, -4.0])[torch.randint(0, 4, (vocab,), generator=g)]
    rows = torch.stack([spread(1, vocab, 2.5, 1)[0][0], spread(1, vocab, 0.4, 2)[0][0], alike, few, torch.zeros(vocab), spread(1, vocab, 2.0, 3, masked=0.7)[0][0]])
    u = torch.rand(len(rows), generator=g, dtype=torch.float64)
    for k in (0, 601, 1024, 1025, 2048, 2049, 9000, vocab - 1):
        for p in (1.0, 0.9, 0.4):
            check(rows, u, {"top_k": k, "top_p": p}, device, dtype)
    check(rows, u, {"top_k": 5000, "top_p": 0.97, "min_p": 0.02, "temperature": 1.3}, device, dtype)
    for p in (1.0, 0.999, 1.0 - 1e-9):
        near = len(rows) if p == 1.0 - 1e-9 else 0    # (what is behind this nucleus is as much as 30000 weights are rounded by: 8.5e-10)
        check(rows, u, {"top_k": 9000, "top_p": p, "temperature": 0.05}, device, dtype, near)      # the 9000th has no weight
        check(rows, u, {"top_p": p, "temperature": 0.3}, device, dtype, near)
    check(rows * 1e30, u, {"top_p": 0.6, "temperature": 1e30}, device, dtype)
    check(rows, u, {"top_k": 7000, "top_p": 0.6, "temperature": math.inf}, device, dtype)


def test_long_cuts_cpu():
    long_cuts("cpu")


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_cuts(dtype):
    long_cuts("cuda", dtype)
