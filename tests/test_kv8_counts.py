"""Attention of single tokens over the 8-bit cache where every key counts: values that say which keys were added up, and how often.

A value row has one number, in the column of its key's place, so that a column of the result is the share of the softmax that its keys have.  A tile that is
left out, or added up twice, changes a column by far more than a rounding does, however long the sequence is; that the check rejects such results is
tested beside it, on the CPU.
"""
import math

import pytest
import torch

from test_kv8 import DTYPES, E4M3, INT8, SHARED, gpu, paged, sequence64, shared_out
from test_kv8_extremes import check_closely
from zml_b200 import ops
from zml_b200.ops import kv8

# columns of n keys: neighbours share one, or those that are a row's length apart (the edge of a window is one key of few)
PATTERNS = {"blocks": lambda at, n, hd: at * hd // n, "stripes": lambda at, n, hd: at % hd}


def counting(lens, hq, hkv, hd, page, dtype, pattern, device, seed=5):
    """Keys with scores of a spread of 0.5, and values of 2^-3 to 2^3 times 8 to 15 eighths, which both types hold exactly."""
    k, v, table, sl = paged(lens, hkv, page, hd, dtype, seed, device, spread=0.5)
    g = torch.Generator().manual_seed(seed)
    for i, n in enumerate(lens):
        if n == 0:
            continue
        at = torch.arange(n)
        rows = torch.zeros(n, hkv, hd)
        size = torch.randint(8, 16, (n, hkv), generator=g).float() / 8 * torch.exp2(torch.randint(-3, 4, (n, hkv), generator=g).float())
        rows[at, :, PATTERNS[pattern](at, n, hd)] = size
        codes, exponents = kv8.quantize(rows, dtype)
        where, line = table[i, at // page].long().to(device), (at % page).to(device)
        v.codes.view(torch.uint8)[where, :, line] = codes.view(torch.uint8).to(device)
        v.exponents[where, :, line] = exponents.to(device)
    q = torch.randn(len(lens), hq, hd, generator=g).bfloat16().to(device)
    return q, k, v, table, sl


CASES = [(*c[:6], {**c[6], "bound": None}) for c in SHARED] + [
    # bounds other than the longest length, as engines give them: a CTA for each pair of many keys, and chunks of short ones
    ("cluster", [200, 5000, 2048, 33], 8, 2, 64, 64, dict(bound=1)),
    ("cluster", [200, 5000, 2048, 33], 8, 2, 256, 64, dict(bound=1, window=1000)),
    ("cluster", [128 + 61 * i for i in range(32)], 32, 8, 128, 64, dict(bound=2048)),
    ("chunks", [128 + 61 * i for i in range(32)], 32, 8, 128, 64, dict(bound=2560)),
    ("chunks", [300] * 64, 32, 8, 128, 64, dict(bound=4096)),
    ("cluster", [131072], 32, 8, 128, 64, dict(bound=4096)),
    ("chunks", [131072], 32, 8, 128, 64, dict(bound=None)),
]


@gpu
@DTYPES
@pytest.mark.parametrize("pattern", sorted(PATTERNS))
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}-{len(c[1])}x{c[2]}-{c[3]}x{c[4]}-{c[6]['bound']}")
def test_every_key_counts_once(case, pattern, dtype):
    kind, lens, hq, hkv, hd, page, more = case
    bound = max(lens) if more["bound"] is None else more["bound"]
    assert shared_out(lens, hq, hkv, hd, bound) == kind
    q, k, v, table, sl = counting(lens, hq, hkv, hd, page, dtype, pattern, "cuda")
    window = more.get("window", 0)
    out = ops.paged_decode(q, k, v, table, sl, window=window, max_seq_len=bound)
    which = [i for i, n in enumerate(lens) if n > 0]
    which = sorted(set(which[:6] + which[-3:] + sorted(which, key=lambda i: -lens[i])[:3]))
    check_closely(out, q, k, v, table, sl, 1 / math.sqrt(hd), which, dtype is INT8, window)
    ops.raise_on_status()


# ------------------------------------------------------------------ the check
def rejected(out, args, window):
    try:
        check_closely(out, *args, window)
    except AssertionError:
        return True
    return False


@pytest.mark.parametrize("dtype,n,hq,hkv,hd,window", [(E4M3, 300, 2, 1, 64, 0), (INT8, 2500, 4, 2, 64, 0), (E4M3, 9000, 2, 1, 128, 0), (INT8, 20000, 2, 1, 64, 0),
                                                      (E4M3, 20000, 2, 1, 256, 0), (E4M3, 5000, 2, 1, 64, 1500), (INT8, 5000, 2, 1, 256, 3000),
                                                      (INT8, 131072, 1, 1, 128, 0)])
def test_the_check_rejects_results_that_are_wrong(dtype, n, hq, hkv, hd, window):
    """The result in 64 bits, rounded, passes; results that lack a tile, or have one twice, or a wrong window, or another head's keys do not pass both patterns."""
    found = {}
    for pattern in PATTERNS:
        q, k, v, table, sl = counting([n], hq, hkv, hd, 64, dtype, pattern, "cpu")
        args = (q, k, v, table, sl, 1 / math.sqrt(hd), [0], dtype is INT8)
        ks, vs = sequence64(k, table[0], n), sequence64(v, table[0], n)
        group = hq // hkv
        p = torch.stack([torch.exp(ks[:, h // group] @ q[0, h].double() / math.sqrt(hd)) for h in range(hq)])      # [heads, keys]
        first = max(0, n - window) if window else 0
        ones = torch.zeros(n, dtype=torch.float64)
        ones[first:] = 1.0

        def result(num, den=None):
            den = num if den is None else den
            return torch.stack([((p[h] * num) @ vs[:, h // group]) / (p[h] * den).sum() for h in range(hq)])[None].bfloat16()

        def keys(a, b, factor):
            x = ones.clone()
            x[a:b] *= factor
            return x
        right = result(ones)
        tile, mid = (16 if hd == 256 else 32), first + (n - first) // 2 // 32 * 32
        last = (n - 1) // tile * tile
        wrong = {"zeros": torch.zeros_like(right), "0.9 of it": (0.9 * right.float()).bfloat16(), "the other sign": -right}
        for name, a, b in (("first", first, first + tile), ("middle", mid, mid + tile), ("last", min(last, n - 2), n), ("first sixteenth", first, first + (n - first) // 16)):
            for factor in (0.0, 2.0):
                wrong[f"{name} x {factor}"] = result(keys(a, b, factor))
                wrong[f"{name} x {factor}, summed without"] = result(keys(a, b, factor), ones)
        if window:
            for name, a in (("one key more", first - 1), ("one key less", first + 1)):
                x = torch.zeros_like(ones)
                x[a:] = 1.0
                wrong[name] = result(x)
        assert not rejected(right, args, window), pattern
        for name, out in wrong.items():
            found[name] = found.get(name, False) or rejected(out, args, window)
    assert all(found.values()), [name for name, yes in found.items() if not yes]
