"""The draw of tokens (ops.sample) from rows and settings at the ends of their types, against the restatement of test_sample.py."""
import math

import pytest
import torch

from test_sample import check
from zml_b200 import ops

gpu = pytest.mark.gpu
LOWEST = torch.finfo(torch.float32).min
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
UNIFORMS = (0.0, 0.13, 0.37, 0.62, 0.87)
CUTS = ({}, {"top_k": 2}, {"top_k": 40}, {"top_k": 1500}, {"top_p": 0.6}, {"top_k": 2, "top_p": 0.6}, {"top_k": 1500, "top_p": 0.7, "min_p": 0.5}, {"min_p": 0.3}, {"top_k": 1})


@pytest.mark.parametrize("device", DEVICES)
def test_rows_at_the_types_lowest_value(device):
    """Masked everywhere, by the lowest number, by it and -inf, or by sums with it: ties, among which -inf has no part."""
    inf = math.inf
    rows = [[LOWEST] * 4, [LOWEST, -inf, LOWEST, -inf], [-inf, LOWEST, -inf, -inf], [-3.4e38, LOWEST, -3.4e38, -inf], [-1e38, -inf, -1e38, -2e38], [-1e31, -1e30, -inf, -1e30]]
    for settings in CUTS:
        for t in (0.5, 0.7, 0.8, 1.0, 2.0, 0.0, 1e-30, 1e30, 1e36, 1e37, math.inf):
            for u in UNIFORMS:
                check(rows, [u] * len(rows), {**settings, "temperature": t}, device)
    for vocab in (1500, 5000, 30000):
        x = torch.full((4, vocab), LOWEST)
        x[1, ::3] = -inf
        x[2] = -inf
        x[2, vocab // 2:] = -1e38
        x[3, : vocab // 2] = torch.randn(vocab // 2, generator=torch.Generator().manual_seed(vocab))      # the usual row: masked in part
        for settings in CUTS:
            for t in (0.7, 1.0, 1e37):
                check(x, [0.11, 0.37, 0.62, 0.87], {**settings, "temperature": t}, device, most_near=1)


@pytest.mark.parametrize("device", DEVICES)
def test_large_logits_at_large_temperatures(device):
    rows = [[3e38, -3e38, 0.0, 1e38], [1e19, -1e19, 5e18, -math.inf], [-1e18, -3e18, -9e18, -1e30], [2.0, 1.0, -1e30, 0.0], [5.0, 1e17, -1e17, 3.0]]
    for t in (1e16, 1e18, 1e19, 1e29, 3e30, 1e31, 1e36, 1e37, 1e38, 3e38, math.inf):
        for settings in ({}, {"top_k": 3}, {"top_p": 0.6}, {"min_p": 0.5}):
            for u in UNIFORMS:
                check(rows, [u] * len(rows), {**settings, "temperature": t}, device)


@gpu
def test_no_row_is_left_without_a_token():
    x = torch.full((9, 3000), LOWEST, device="cuda")
    for settings in CUTS:
        out = torch.full((9,), -7, dtype=torch.int32, device="cuda")
        ops.sample(x, torch.rand(9, device="cuda"), 0.8, out=out, **settings)
        assert bool(((out >= 0) & (out < 3000)).all())


@pytest.mark.parametrize("device", DEVICES)
def test_a_largest_logit_of_zero_at_the_smallest_temperatures(device):
    rows = [[0.0, -1.0, -1e-3, -1e-45], [-1.0, -0.0, -1e-40, -math.inf], [-5.0, 0.0, 0.0, -1e-45], [1e-45, 0.0, -1.0, -1e-45], [-1e-45, -2e-45, -1.0, -1e-40]]
    for t in (1e-44, 1e-46, 1e-48, 1e-60, 1e-100, 1e-300, 5e-324):
        for settings in ({}, {"top_k": 3}, {"top_p": 0.9}, {"min_p": 1e-3}, {"top_k": 3, "top_p": 0.9}):
            for u in UNIFORMS:
                check(rows, [u] * len(rows), {**settings, "temperature": t}, device)
    x = -torch.rand((2, 5000), generator=torch.Generator().manual_seed(1))
    x[:, 4321] = 0.0
    for settings in CUTS:
        check(x, [0.1, 0.9], {**settings, "temperature": 1e-60}, device)


@gpu
@pytest.mark.parametrize("vocab,longer", [(50257, 65536), (50304, 65536), (16385, 32000), (100352, 128256)])
def test_no_length_leaves_the_list(vocab, longer):
    """A draw with a small top_k ends in a list, for every length of a row: it takes about as long as that of a longer row (up to 1.4 times where rows do
    not start on 16 bytes), and not twice and more, as where CTAs without logits left no bound."""
    def took(n, rows):
        x = torch.randn((rows, n), device="cuda", generator=torch.Generator(device="cuda").manual_seed(n)) * 2.5
        u = torch.rand(rows, device="cuda")
        ops.sample(x, u, 1.0, 50)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(20):
                ops.sample(x, u, 1.0, 50)
        graph.replay()
        best = math.inf
        for _ in range(10):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            graph.replay()
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best
    for rows in (1, 32):
        assert took(vocab, rows) < 1.75 * took(longer, rows)
