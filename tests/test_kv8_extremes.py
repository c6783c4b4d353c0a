"""The 8-bit key / value cache where numbers are very large, very small or far apart, and where bounds that a caller gives are wrong.

Oracles are restatements in 64 bits; tolerances are derived beside their tests.  A rounding to a format is off by at most half a step: 2^-8 relative in
bf16, 2^-11 in f16.
"""
import pytest
import torch

from test_kv8 import DTYPES, gpu, values64
from zml_b200 import ops


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
