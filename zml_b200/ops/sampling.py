"""The draw of one token for each row of logits, with settings of every row's own.

With weights w_i = exp((x_i - max x) / temperature), in this order:

* only the `top_k` largest logits stay (0 or less: all; of equal logits those of lower index);
* of these, from the largest down, a token stays while the weights in front of it are less than `top_p` of the sum of all (the first one always; 1 or
  more: all);
* and while w_i >= `min_p` (the largest always; 0 or less: all);
* the token is the first one, in the vocabulary's order, up to which the weights that stayed sum to more than `uniform` times their whole sum.

A temperature that is not above zero takes the first of the largest logits.  A NaN among the logits counts as -inf, which is never drawn; a
row without anything else gives token 0 with a log-probability of NaN.  A NaN among the settings switches the cut off (as a temperature: takes the first of
the largest).  Numbers outside of [0, 1) draw the first or the last token that stayed.

`nn.sampling.sample_tokens_dynamic` cuts at the reference's border instead: there a token stays while the sum up to AND INCLUDING it is at most
`top_p` (zml/nn.zig:2121-2159).  Here it is the smallest set that reaches `top_p`, as servers' interfaces have it.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Optional

import torch

from . import _lib

_lib.register_signature("zb_sample", C.c_int, [C.c_void_p])
_CALL = struct.Struct("10P q 3d 5i 4x").pack                              # ZbSample (csrc/sample.cu)

MAX_VOCAB = 8 * 49152
_current = getattr(torch._C, "_cuda_getDevice", None)                     # absent in builds of torch without CUDA
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _check(name, value, dtype, rows: int, index: int) -> int:
    """The address of a setting per row, 0 for a number."""
    if not isinstance(value, torch.Tensor):
        return 0
    if value.dtype is not dtype or value.shape != (rows,) or value.get_device() != index or not value.is_contiguous():
        raise ValueError(f"{name}: a number, or {rows} contiguous numbers of {dtype} on the logits' device, got {value.dtype} {tuple(value.shape)} on "
                         f"{value.device}")
    return value.data_ptr()


def sample(logits, uniforms=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, return_logprobs: bool = False, rng=None, out=None):
    """Tokens int32 [rows] drawn from float32 or bfloat16 logits [rows, vocab]; with `return_logprobs` also float32 [rows], the logarithms of the
    probabilities that they were drawn with (after all cuts).

    `uniforms`: float32 or float64 [rows] in [0, 1).  Without them `rng`, int64 {seed, draws so far} on the logits' device, whose numbers are a function
    of seed, draws and row; the counter is the caller's to advance (`advance_rng`).
    `temperature`, `top_p`, `min_p`: numbers, or float32 [rows]; `top_k`: a number, or int32 [rows].  See the module for what they cut.
    Weights are sums of 2^-44 of the largest: two runs draw the same, whatever the order of the additions.  (A token of less than 2^-45 is not drawn.)"""
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"logits [rows, vocab] in float32 or bfloat16, got {logits.dtype} {tuple(logits.shape)}")
    rows, vocab = logits.shape
    index = logits.get_device()
    if not 0 < vocab <= MAX_VOCAB:
        raise ValueError(f"a vocabulary of 1 to {MAX_VOCAB} tokens, got {vocab}")
    if (uniforms is None) == (rng is None):
        raise ValueError("either uniforms or rng")
    if uniforms is not None:
        if (uniforms.dtype is not torch.float32 and uniforms.dtype is not torch.float64) or uniforms.shape != (rows,) or uniforms.get_device() != index \
                or not uniforms.is_contiguous():
            raise ValueError(f"uniforms: {rows} contiguous float32 or float64 numbers on {logits.device}, got {uniforms.dtype} {tuple(uniforms.shape)} on "
                             f"{uniforms.device}")
    elif rng.dtype is not torch.int64 or rng.numel() < 2 or rng.get_device() != index or not rng.is_contiguous():
        raise ValueError(f"rng: int64 {{seed, draws so far}} on {logits.device}")
    f32 = torch.float32
    at = (_check("temperature", temperature, f32, rows, index), _check("top_p", top_p, f32, rows, index), _check("min_p", min_p, f32, rows, index),
          _check("top_k", top_k, torch.int32, rows, index))
    if out is not None and (out.dtype is not torch.int32 or out.shape != (rows,) or out.get_device() != index or not out.is_contiguous()):
        raise ValueError(f"out: {rows} contiguous int32 numbers on {logits.device}")
    if index < 0:
        token, logprob = _sample_cpu(logits, uniforms, temperature, top_k, top_p, min_p, rng)
        token = token if out is None else out.copy_(token)
        return (token, logprob) if return_logprobs else token
    if _current() != index:
        with torch.cuda.device(index):
            return sample(logits, uniforms, temperature, top_k, top_p, min_p, return_logprobs, rng, out)
    if logits.stride(1) != 1 and vocab > 1:
        logits = logits.contiguous()
    token = logits.new_empty((rows,), dtype=torch.int32) if out is None else out
    logprob = logits.new_empty((rows,), dtype=f32) if return_logprobs else None
    rc = _lib.lib().zb_sample(_CALL(
        logits.data_ptr(), token.data_ptr(), 0 if logprob is None else logprob.data_ptr(), 0 if uniforms is None else uniforms.data_ptr(),
        0 if rng is None else rng.data_ptr(), *at, _stream(index), logits.stride(0), 0.0 if at[0] else temperature, 0.0 if at[1] else top_p,
        0.0 if at[2] else min_p, 0 if at[3] else max(0, min(int(top_k), vocab)), rows, vocab, logits.dtype is torch.bfloat16,
        uniforms is not None and uniforms.dtype is torch.float64))
    if rc:
        _lib.check(rc, "zb_sample")
    return (token, logprob) if return_logprobs else token


def uniform(seed: int, draws: int, row: int) -> float:
    """The number in [0, 1) that `rng` stands for in a row."""
    m = 2 ** 64 - 1
    z = (seed + 0x9E3779B97F4A7C15 * ((draws * 0x100000000 + row + 1) & m)) & m
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & m
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & m
    return ((z ^ (z >> 31)) >> 11) * 2.0 ** -53


def _sample_cpu(logits, uniforms, temperature, top_k, top_p, min_p, rng):
    """The restatement, by sorting, in 64 bits."""
    rows, vocab = logits.shape

    def column(value):
        return value.double()[:, None] if isinstance(value, torch.Tensor) else torch.full((rows, 1), float(value), dtype=torch.float64)

    if uniforms is None:
        uniforms = torch.tensor([uniform(int(rng[0]) % 2 ** 64, int(rng[1]) % 2 ** 64, r) for r in range(rows)], dtype=torch.float64)
    u, t, k, p, m = uniforms.double()[:, None].nan_to_num(0.0).clamp(0.0, 1.0), column(temperature), column(top_k), column(top_p), column(min_p)
    greedy = ~(t > 0) | (p <= 0)
    k = torch.where(greedy, 1.0, k)
    x, index = torch.sort(logits.double().nan_to_num(nan=-torch.inf, posinf=torch.inf, neginf=-torch.inf), dim=-1, descending=True, stable=True)
    top = x[:, :1]
    z = torch.where(x == top, 0.0, (x - top) / torch.where(t > 0, t, 1.0))
    w = torch.exp(z.nan_to_num(nan=-torch.inf, neginf=-torch.inf))
    place = torch.arange(vocab)
    w = torch.where((place < k) | ~(k > 0), w, 0.0)
    upto = w.cumsum(-1)
    keep = ((upto - w < p * upto[:, -1:]) | ~(p < 1) | (place == 0)) & ((w >= m.clamp(max=1.0)) | ~(m > 0))
    w = torch.zeros_like(w).scatter_(1, index, torch.where(keep, w, 0.0))
    upto = w.cumsum(-1)
    total = upto[:, -1:]
    last = vocab - 1 - (w > 0).flip(-1).int().argmax(-1, keepdim=True)
    token = torch.minimum((upto <= u * total).sum(-1, keepdim=True), last)
    nothing = top == -torch.inf
    logprob = torch.where(nothing, torch.nan, torch.log(w.gather(1, token) / total))
    return torch.where(nothing, 0, token)[:, 0].int(), logprob[:, 0].float()
