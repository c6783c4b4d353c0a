"""Paged key / value cache in 8 bits: the form of the cache, and the ops that write it, attend to it and read it back.

A row is one token's key (or value) of one head, x of `hd` numbers.  Its scale is the smallest power of two 2^k with max |x| <= R 2^k, R = 448 for
float8_e4m3fn and 127 for int8; its codes are x / 2^k rounded to the cache's type, and it stands for codes * 2^k, which are bf16 numbers: reading
back is exact.  (A number that would round to 2^128 takes the code below, so that what is finite reads as finite.)  The scale is held as the byte
k + 127.  A row that holds an infinity or a NaN has the byte 255 and codes of zero, and reads as NaN.  A row takes hd + 1 bytes where the bf16
cache has 2 hd.

The ops of the bf16 cache take a `QuantKV` in the place of a cache tensor: `ops.rope_kvwrite`, `ops.paged_decode`, `ops.paged_prefill`;
`ops.paged_read` reads sequences back to bf16.  `QuantKVCache` is the whole cache of a model, indexed as the engine's bf16 tensor is.
(The reference's paged kernels take an fp8 cache with per-tensor scales, zml/attention/triton_attention.zig:308-315, which every call site
turns off.)
"""
from __future__ import annotations

import ctypes as C
import math
import struct
import threading
from typing import Optional

import torch

from . import _lib

# a call's arguments travel as one packed struct: ZbKv8Write, ZbKv8Read (csrc/kv8.cu), ZbKv8Decode (csrc/kv8_attention.cu).  ctypes takes 2.6 us to
# convert 22 arguments one by one, packing takes 0.6
for _name in ("zb_kv8_write", "zb_kv8_read", "zb_kv8_decode"):
    _lib.register_signature(_name, C.c_int, [C.c_void_p])
_lib.register_signature("zb_kv8_decode_plan", C.c_int, [C.c_int] * 5 + [C.c_void_p])
_WRITE = struct.Struct("12P 2q 9i 2f").pack
_READ = struct.Struct("11P 10i").pack
_DECODE = struct.Struct("11P q 10i f").pack

# names that the engine and the command line take -> type of the codes
KV_DTYPES = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
_RANGE = {torch.float8_e4m3fn: (8, 1.75), torch.int8: (6, 1.984375)}     # R = 2^e * m
HEAD_DIMS = (64, 128, 256)
MIN_EXPONENT, NAN_EXPONENT = 27, 255                                     # the smallest scale that is written is 2^-100


class QuantKV:
    """Keys or values of one layer: `codes` [pages, kv_heads, page_size, hd] (float8_e4m3fn or int8) and the scales' `exponents` uint8 [pages,
    kv_heads, page_size].  A page of one head is contiguous."""
    __slots__ = ("_codes", "_exponents", "_shape", "_index")

    def __init__(self, codes: torch.Tensor, exponents: torch.Tensor):
        if codes.dtype not in _RANGE:
            raise TypeError(f"a quantised cache holds float8_e4m3fn or int8 codes, got {codes.dtype}")
        if exponents.dtype is not torch.uint8:
            raise TypeError(f"the exponents of a quantised cache are uint8, got {exponents.dtype}")
        shape = codes.shape
        if len(shape) != 4 or exponents.shape != shape[:3]:
            raise ValueError(f"codes [pages, heads, page_size, hd] with exponents [pages, heads, page_size], got {tuple(shape)} and "
                             f"{tuple(exponents.shape)}")
        self._index = codes.get_device()
        if exponents.get_device() != self._index or not codes.is_contiguous() or not exponents.is_contiguous():
            raise ValueError("codes and exponents are contiguous and on one device")
        self._codes, self._exponents, self._shape = codes, exponents, shape

    codes = property(lambda self: self._codes)
    exponents = property(lambda self: self._exponents)

    @staticmethod
    def alloc(pages: int, kv_heads: int, page_size: int, hd: int, dtype=torch.float8_e4m3fn, device="cpu") -> "QuantKV":
        """Zeros."""
        return QuantKV(torch.zeros((pages, kv_heads, page_size, hd), dtype=dtype, device=device),
                       torch.zeros((pages, kv_heads, page_size), dtype=torch.uint8, device=device))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def page_size(self) -> int:
        return self.codes.shape[2]

    def dequantize(self, dtype=torch.float32) -> torch.Tensor:
        """What all rows stand for, in the layout of a bf16 cache: [pages, page_size, kv_heads, hd]."""
        return _values(self.codes, self.exponents).transpose(1, 2).to(dtype)


class QuantKVCache:
    """Codes [layers, 2, pages, kv_heads, page_size, hd] and exponents of a whole model; `cache[layer, 0]` are the keys of a layer, `cache[layer, 1]`
    its values, as `QuantKV`."""

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, hd: int, dtype=torch.float8_e4m3fn, device="cpu"):
        if dtype not in _RANGE:
            raise TypeError(f"a quantised cache holds float8_e4m3fn or int8 codes, got {dtype}")
        if hd not in HEAD_DIMS or page_size % 16 or page_size <= 0:
            raise ValueError(f"a quantised cache has heads of {HEAD_DIMS} and pages of a multiple of 16 tokens, got {hd} and {page_size}")
        self.codes = torch.zeros((layers, 2, pages, kv_heads, page_size, hd), dtype=dtype, device=device)
        self.exponents = torch.zeros((layers, 2, pages, kv_heads, page_size), dtype=torch.uint8, device=device)
        self._layers = [[QuantKV(self.codes[l, i], self.exponents[l, i]) for i in range(2)] for l in range(layers)]

    def __getitem__(self, at) -> QuantKV:
        layer, which = at
        return self._layers[layer][which]

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def nbytes(self) -> int:
        return self.codes.numel() + self.exponents.numel()

    def decode_plan(self, batch: int, hq: int, max_seq_len: int) -> int:
        """A number for how `paged_decode` of these sizes is launched on the GPU: a captured launch serves any lengths, but is the one that the
        `max_seq_len` of its capture asked for."""
        k = self[0, 0]
        return _plan(k._index, batch, hq, k._shape[1], k._shape[3], max_seq_len)[0]


def kv_dtype(name) -> torch.dtype:
    """The code type that "fp8", "int8" or a torch dtype names."""
    dt = KV_DTYPES.get(name, name)
    if dt not in _RANGE:
        raise ValueError(f"unknown cache type {name!r}; known: {', '.join(KV_DTYPES)}")
    return dt


def _power(exponents: torch.Tensor) -> torch.Tensor:
    """The powers of two that exponent bytes stand for, NaN for 255."""
    p = (exponents.int() << 23).view(torch.float32)
    return torch.where(exponents == NAN_EXPONENT, float("nan"), p)


def _values(codes, exponents) -> torch.Tensor:
    return codes.float() * _power(exponents)[..., None]


def quantize(x: torch.Tensor, dtype=torch.float8_e4m3fn):
    """Rows x [..., hd] -> (codes, exponents [...]); the restatement of what the writing kernel does."""
    e, m = _RANGE[dtype]
    xf = x.float()
    a = xf.abs().amax(-1)
    ok = torch.isfinite(a)
    frac, exp = torch.frexp(torch.where(ok, a, torch.ones_like(a)))          # a = frac 2^exp, frac in [0.5, 1)
    byte = (exp - 1 - e + (2 * frac > m) + 127).clamp_min(MIN_EXPONENT)
    y = torch.where(ok[..., None], xf * _power(254 - byte)[..., None], 0.0)
    y = y.round() if dtype is torch.int8 else y
    top, most = (249, 63.0) if dtype is torch.int8 else (247, 240.0)         # the largest byte, and its largest code below 2^128
    y = torch.where((byte == top)[..., None], y.clamp(-most, most), y)
    return y.to(dtype), torch.where(ok, byte, NAN_EXPONENT).to(torch.uint8)


# ------------------------------------------------------------------ checks
def _pair(k, v) -> tuple[int, int, int, int]:
    """The common shape of keys and values that the kernels take."""
    if type(k) is not QuantKV or type(v) is not QuantKV:
        raise TypeError("keys and values are both quantised or both not")
    kc, vc, n = k._codes, v._codes, k._shape
    if kc.dtype is not vc.dtype or n != v._shape or k._index != v._index:
        raise ValueError("keys and values of one type, shape and device")
    pages, heads, page_size, hd = n
    if hd not in HEAD_DIMS or page_size % 16 or page_size == 0 or pages == 0 or heads == 0:
        raise ValueError(f"a quantised cache has heads of {HEAD_DIMS} and pages of a multiple of 16 tokens, got {tuple(n)}")
    if (kc.data_ptr() | vc.data_ptr() | k._exponents.data_ptr() | v._exponents.data_ptr()) % 16:
        raise ValueError("codes and exponents start on 16 bytes")
    if pages * heads * page_size >= 2 ** 31:
        raise ValueError("a quantised cache of a layer has fewer than 2^31 rows")
    return n


def _ints(index: int, name: str, t) -> None:
    if t.dtype is not torch.int32 or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous int32 on the cache's device, got {t.dtype} on {t.device}")


def _table(k: QuantKV, block_table, seq_lens) -> tuple[int, int]:
    index = k._index
    if (block_table.dtype is not torch.int32 or seq_lens.dtype is not torch.int32 or block_table.get_device() != index or seq_lens.get_device() != index
            or not block_table.is_contiguous() or not seq_lens.is_contiguous()):
        _ints(index, "block_table", block_table)
        _ints(index, "seq_lens", seq_lens)
    shape = block_table.shape
    if len(shape) != 2 or seq_lens.shape != shape[:1]:
        raise ValueError(f"block_table [batch, pages] with seq_lens [batch], got {tuple(shape)} and {tuple(seq_lens.shape)}")
    return shape


def _queries(q, k: QuantKV, out) -> tuple[int, int, int]:
    shape = q.shape
    if q.dtype is not torch.bfloat16 or q.get_device() != k._index or len(shape) != 3:
        raise TypeError(f"queries [rows, heads, hd] in bfloat16 on {k.device}, got {q.dtype} {tuple(shape)} on {q.device}")
    if shape[2] != k._shape[3] or shape[1] % k._shape[1] or shape[1] == 0:
        raise ValueError(f"{shape[1]} query heads of {shape[2]} do not go with {k._shape[1]} key heads of {k._shape[3]}")
    if out is not None and (out.dtype is not torch.bfloat16 or out.shape != shape or out.get_device() != k._index or not out.is_contiguous()):
        raise ValueError("out: contiguous bfloat16 of the queries' shape")
    return shape


_current = getattr(torch._C, "_cuda_getDevice", None)                     # absent in builds of torch without CUDA
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", None)


# ------------------------------------------------------------------ writer
def rope_kvwrite(qkv, positions, slot_mapping, inv_freq, k: QuantKV, v: QuantKV, hq: int, hkv: int, hd: int, layout: int = 0,
                 rot_dim: Optional[int] = None, attn_factor: float = 1.0, q_norm_w=None, k_norm_w=None, norm_eps: float = 1e-6,
                 norm_unit_offset: bool = False, q_out=None):
    """`ops.rope_kvwrite` on a quantised cache.  From the projection to the one rounding at the end all is 32 bits, and angles are formed in 64.
    The slots of one call differ from one another."""
    pages, heads, page_size, head = _pair(k, v)
    t, columns = qkv.shape
    rot, index = hd if rot_dim is None else rot_dim, k._index
    if qkv.dtype is not torch.bfloat16 or qkv.get_device() != index or qkv.stride()[1] != 1:
        raise TypeError(f"qkv [tokens, (hq + 2 hkv) hd] in bfloat16 on {k.device}, got {qkv.dtype} {tuple(qkv.shape)} on {qkv.device}")
    if heads != hkv or head != hd or hq <= 0 or columns != (hq + 2 * hkv) * hd:
        raise ValueError(f"a projection of {columns} columns and a cache of {heads} heads of {head} for {hq} + 2 x {hkv} heads of {hd}")
    if rot % 2 or not 0 <= rot <= hd or layout not in (0, 1, 2):
        raise ValueError(f"rotation of {rot} of {hd} columns in layout {layout}")
    _ints(index, "positions", positions)
    _ints(index, "slot_mapping", slot_mapping)
    if positions.shape != (t,) or slot_mapping.shape != (t,):
        raise ValueError(f"{t} tokens with positions {tuple(positions.shape)} and slots {tuple(slot_mapping.shape)}")
    if inv_freq.dtype is not torch.float32 or inv_freq.get_device() != index or inv_freq.numel() < rot // 2 or not inv_freq.is_contiguous():
        raise ValueError(f"inv_freq: {rot // 2} contiguous float32 numbers on {k.device}")
    for w in (q_norm_w, k_norm_w):
        if w is not None and (w.dtype is not torch.bfloat16 or w.shape != (hd,) or w.get_device() != index or not w.is_contiguous()):
            raise ValueError(f"norm weights: {hd} contiguous bfloat16 numbers on {k.device}")
    if q_out is not None and (q_out.dtype is not torch.bfloat16 or q_out.shape != (t, hq, hd) or q_out.get_device() != index or not q_out.is_contiguous()):
        raise ValueError(f"q_out: contiguous bfloat16 [{t}, {hq}, {hd}] on {k.device}")
    if index < 0:
        q = _rope_kvwrite_cpu(qkv, positions, slot_mapping, inv_freq, k, v, hq, hkv, hd, layout, rot, attn_factor, q_norm_w, k_norm_w, norm_eps,
                              norm_unit_offset)
        return q if q_out is None else q_out.copy_(q)
    if _current() != index:
        with torch.cuda.device(index):
            return rope_kvwrite(qkv, positions, slot_mapping, inv_freq, k, v, hq, hkv, hd, layout, rot, attn_factor, q_norm_w, k_norm_w, norm_eps,
                                norm_unit_offset, q_out)
    if q_out is None:
        q_out = qkv.new_empty((t, hq, hd))
    kc = k._codes
    rc = _lib.lib().zb_kv8_write(_WRITE(
        qkv.data_ptr(), q_out.data_ptr(), kc.data_ptr(), k._exponents.data_ptr(), v._codes.data_ptr(), v._exponents.data_ptr(), positions.data_ptr(),
        slot_mapping.data_ptr(), inv_freq.data_ptr(), 0 if q_norm_w is None else q_norm_w.data_ptr(), 0 if k_norm_w is None else k_norm_w.data_ptr(),
        _stream(index), qkv.stride()[0], pages * page_size, t, hq, hkv, hd, rot, layout, page_size, bool(norm_unit_offset),
        kc.dtype is torch.int8, attn_factor, norm_eps))
    if rc:
        _lib.check(rc, "zb_kv8_write")
    return q_out


def _rope_kvwrite_cpu(qkv, positions, slot_mapping, inv_freq, k, v, hq, hkv, hd, layout, rot, attn_factor, q_norm_w, k_norm_w, norm_eps, norm_unit_offset):
    t, half = qkv.shape[0], rot // 2
    x = qkv.float().reshape(t, hq + 2 * hkv, hd)
    angle = positions.double()[:, None] * inv_freq.double()[None, :half]
    cos, sin = (angle.cos().float() * attn_factor)[:, None], (angle.sin().float() * attn_factor)[:, None]
    i = torch.arange(half)
    i, j = {0: (i, i + half), 1: (2 * i, 2 * i + 1), 2: (i, i + hd // 2)}[layout]

    def turned(y, w):
        if w is not None:
            y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + norm_eps) * (w.float() + (1.0 if norm_unit_offset else 0.0))
        out = y.clone()
        out[..., i] = y[..., i] * cos - y[..., j] * sin
        out[..., j] = y[..., j] * cos + y[..., i] * sin
        return out

    slots = slot_mapping.long()
    n = k.codes.shape[0] * k.page_size
    if bool((slots >= n).any()):
        raise IndexError(f"slot {int(slots.max())} of a cache of {n}")
    at = slots >= 0
    page, row = slots[at] // k.page_size, slots[at] % k.page_size
    for cache, y in ((k, turned(x[:, hq:hq + hkv], k_norm_w)), (v, x[:, hq + hkv:])):
        codes, exponents = quantize(y[at], cache.codes.dtype)
        cache.codes.view(torch.uint8)[page, :, row] = codes.view(torch.uint8)
        cache.exponents[page, :, row] = exponents
    return turned(x[:, :hq], q_norm_w).to(qkv.dtype)


# ------------------------------------------------------------------ reader
def paged_read(k: QuantKV, v: QuantKV, block_table, seq_lens, num_pages: Optional[int] = None):
    """Reads whole sequences back: (keys, values, table) with keys and values bfloat16 [num_pages, page_size, kv_heads, hd], the pages of sequence
    after sequence, and the block table int32 [batch, pages] that finds them there (zeros behind a sequence's pages).  Rows behind a sequence's
    end in its last page are zero.  `num_pages`: pages that the sequences hold together, where the caller knows it (else room for as many as
    the block table has; those behind the last sequence are not written).  Fewer than they hold are read as far as they go, and reported (`raise_on_status`)."""
    pages, heads, page_size, hd = _pair(k, v)
    b, width = _table(k, block_table, seq_lens)
    index = k._index
    n = b * width if num_pages is None else int(num_pages)
    if n < 0:
        raise ValueError(f"{n} pages")
    if index < 0:
        return _paged_read_cpu(k, v, block_table, seq_lens, n)
    if _current() != index:
        with torch.cuda.device(index):
            return _read(k, v, block_table, seq_lens, page_size, width, n)
    return _read(k, v, block_table, seq_lens, page_size, width, n)


def _read(k, v, block_table, seq_lens, size, width, n, lens=None):
    """`paged_read` into n pages of `size` tokens, `width` of a sequence at most, on the current device.  `lens` takes the lengths that were read:
    no more than the block table has, none below zero, and zero for a sequence that the n pages do not hold whole."""
    pages, heads, page_size, hd = k._shape
    kc = k._codes
    kd = block_table.new_empty((n, size, heads, hd), dtype=torch.bfloat16)
    vd = torch.empty_like(kd)
    table = block_table.new_empty((block_table.shape[0], width))
    rc = _lib.lib().zb_kv8_read(_READ(
        kc.data_ptr(), k._exponents.data_ptr(), v._codes.data_ptr(), v._exponents.data_ptr(), kd.data_ptr(), vd.data_ptr(), block_table.data_ptr(),
        seq_lens.data_ptr(), table.data_ptr(), 0 if lens is None else lens.data_ptr(), _stream(k._index), block_table.shape[0], heads, hd, page_size,
        block_table.shape[1], pages, size, width, n, kc.dtype is torch.int8))
    if rc:
        _lib.check(rc, "zb_kv8_read")
    return kd, vd, table


def _paged_read_cpu(k, v, block_table, seq_lens, n):
    pages, heads, page_size, hd = k.codes.shape
    b, width = block_table.shape
    out = torch.zeros((2, n, page_size, heads, hd), dtype=torch.bfloat16)
    table = torch.zeros((b, width), dtype=torch.int32)
    lens = seq_lens.clamp(0, width * page_size).tolist()
    if sum(-(-x // page_size) for x in lens) > n:
        raise ValueError(f"the sequences hold more than {n} pages")
    at = 0
    for i, length in enumerate(lens):
        m = -(-length // page_size)
        source = block_table[i, :m].long()
        for to, cache in zip(out, (k, v)):
            x = _values(cache.codes.view(torch.uint8)[source].view(cache.codes.dtype), cache.exponents[source])
            to[at:at + m] = x.transpose(1, 2).to(torch.bfloat16)
            to[at:at + m].reshape(m * page_size, heads, hd)[length:] = 0
        table[i, :m] = torch.arange(at, at + m, dtype=torch.int32)
        at += m
    return out[0], out[1], table


# ------------------------------------------------------------------ attention
_PLANS: dict = {}


def _plan(index, b, hq, hkv, hd, max_len) -> tuple[int, int]:
    """(how a decode call is cut, numbers of its workspace): a function of its sizes."""
    key = (index, b, hq, hkv, hd, -(-max_len // 16))
    got = _PLANS.get(key)
    if got is None:
        n = C.c_longlong()
        parts = _lib.lib().zb_kv8_decode_plan(b, hq, hkv, hd, max_len, C.byref(n))
        if parts == -2 ** 31:
            raise _lib.KernelError(f"no plan for {b} sequences of up to {max_len} keys, {hq} / {hkv} heads of {hd}")
        if len(_PLANS) >= 4096:
            _PLANS.clear()
        got = _PLANS[key] = (parts, n.value)
    return got


_TICKETS: dict = {}
_CAPTURED: dict = {}                                                      # device -> [stock, how much of it captured calls have]
_STOCK = threading.Lock()                                                 # captures of several threads take pieces of one stock
CAPTURED_TICKETS = 1 << 20


def _tickets(q, index: int, stream: int, n: int):
    """At least n zeros (int32) that no other call in flight uses; the kernel leaves zeros behind.  The calls of one stream follow one another and
    share theirs.  Graphs may be replayed on any streams, so a captured call has its own for good: a piece of a stock that an earlier eager call
    has cleared, or, where there is none or it has come to an end, an allocation that every replay clears."""
    if _capturing():
        with _STOCK:
            stock = _CAPTURED.get(index)
            if stock is not None and stock[1] + n <= CAPTURED_TICKETS:
                at = stock[1]
                stock[1] = at + n
                return stock[0][at:at + n]
        return q.new_zeros((n,), dtype=torch.int32)
    if index not in _CAPTURED:
        stock = q.new_zeros((CAPTURED_TICKETS,), dtype=torch.int32)
        torch.cuda.current_stream(index).synchronize()                       # whatever stream replays
        with _STOCK:
            _CAPTURED.setdefault(index, [stock, 0])                          # another thread's may be in use already
    got = _TICKETS.get((index, stream))
    if got is None or got.numel() < n:
        if len(_TICKETS) >= 256:
            _TICKETS.clear()
        got = _TICKETS[(index, stream)] = q.new_zeros((max(n, 4096),), dtype=torch.int32)
    return got


def paged_decode(q, k: QuantKV, v: QuantKV, block_table, seq_lens, scale: Optional[float] = None, window: int = 0,
                 max_seq_len: Optional[int] = None, out=None):
    """`ops.paged_decode` on a quantised cache.  The keys are split over the GPU on the device, from the lengths there (`max_seq_len` bounds
    the launch only); any number of query heads for a key head.  Sums are fp32; weights times values' scales are f16, 2^-11 each and 2^-32 of a head's largest;
    beside int8 keys a query's numbers are rounded to 2^-15 of its largest."""
    pages, hkv, page_size, _ = _pair(k, v)
    sequences, width = _table(k, block_table, seq_lens)
    b, hq, hd = _queries(q, k, out)
    index = k._index
    if sequences != b:
        raise ValueError(f"{b} queries for {sequences} sequences")
    if index < 0:
        from . import reference
        a = reference.paged_decode(q.float(), k.dequantize(), v.dequantize(), block_table, seq_lens.clamp(0, width * page_size), scale, window).to(q.dtype)
        return a if out is None else out.copy_(a)
    if _current() != index:
        with torch.cuda.device(index):
            return paged_decode(q, k, v, block_table, seq_lens, scale, window, max_seq_len, out)
    s0, s1, s2 = q.stride()
    if s2 != 1 or s1 != hd or s0 % 4 or q.data_ptr() % 8:
        q = q.clone(memory_format=torch.contiguous_format)                   # the kernel reads 8 bytes of a row at a time
        s0 = hq * hd
    if out is None:
        out = torch.empty_like(q) if s0 == hq * hd else q.new_empty((b, hq, hd))      # 1.4 us where new_empty takes 2.0
    elif out.data_ptr() % 8:                                                 # and writes as many
        return out.copy_(paged_decode(q, k, v, block_table, seq_lens, scale, window, max_seq_len))
    most = width * page_size
    parts, numbers = _plan(index, b, hq, hkv, hd, most if max_seq_len is None else min(max_seq_len, most))
    stream = _stream(index)
    work = tickets = 0
    if numbers:                                                               # chunks leave sums, and draw tickets
        partial = q.new_empty((numbers,), dtype=torch.float32)
        ticket = _tickets(q, index, stream, b * hkv * -(-hq // (8 * hkv)))
        work, tickets = partial.data_ptr(), ticket.data_ptr()
    kc = k._codes
    rc = _lib.lib().zb_kv8_decode(_DECODE(
        q.data_ptr(), kc.data_ptr(), k._exponents.data_ptr(), v._codes.data_ptr(), v._exponents.data_ptr(), out.data_ptr(), block_table.data_ptr(),
        seq_lens.data_ptr(), work, tickets, stream, s0, b, hq, hkv, hd, page_size, width, pages, window, kc.dtype is torch.int8, parts,
        1.0 / math.sqrt(hd) if scale is None else scale))
    if rc:
        _lib.check(rc, "zb_kv8_decode")
    return out


def paged_prefill(q, k: QuantKV, v: QuantKV, block_table, seq_lens, q_start, scale: Optional[float] = None, window: int = 0, out=None,
                  total_q_blocks: Optional[int] = None, impl: str = "auto", max_seq_len: Optional[int] = None, kv_pages: Optional[int] = None):
    """`ops.paged_prefill` on a quantised cache: the sequences are read back to bf16 pages of 64 tokens, which is what the tcgen05 kernels take, and the
    bf16 kernels attend to that.  Prompts with many new tokens are bound by their products: reading back moves 6 bytes a key, head and column once,
    where every query of the group makes 4 operations of them.  Few new tokens on a long past read the whole past back, too.  The workspace
    lives as long as the call; it holds what the block table could name, or, less, `kv_pages` pages of the cache: what the sequences hold
    together, where the caller knows it.  Sequences that do not fit into that are reported (`raise_on_status`), and their outputs are zero.  `max_seq_len` chooses the kernel only."""
    page_size = _pair(k, v)[2]
    b, width = _table(k, block_table, seq_lens)
    _queries(q, k, out)
    _ints(k._index, "q_start", q_start)
    if q_start.shape != (b + 1,):
        raise ValueError(f"q_start has one number more than the {b} sequences, got {tuple(q_start.shape)}")
    if q.shape[0] == 0:
        return q.new_empty(q.shape) if out is None else out
    from . import paged_prefill as bf16_prefill
    if k._index < 0:
        kd, vd, table = paged_read(k, v, block_table, seq_lens, kv_pages)
        lens = seq_lens.clamp(0, width * page_size)
    else:
        if _current() != k._index:
            with torch.cuda.device(k._index):
                return paged_prefill(q, k, v, block_table, seq_lens, q_start, scale, window, out, total_q_blocks, impl, max_seq_len, kv_pages)
        n = b * -(-width * page_size // 64)
        if kv_pages is not None:                                             # at most 63 tokens behind each sequence
            n = min(n, kv_pages * page_size // 64 + b)
        lens = torch.empty_like(seq_lens)
        columns = max(1, -(-width * page_size // 64))                        # the bf16 kernels read the first one, whatever the lengths are
        kd, vd, table = _read(k, v, block_table, seq_lens, 64, columns, max(1, n), lens)
    a = bf16_prefill(q, kd, vd, table, lens, q_start, scale, window, out=out, total_q_blocks=total_q_blocks, impl=impl, max_seq_len=max_seq_len)
    return a if out is None or a is out else out.copy_(a)
