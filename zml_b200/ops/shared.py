"""Attention of single tokens in a batch whose sequences share their first keys: the answers to one prompt, users behind one long instruction.

`SharedPrefix` says which sequences have the same pages in front; `ops.paged_decode(..., shared=...)` then reads these once for all of them.  The
result is that of `ops.paged_decode` without it, up to rounding.  (The reference's paged kernels know no shared pages:
zml/attention/paged_attention.zig:19-293 gives every sequence its own.)
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from typing import Optional, Sequence

import torch

from . import _lib

_lib.register_signature("zb_shared_decode", C.c_int, [C.c_void_p])
_lib.register_signature("zb_shared_decode_workspace", C.c_longlong, [C.c_int] * 7)
_CALL = struct.Struct("11P q 9i f").pack                                  # ZbSharedDecode (csrc/attention_shared.cu)

HEAD_DIMS = (64, 128, 256)
MAX_BATCH = 1024
MAX_GROUP = 128                                                           # query heads of a key head


class SharedPrefix:
    """Groups of sequences with the same pages in front, as int32 tensors on the cache's device, which may change between the calls (and the
    replays of a captured one):

    `rows` [n]: the members' places in the batch, group after group, each once (of two places the last one counts); a sequence that is in no group is
    not listed.
    `starts` [groups + 1]: group g has rows[starts[g]] .. rows[starts[g + 1] - 1]; groups may be empty.
    `lens` [groups]: keys that the members of a group share, any number.  The block table's pages that hold them are the same for all members, or
    hold the same (a page that the shared keys fill in part is each member's own), as far as a member's own length goes.  As many are read together as
    the shortest member has; one whose length is zero (a sequence that has ended) takes no part.
    """
    __slots__ = ("rows", "starts", "lens")

    def __init__(self, rows: torch.Tensor, starts: torch.Tensor, lens: torch.Tensor):
        for name, t in (("rows", rows), ("starts", starts), ("lens", lens)):
            if t.dtype is not torch.int32 or t.dim() != 1 or not t.is_contiguous():
                raise ValueError(f"{name}: a contiguous int32 vector, got {t.dtype} {tuple(t.shape)}")
        if starts.shape[0] != lens.shape[0] + 1:
            raise ValueError(f"starts has one number more than lens, got {starts.shape[0]} and {lens.shape[0]}")
        if rows.get_device() != starts.get_device() or rows.get_device() != lens.get_device():
            raise ValueError("rows, starts and lens are on one device")
        self.rows, self.starts, self.lens = rows, starts, lens

    @staticmethod
    def of(groups: Sequence[tuple[Sequence[int], int]], device="cpu") -> "SharedPrefix":
        """From (members, keys that they share) of every group."""
        starts = [0]
        for members, _ in groups:
            starts.append(starts[-1] + len(members))
        i32 = dict(dtype=torch.int32, device=device)
        return SharedPrefix(torch.tensor([b for m, _ in groups for b in m], **i32), torch.tensor(starts, **i32), torch.tensor([n for _, n in groups], **i32))


_current = getattr(torch._C, "_cuda_getDevice", None)                     # absent in builds of torch without CUDA
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_WORK: dict = {}


def _workspace(index: int, *sizes: int) -> int:
    key = (index, *sizes)
    n = _WORK.get(key)
    if n is None:
        n = int(_lib.lib().zb_shared_decode_workspace(*sizes))
        if len(_WORK) >= 4096:
            _WORK.clear()
        _WORK[key] = n
    return n


def paged_decode(q, k_cache, v_cache, block_table, seq_lens, shared: SharedPrefix, scale: Optional[float] = None, out=None):
    """`ops.paged_decode` with `shared`: bfloat16, heads of 64, 128 or 256, up to 128 query heads for a key head, pages of 16, 32 or a multiple of 64
    tokens, up to 1024 sequences, a scale above zero, no window.  Sums are fp32; a weight is rounded to bf16 once (2^-8), as the product with
    the values takes it."""
    if type(shared) is not SharedPrefix:
        raise TypeError(f"shared: a SharedPrefix, got {type(shared).__name__}")
    bf16, index = torch.bfloat16, q.get_device()
    if q.dtype is not bf16 or k_cache.dtype is not bf16 or v_cache.dtype is not bf16:
        if index >= 0:
            raise TypeError(f"attention behind a shared prefix takes bfloat16, got {q.dtype}, {k_cache.dtype} and {v_cache.dtype}")
    shape, cache, table = q.shape, k_cache.shape, block_table.shape
    if len(shape) != 3 or len(cache) != 4 or v_cache.shape != cache:
        raise ValueError(f"queries [batch, heads, hd] with caches [pages, page, heads, hd], got {tuple(shape)}, {tuple(cache)} and {tuple(v_cache.shape)}")
    b, hq, hd = shape
    pages, page, hkv, head = cache
    if head != hd or hkv == 0 or hq == 0 or hq % hkv or hq > MAX_GROUP * hkv or hd not in HEAD_DIMS:
        raise ValueError(f"{hq} query heads of {hd} do not go with {hkv} key heads of {head}")
    if page not in (16, 32) and (page % 64 or page == 0):
        raise ValueError(f"pages of 16, 32 or a multiple of 64 tokens, got {page}")
    if pages == 0 or pages * page >= 2 ** 31 - 256:
        raise ValueError(f"a cache of {pages} pages of {page} tokens")
    if len(table) != 2 or table[0] != b or seq_lens.shape != (b,) or table[1] == 0:
        raise ValueError(f"block_table [{b}, pages] with seq_lens [{b}], got {tuple(table)} and {tuple(seq_lens.shape)}")
    rows, starts, lens = shared.rows, shared.starts, shared.lens
    listed, groups = rows.shape[0], lens.shape[0]
    if listed > b or groups > b:
        raise ValueError(f"{listed} members of {groups} groups in a batch of {b}")
    if b > MAX_BATCH:
        raise ValueError(f"up to {MAX_BATCH} sequences, got {b}")
    scale = 1.0 / math.sqrt(hd) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"a scale above zero, got {scale}")
    for name, t in (("block_table", block_table), ("seq_lens", seq_lens)):
        if t.dtype is not torch.int32 or not t.is_contiguous():
            raise ValueError(f"{name}: contiguous int32, got {t.dtype}")
    for t in (k_cache, v_cache, block_table, seq_lens, rows):
        if t.get_device() != index:
            raise ValueError(f"all tensors are on the queries' device, {q.device}")
    if not k_cache.is_contiguous() or not v_cache.is_contiguous():
        raise ValueError("caches are contiguous")
    if out is not None and (out.dtype is not q.dtype or out.shape != shape or out.get_device() != index or not out.is_contiguous()):
        raise ValueError("out: contiguous, of the queries' shape and type")
    if index < 0:
        from . import reference
        a = reference.paged_decode(q, k_cache, v_cache, block_table, seq_lens.clamp(0, table[1] * page), scale)
        return a if out is None else out.copy_(a)
    if (k_cache.data_ptr() | v_cache.data_ptr()) % 16:
        raise ValueError("caches start on 16 bytes")
    if _current() != index:
        with torch.cuda.device(index):
            return paged_decode(q, k_cache, v_cache, block_table, seq_lens, shared, scale, out)
    if b == 0:
        return torch.empty_like(q) if out is None else out
    s0, s1, s2 = q.stride()
    if s2 != 1 or s1 != hd or s0 % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)                   # rows are read in pieces of 16 bytes
        s0 = hq * hd
    target = out
    if out is None:
        out = q.new_empty(shape)
    elif out.data_ptr() % 4:
        out = q.new_empty(shape)
    work = q.new_empty((_workspace(index, b, listed, groups, hq, hkv, hd, page),), dtype=torch.uint8)
    rc = _lib.lib().zb_shared_decode(_CALL(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), rows.data_ptr(),
        starts.data_ptr(), lens.data_ptr(), work.data_ptr(), _stream(index), s0, b, listed, groups, hq, hkv, hd, page, table[1], pages, scale))
    if rc:
        _lib.check(rc, "zb_shared_decode")
    return out if target is None or target is out else target.copy_(out)
