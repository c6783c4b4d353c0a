"""The paged key / value cache in 8 bits (ops.kv8): its form, the writer, the reader, attention of single tokens and of prompts.

Oracles are restatements in 64 bits.  Where tolerances come from is written beside them; a rounding to a format is off by at most half a step:
2^-8 relative in bf16, 2^-11 in f16, 2^-4 in e4m3 (2^-10 in units of the scale among its subnormals), half a unit in int8.
"""
import math

import pytest
import torch

from zml_b200 import ops
from zml_b200.ops import kv8

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
gpu = pytest.mark.gpu
DTYPES = pytest.mark.parametrize("dtype", [E4M3, INT8], ids=["e4m3", "int8"])


# ------------------------------------------------------------------ oracles
def values64(cache):
    """[pages, heads, page, hd] in 64 bits; NaN where the exponent says so."""
    p = torch.exp2(cache.exponents.double() - 127.0)
    p = torch.where(cache.exponents == 255, math.nan, p)
    return cache.codes.cpu().double().to(p.device) * p[..., None]


def sequence64(cache, table_row, n):
    page = cache.codes.shape[2]
    pages = table_row[:-(-n // page)].long().to(cache.codes.device)
    codes = cache.codes.view(torch.uint8)[pages].view(cache.codes.dtype)
    return values64(ops.QuantKV(codes, cache.exponents[pages])).transpose(1, 2).reshape(-1, cache.codes.shape[1], cache.codes.shape[3])[:n]


def attend64(q, k, v, scale, window):
    """q [rows, hq, hd] the last rows of k, v [n, hkv, hd] -> (out, attention of |v|, largest sum of |q k| scale), in 64 bits."""
    rows, hq, hd = q.shape
    n, hkv, _ = k.shape
    out, mag = torch.zeros(rows, hq, hd, dtype=torch.float64, device=q.device), torch.zeros(rows, hq, hd, dtype=torch.float64, device=q.device)
    most = 0.0
    if n == 0:
        return out, mag, most
    q_pos, k_pos = torch.arange(n - rows, n, device=q.device)[:, None], torch.arange(n, device=q.device)[None]
    seen = k_pos <= q_pos
    if window > 0:
        seen &= k_pos > q_pos - window
    for h in range(hq):
        kh, vh = k[:, h // (hq // hkv)], v[:, h // (hq // hkv)]
        some = seen.any(0)
        kz, vz = torch.where(some[:, None], kh, 0.0), torch.where(some[:, None], vh, 0.0)
        s = (q[:, h].double() @ kz.t()) * scale
        most = max(most, float((q[:, h].double().abs() @ kz.abs().t()).max()) * abs(scale))
        p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
        out[:, h], mag[:, h] = p @ vz, p @ vz.abs()
    return out, mag, most


def rot64(x, pos, freq, rot, layout, factor):
    hd, half = x.shape[-1], rot // 2
    a = pos.double()[:, None, None] * freq.double()[:half]
    i = torch.arange(half, device=x.device)
    i, j = {0: (i, i + half), 1: (2 * i, 2 * i + 1), 2: (i, i + hd // 2)}[layout]
    y = x.clone()
    y[..., i] = (x[..., i] * a.cos() - x[..., j] * a.sin()) * factor
    y[..., j] = (x[..., j] * a.cos() + x[..., i] * a.sin()) * factor
    return y


def check_rows(cache, page, row, x, rel):
    """The cache's rows at (page[t], row[t]) stand for x [tokens, heads, hd] (64 bits), which the kernel knows up to rel of a row's largest number."""
    dtype = cache.codes.dtype
    codes = cache.codes.view(torch.uint8)[page, :, row].view(dtype)
    exps = cache.exponents[page, :, row]
    s = torch.exp2(exps.double() - 127.0)
    a = x.abs().amax(-1)
    r = 448.0 if dtype is E4M3 else 127.0
    live = a > 2.0 ** -90
    # the smallest power of two with a <= r s
    assert bool((a <= r * s * (1 + rel))[live].all()) and bool((a > r * s / 2 * (1 - rel))[live].all())
    err = (codes.cpu().double().to(x.device) * s[..., None] - x).abs()
    half = torch.maximum(x.abs() * 2.0 ** -4, s[..., None] * 2.0 ** -10) if dtype is E4M3 else s[..., None] * 0.5
    assert bool((err <= half + 2 * rel * a[..., None] + 2.0 ** -100).all()), float((err - half).max())


# ------------------------------------------------------------------ the form
@DTYPES
def test_quantize_is_the_definition(dtype):
    g = torch.Generator().manual_seed(1)
    r = 448.0 if dtype is E4M3 else 127.0
    x = torch.randn(200, 64, generator=g) * torch.exp(3 * torch.randn(200, 1, generator=g))
    x[0] = 0.0
    x[1, :] = 1e-20
    x[2, 0], x[3, 0] = 448.0 * 2.0 ** 9, 127.0 * 2.0 ** -9
    x[2, 1:], x[3, 1:] = 1.0, 2.0 ** -12
    x[4, 0] = 3e38
    codes, exps = kv8.quantize(x, dtype)
    s = torch.exp2(exps.double() - 127.0)
    a = x.double().abs().amax(-1)
    want = torch.exp2(torch.ceil(torch.log2(a / r)))
    assert torch.equal(s[1:], want[1:])
    y = x.double() / s[:, None]
    if dtype is INT8:
        assert torch.equal(codes.double(), y.round())
    else:
        grid = torch.arange(127, dtype=torch.uint8).view(E4M3).double()           # ascending, even codes at even places
        at = torch.bucketize(y.abs(), (grid[1:] + grid[:-1]) / 2)                  # ties down
        tie = torch.isclose(y.abs(), ((grid[1:] + grid[:-1]) / 2)[at.clamp_max(125)], rtol=0, atol=0)
        at = torch.where(tie & (at % 2 == 1), at + 1, at)
        assert torch.equal(codes.double().abs(), grid[at])
    assert not codes[0].float().any()


@DTYPES
def test_rows_that_are_not_finite_read_as_nan(dtype):
    x = torch.ones(3, 64)
    x[0, 5], x[1, 7] = math.inf, math.nan
    codes, exps = kv8.quantize(x, dtype)
    assert exps.tolist() == [255, 255, exps[2].item()] and exps[2] < 255
    assert not codes[:2].float().any()
    kv = ops.QuantKV(codes.view(1, 1, 3, 64).repeat(1, 1, 6, 1)[:, :, :16].contiguous(), exps.view(1, 1, 3).repeat(1, 1, 6)[:, :, :16].contiguous())
    d = kv.dequantize()
    assert bool(d[0, 0].isnan().all()) and bool(d[0, 1].isnan().all()) and bool((d[0, 2] == 1).all())


def test_the_whole_cache_and_its_names():
    c = ops.QuantKVCache(3, 5, 32, 2, 64, torch.int8)
    assert c.nbytes() == 3 * 2 * 5 * 2 * 32 * 65 and c[2, 1].codes.shape == (5, 2, 32, 64)
    c[1, 0].codes.fill_(7)
    assert int(c.codes[1, 0].min()) == 7 and int(c.codes[1, 1].max()) == 0
    assert kv8.kv_dtype("fp8") is E4M3 and kv8.kv_dtype(torch.int8) is INT8
    for bad in ("bf16", torch.float16, None):
        with pytest.raises(ValueError):
            kv8.kv_dtype(bad)
    for args in ((1, 2, 24, 2, 64), (1, 2, 64, 2, 96), (1, 2, 0, 2, 64)):
        with pytest.raises(ValueError):
            ops.QuantKVCache(*args)
    with pytest.raises(TypeError):
        ops.QuantKVCache(1, 2, 64, 2, 64, torch.float16)


def make_cache(pages, hkv, page, hd, dtype, seed=0, device="cpu", spread=2.0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for i in range(2):
        x = torch.randn(pages, hkv, page, hd, generator=g) * spread * torch.exp(0.5 * torch.randn(pages, hkv, page, 1, generator=g))
        out.append(ops.QuantKV(*(t.to(device) for t in kv8.quantize(x, dtype))))
    return out


def test_refusals():
    k, v = make_cache(4, 2, 16, 64, E4M3)
    i8, _ = make_cache(4, 2, 16, 64, INT8)
    bt, sl = torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    qs = torch.arange(4, dtype=torch.int32)
    for codes, exps, err in ((k.codes.float(), k.exponents, TypeError), (k.codes, k.exponents.float(), TypeError), (k.codes, k.exponents[:3], ValueError),
                             (k.codes[0], k.exponents, ValueError), (k.codes.transpose(1, 2), k.exponents.transpose(1, 2), ValueError)):
        with pytest.raises(err):
            ops.QuantKV(codes, exps)
    for a, b, err in ((k, v.dequantize(torch.bfloat16), TypeError), (k.dequantize(torch.bfloat16), v, TypeError), (k, i8, ValueError)):
        with pytest.raises(err):
            ops.paged_decode(q, a, b, bt, sl)
        with pytest.raises(err):
            ops.paged_prefill(q, a, b, bt, sl, qs)
        with pytest.raises(err):
            ops.paged_read(a, b, bt, sl)
    for args, err in (((q.float(), k, v, bt, sl), TypeError), ((q[:, :, :32], k, v, bt, sl), ValueError), ((q[:, :3], k, v, bt, sl), ValueError),
                      ((q, k, v, bt.long(), sl), ValueError), ((q, k, v, bt, sl.long()), ValueError), ((q[:2], k, v, bt, sl), ValueError),
                      ((q, k, v, bt[:2], sl), ValueError), ((q, k, v, bt[0], sl), ValueError)):
        with pytest.raises(err):
            ops.paged_decode(*args)
    with pytest.raises(ValueError):
        ops.paged_decode(q, k, v, bt, sl, out=torch.zeros(3, 4, 32, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        ops.paged_decode(q, k, v, bt, sl, ext=object())
    with pytest.raises(ValueError):
        ops.paged_prefill(q, k, v, bt, sl, qs, ext=object())
    with pytest.raises(ValueError):
        ops.paged_prefill(q, k, v, bt, sl, qs.long())
    with pytest.raises(ValueError):
        ops.paged_read(k, v, bt, sl, num_pages=2)              # three sequences of a page each
    with pytest.raises(ValueError):
        ops.paged_read(k, v, bt, sl, num_pages=-1)
    for hd, page in ((96, 16), (64, 24)):
        a, b = make_cache(4, 2, page, hd, E4M3)
        with pytest.raises(ValueError):
            ops.paged_decode(torch.zeros(3, 4, hd, dtype=torch.bfloat16), a, b, bt, sl)
    qkv, pos = torch.zeros(3, 8 * 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    slots, freq = torch.tensor([0, 1, -1], dtype=torch.int32), torch.ones(32)
    good = dict(qkv=qkv, positions=pos, slot_mapping=slots, inv_freq=freq, k_cache=k, v_cache=v, hq=4, hkv=2, hd=64)
    ops.rope_kvwrite(**good)
    w = torch.ones(64, dtype=torch.bfloat16)
    for change, err in ((dict(qkv=qkv.float()), TypeError), (dict(qkv=qkv[:, :-64]), ValueError), (dict(hq=5), ValueError), (dict(hkv=1), ValueError),
                        (dict(positions=pos.long()), ValueError), (dict(positions=pos[:2]), ValueError), (dict(slot_mapping=slots[:2]), ValueError),
                        (dict(slot_mapping=slots.long()), ValueError), (dict(inv_freq=freq.double()), ValueError), (dict(inv_freq=freq[:31]), ValueError),
                        (dict(rot_dim=63), ValueError), (dict(rot_dim=66), ValueError), (dict(layout=3), ValueError), (dict(q_norm_w=w.float()), ValueError),
                        (dict(k_norm_w=w[:32]), ValueError), (dict(q_out=torch.zeros(3, 4, 64)), ValueError), (dict(k_cache=i8), ValueError),
                        (dict(v_cache=v.dequantize(torch.bfloat16)), TypeError), (dict(slot_mapping=slots + 64), IndexError)):
        with pytest.raises(err):
            ops.rope_kvwrite(**{**good, **change})


# ------------------------------------------------------------------ writer
def write_case(tokens, hq, hkv, hd, page, dtype, norm=False, rot=None, layout=0, factor=1.0, unit=False, shift=0, pos0=0, device="cpu", spread=1.0, seed=0,
               far=0):
    """Runs the writer and holds it to 64 bits: q within 2^-8 and rows within half a step, both over what fp32 gives up on the way.  That is
    relative to a row's largest number: 2^-24 for each of the norm's sum (hd / 16 in line, 5 across), its root, two products, cosine and sine at 2
    ulp, two products and a sum, together below 32 x 2^-24; the rotation grows a number by sqrt 2 at most, which the row's largest has seen."""
    rot = hd if rot is None else rot
    g = torch.Generator().manual_seed(seed)
    cols = (hq + 2 * hkv) * hd
    buf = torch.randn(tokens, cols + 8 + shift, generator=g).mul_(spread * torch.exp(0.5 * torch.randn(1, cols + 8 + shift, generator=g))).bfloat16()
    qkv = buf.to(device)[:, shift:shift + cols]
    k, v = make_cache(-(-tokens // page) + 2, hkv, page, hd, dtype, seed + 1, device)
    slots = torch.randperm(k.codes.shape[0] * page, generator=g)[:tokens].int()
    if tokens > 2:
        slots[tokens // 2] = -1
    pos = (pos0 + torch.arange(tokens) + far * torch.randint(0, 2, (tokens,), generator=g)).int()
    freq = (10000.0 ** (-torch.arange(max(1, rot // 2), dtype=torch.float64) / max(1, rot // 2))).float()
    qw, kw = ((torch.randn(hd, generator=g) * 0.1 + (0.0 if unit else 1.0)).bfloat16().to(device) for _ in range(2)) if norm else (None, None)
    before = [t.clone() for c in (k, v) for t in (c.codes.view(torch.uint8), c.exponents)]
    q = ops.rope_kvwrite(qkv, pos.to(device), slots.to(device), freq.to(device), k, v, hq, hkv, hd, layout, rot, factor, qw, kw, 1e-6, unit)
    x = qkv.double().reshape(tokens, hq + 2 * hkv, hd)
    parts = list(x.split([hq, hkv, hkv], 1))
    for i, w in ((0, qw), (1, kw)):
        if w is not None:
            parts[i] = parts[i] / (parts[i].square().mean(-1, keepdim=True) + 1e-6).sqrt() * (w.double() + (1.0 if unit else 0.0))
        parts[i] = rot64(parts[i], pos.to(device), freq.to(device), rot, layout, factor)
    rel = 32 * 2.0 ** -24
    assert q.shape == (tokens, hq, hd) and q.dtype is torch.bfloat16
    if tokens:
        err = (q.double() - parts[0]).abs()
        top = math.sqrt(2) * parts[0].abs().amax(-1, keepdim=True)
        assert bool((err <= 2.0 ** -8 * parts[0].abs() + rel * top + 2.0 ** -133).all()), float(err.max())
    live = slots >= 0
    page_at, row_at = (slots[live].long() // page).to(device), (slots[live].long() % page).to(device)
    check_rows(k, page_at, row_at, parts[1][live.to(device)], 2 * rel)
    check_rows(v, page_at, row_at, parts[2][live.to(device)], 0.0)
    # V is not computed on: its codes are the definition's, bit for bit
    codes, exps = kv8.quantize(parts[2][live.to(device)].float(), dtype)
    assert torch.equal(v.codes.view(torch.uint8)[page_at, :, row_at], codes.view(torch.uint8)) and torch.equal(v.exponents[page_at, :, row_at], exps)
    # nothing else was touched
    for t, b in zip((k.codes.view(torch.uint8), k.exponents, v.codes.view(torch.uint8), v.exponents), before):
        now, was = t.clone(), b
        now[page_at, :, row_at] = 0
        was[page_at, :, row_at] = 0
        assert torch.equal(now, was)
    return q, k, v


WRITES = [
    # tokens, hq, hkv, hd, page, more
    (1, 4, 1, 64, 16, {}),
    (0, 4, 1, 64, 16, {}),
    (5, 32, 8, 128, 64, {}),
    (70, 6, 2, 128, 32, dict(norm=True)),
    (33, 16, 4, 256, 64, dict(norm=True, rot=64, unit=True)),
    (9, 5, 5, 64, 48, dict(layout=1)),
    (9, 5, 1, 128, 16, dict(layout=1, rot=24, norm=True)),
    (9, 3, 3, 256, 16, dict(layout=1, rot=100)),
    (9, 5, 1, 64, 16, dict(layout=2, rot=32, norm=True)),
    (9, 2, 1, 128, 16, dict(layout=2)),
    (9, 5, 1, 128, 128, dict(rot=24)),
    (9, 5, 1, 256, 16, dict(rot=0, norm=True)),
    (9, 5, 3, 64, 16, dict(shift=3)),
    (9, 7, 1, 256, 16, dict(shift=1, norm=True, layout=1)),
    (9, 4, 2, 128, 64, dict(factor=1.37)),
    (40, 64, 8, 128, 64, dict(far=1000000)),
    (17, 4, 2, 128, 64, dict(spread=1e-20)),
    (17, 4, 2, 128, 64, dict(spread=1e30)),
    (3, 100, 3, 128, 64, dict(norm=True)),
]


@DTYPES
@pytest.mark.parametrize("case", WRITES, ids=str)
def test_writer_cpu(case, dtype):
    *sizes, more = case
    write_case(*sizes, dtype, **more)


@gpu
@DTYPES
@pytest.mark.parametrize("case", WRITES + [(2500, 8, 2, 128, 64, {}), (1200, 8, 2, 64, 64, dict(norm=True, layout=1))], ids=str)
def test_writer(case, dtype):
    *sizes, more = case
    write_case(*sizes, dtype, device="cuda", **more)
    ops.raise_on_status()


@gpu
@DTYPES
@pytest.mark.parametrize("shift", [0, 1])
def test_writer_rows_that_are_not_finite(dtype, shift):
    hq, hkv, hd = 2, 2, 128
    cols = (hq + 2 * hkv) * hd
    buf = torch.ones(4, cols + 8, dtype=torch.bfloat16, device="cuda")
    qkv = buf[:, shift:shift + cols]
    qkv[0, hq * hd + 3] = math.inf               # key head 0 of token 0
    qkv[1, (hq + hkv) * hd + hd + 5] = math.nan  # value head 1 of token 1
    k, v = make_cache(1, hkv, 16, hd, dtype, 3, "cuda")
    ids = torch.arange(4, dtype=torch.int32, device="cuda")
    ops.rope_kvwrite(qkv, torch.zeros_like(ids), ids, torch.ones(64, device="cuda"), k, v, hq, hkv, hd)
    kb, vb = k.exponents[0].cpu(), v.exponents[0].cpu()
    assert [kb[0, t].item() == 255 for t in range(4)] == [True, False, False, False] and not bool((kb[1, :4] == 255).any())
    assert [vb[1, t].item() == 255 for t in range(4)] == [False, True, False, False] and not bool((vb[0, :4] == 255).any())
    assert not bool(k.codes[0, 0, 0].float().any()) and not bool(v.codes[0, 1, 1].float().any())


@gpu
def test_writer_reports_a_slot_behind_the_cache():
    k, v = make_cache(2, 1, 16, 64, E4M3, 0, "cuda")
    was = k.codes.view(torch.uint8).clone()
    qkv = torch.ones(1, 3 * 64, dtype=torch.bfloat16, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    ops.rope_kvwrite(qkv, torch.zeros(1, **i32), torch.tensor([32], **i32), torch.ones(32, device="cuda"), k, v, 1, 1, 64)
    with pytest.raises(ops.KernelError):
        ops.raise_on_status()
    assert torch.equal(was, k.codes.view(torch.uint8))


# ------------------------------------------------------------------ paged batches
def paged(lens, hkv, page, hd, dtype, seed=0, device="cpu", width=None, stale=True, spread=2.0, spare=1):
    """A cache that holds sequences of `lens` tokens in shuffled pages.  Rows behind a sequence's end hold NaN (codes and exponents), and so do the
    pages of nobody; entries of the table behind a sequence's pages are no pages at all."""
    held = [-(-n // page) for n in lens]
    pages = sum(held) + spare
    k, v = make_cache(pages, hkv, page, hd, dtype, seed, device, spread)
    g = torch.Generator().manual_seed(seed + 7)
    order = torch.randperm(pages, generator=g).int()
    width = width or max(1, max(held))
    table = torch.where(torch.rand(len(lens), width, generator=g) < 0.5, -7, 1 << 30).int()
    used = torch.zeros(pages, page, dtype=torch.bool)
    at = 0
    for i, (n, m) in enumerate(zip(lens, held)):
        table[i, :m] = order[at:at + m]
        for j in range(m):
            used[order[at + j], :min(page, n - j * page)] = True
        at += m
    if stale:
        dead = (~used)[:, None].expand(pages, hkv, page).to(device)
        for c in (k, v):
            c.exponents[dead] = 255
            c.codes.view(torch.uint8)[dead] = 0x7f
    return k, v, table.to(device), torch.tensor(lens, dtype=torch.int32, device=device)


def check_attention(out, q, k, v, table, lens, starts, scale, window):
    """Against 64 bits on what the cache holds.  The result is rounded to bf16 (2^-8).  Weights p s_v are f16 (2^-11 each, and 2^-24 of the largest
    value's weight among the subnormals, half a step of 2^-24); the bf16 kernels of prompts round p to bf16 (2^-8).  Scores are fp32 sums of hd products:
    hd 2^-24 of the sum of their magnitudes, twice (numerator and denominator), and exp2 gives 2^-21."""
    hd = q.shape[2]
    weight = 2.0 ** -11 if starts is None else 2.0 ** -8
    for i, n in enumerate(lens.tolist()):
        a, b = (i, i + 1) if starts is None else (int(starts[i]), int(starts[i + 1]))
        if a == b:
            continue
        n = max(n, 0)
        ks, vs = sequence64(k, table[i], n), sequence64(v, table[i], n)
        want, mag, most = attend64(q[a:b], ks, vs, scale, window)
        seen = vs[max(0, n - (b - a) - window + 1):] if window > 0 else vs
        small = 0.0 if starts is not None or n == 0 else n * 2.0 ** -25 * float(seen.abs().max()) * 2 ** 9
        tol = 2.0 ** -8 * want.abs() + (weight + 2 * (hd + 8) * 2.0 ** -24 * most + 2.0 ** -20) * mag + small + 1e-30
        err = (out[a:b].double() - want).abs()
        assert bool(torch.isfinite(out[a:b]).all())
        assert bool((err <= tol).all()), (i, n, float((err - tol).max()), float(err.max()))


DECODES = [
    # lens, hq, hkv, hd, page, more
    ([1], 1, 1, 64, 16, {}),
    ([512], 32, 8, 64, 64, {}),
    ([0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129], 4, 2, 128, 64, {}),
    ([0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129], 8, 1, 64, 16, {}),
    ([0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129], 6, 2, 256, 32, {}),
    ([300, 7, 0, 1000], 7, 1, 128, 48, {}),
    ([300, 7, 0, 1000], 9, 1, 128, 128, {}),
    ([300, 7, 0, 1000], 32, 2, 64, 192, {}),
    ([300, 7, 0, 1000], 20, 1, 256, 64, {}),
    ([300, 7, 0, 1000], 40, 2, 128, 80, {}),
    ([300, 7, 0, 1000, 1], 5, 5, 64, 64, dict(window=1)),
    ([300, 7, 0, 1000, 64], 8, 2, 128, 64, dict(window=70)),
    ([300, 7, 0, 1000, 65], 8, 2, 256, 16, dict(window=64)),
    ([300, 9, 1000], 16, 1, 128, 64, dict(window=333)),
    ([4000, 16000], 8, 2, 128, 64, {}),
    ([0, 0, 0], 4, 2, 128, 64, {}),
    ([200, 333], 8, 2, 128, 64, dict(scale=-0.3)),
    ([200, 333], 8, 2, 128, 64, dict(scale=0.0)),
    ([200, 333], 8, 2, 64, 64, dict(q_spread=1e30, scale=1e-31)),
    ([200, 333], 8, 2, 64, 64, dict(q_spread=1e-30, scale=1e29)),
    ([200, 333], 8, 2, 64, 64, dict(spread=1e-12, scale=1e12)),
    ([100 + 13 * i for i in range(77)], 8, 2, 64, 64, {}),
]


def decode_case(lens, hq, hkv, hd, page, dtype, window=0, scale=None, q_spread=1.0, spread=2.0, device="cpu", max_seq_len=None, width=None):
    k, v, table, sl = paged(lens, hkv, page, hd, dtype, 5, device, spread=spread, width=width)
    g = torch.Generator().manual_seed(11)
    q = (torch.randn(len(lens), hq, hd, generator=g) * q_spread).bfloat16().to(device)
    out = ops.paged_decode(q, k, v, table, sl, scale, window, max_seq_len=max_seq_len)
    assert out.shape == q.shape and out.dtype is torch.bfloat16
    check_attention(out, q, k, v, table, sl, None, 1 / math.sqrt(hd) if scale is None else scale, window)
    for i, n in enumerate(lens):
        if n == 0:
            assert not bool(out[i].any())
    return out


@DTYPES
@pytest.mark.parametrize("case", [c for c in DECODES if sum(c[0]) < 3000], ids=str)
def test_decode_cpu(case, dtype):
    *sizes, more = case
    decode_case(*sizes, dtype, **more)


@gpu
@DTYPES
@pytest.mark.parametrize("case", DECODES, ids=str)
def test_decode(case, dtype):
    *sizes, more = case
    decode_case(*sizes, dtype, device="cuda", **more)
    ops.raise_on_status()


@gpu
def test_decode_any_bound_of_the_lengths():
    """`max_seq_len` decides the launch, not the result, wherever it lies."""
    lens = [1, 700, 64, 129]
    a = [decode_case(lens, 8, 2, 128, 64, E4M3, device="cuda", max_seq_len=m, width=w) for m, w in ((None, None), (700, None), (1, None), (10 ** 6, None), (None, 500))]
    for b in a[1:]:
        assert float((a[0].float() - b.float()).abs().max()) <= 2.0 ** -7 * float(a[0].float().abs().max())


@gpu
def test_decode_strided_and_unaligned_queries():
    k, v, table, sl = paged([70, 200], 2, 64, 128, E4M3, 5, "cuda")
    g = torch.Generator().manual_seed(3)
    flat = torch.randn(2, 1500, generator=g).bfloat16().cuda()
    for shift in (0, 4, 1):
        q = flat[:, shift:shift + 8 * 128].view(2, 8, 128)
        assert torch.equal(ops.paged_decode(q, k, v, table, sl), ops.paged_decode(q.contiguous(), k, v, table, sl))
    q = torch.randn(2, 128, 8, generator=g).bfloat16().cuda().transpose(1, 2)
    out = torch.full((2, 8, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    assert ops.paged_decode(q, k, v, table, sl, out=out) is out
    assert torch.equal(out, ops.paged_decode(q.contiguous(), k, v, table, sl))


@gpu
@DTYPES
def test_decode_rows_that_are_nan(dtype):
    """A key or value that is NaN makes its sequence and head NaN where it is seen, and nothing where a window hides it."""
    lens = [100, 100, 100]
    k, v, table, sl = paged(lens, 2, 64, 128, dtype, 5, "cuda")
    for cache, seq, head in ((k, 0, 1), (v, 1, 0)):
        page = int(table[seq, 0])
        cache.exponents[page, head, 10] = 255
        cache.codes.view(torch.uint8)[page, head, 10] = 0
    q = torch.randn(3, 8, 128, device="cuda").bfloat16()
    out = ops.paged_decode(q, k, v, table, sl).isnan().view(3, 2, -1)
    assert [[bool(out[i, h].all()) for h in range(2)] for i in range(3)] == [[False, True], [True, False], [False, False]]
    assert [[bool(out[i, h].any()) for h in range(2)] for i in range(3)] == [[False, True], [True, False], [False, False]]
    hidden = ops.paged_decode(q, k, v, table, sl, window=89)                    # keys 11 .. 99
    assert not bool(hidden.isnan().any())
    check_attention(hidden, q, k, v, table, sl, None, 1 / math.sqrt(128), 89)


@gpu
def test_decode_values_of_unequal_size():
    """Value rows from 2^-60 to 2^60 in one sequence, small and large ones in front."""
    for down in (False, True):
        k, v, table, sl = paged([1000], 1, 64, 64, E4M3, 5, "cuda")
        e = 67 + torch.arange(1000) // 8
        e = e.flip(0) if down else e
        for j in range(16):
            n = min(64, 1000 - 64 * j)
            v.exponents[int(table[0, j]), 0, :n] = e[64 * j:64 * j + n].to(torch.uint8).cuda()
        q = torch.randn(1, 4, 64, device="cuda").bfloat16()
        check_attention(ops.paged_decode(q, k, v, table, sl), q, k, v, table, sl, None, 0.125, 0)


@gpu
def test_decode_reports_a_page_that_is_none():
    k, v, table, sl = paged([100], 1, 64, 64, E4M3, 5, "cuda")
    q = torch.randn(1, 4, 64, device="cuda").bfloat16()
    for bad in (-1, k.codes.shape[0]):
        table[0, 1] = bad
        ops.paged_decode(q, k, v, table, sl)
        with pytest.raises(ops.KernelError):
            ops.raise_on_status()


@gpu
def test_decode_far_into_a_large_cache():
    """Offsets of codes beyond 2^31, lengths that reach beyond the table, and the reader on the same pages."""
    pages, hkv, page, hd = 36000, 8, 64, 128
    k = ops.QuantKV.alloc(pages, hkv, page, hd, INT8, "cuda")
    v = ops.QuantKV.alloc(pages, hkv, page, hd, INT8, "cuda")
    a, b = make_cache(4, hkv, page, hd, INT8, 9, "cuda")
    at = torch.tensor([pages - 1, 3, 33000, pages - 7], device="cuda")
    for big, small in ((k, a), (v, b)):
        big.codes[at], big.exponents[at] = small.codes, small.exponents
    table = at.int()[None].contiguous()
    sl = torch.tensor([10 ** 6], dtype=torch.int32, device="cuda")               # 256 are there
    q = torch.randn(1, 16, hd, device="cuda").bfloat16()
    out = ops.paged_decode(q, k, v, table, sl)
    small = torch.arange(4, dtype=torch.int32, device="cuda")[None].contiguous()
    n = torch.tensor([256], dtype=torch.int32, device="cuda")
    assert torch.equal(out, ops.paged_decode(q, a, b, small, n))
    check_attention(out, q, a, b, small, n, None, 1 / math.sqrt(hd), 0)
    kd, vd, t = ops.paged_read(k, v, table, sl)
    assert torch.equal(kd, a.dequantize(torch.bfloat16)) and torch.equal(vd, b.dequantize(torch.bfloat16)) and t.tolist() == [[0, 1, 2, 3]]


@gpu
def test_decode_in_graphs_and_streams():
    """A captured call follows lengths and tables that change on the device; two captures and two streams share nothing."""
    k, v, table, sl = paged([1500, 40, 700, 64], 4, 64, 128, E4M3, 5, "cuda", width=40)
    q = torch.randn(4, 16, 128, device="cuda").bfloat16()
    lens = [[1500, 40, 700, 64], [1, 33, 500, 0], [1400, 17, 64, 63]]
    want = []
    for n in lens:
        want.append(ops.paged_decode(q, k, v, table, torch.tensor(n, dtype=torch.int32, device="cuda")))
    graphs, outs, sls = [], [], []
    for _ in range(2):
        s = sl.clone()
        ops.paged_decode(q, k, v, table, s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.paged_decode(q, k, v, table, s))
        graphs.append(g)
        sls.append(s)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(12):
        pick = [i % 3, (i + 1) % 3]
        for s, p in zip(sls, pick):
            s.copy_(torch.tensor(lens[p], dtype=torch.int32))
        torch.cuda.synchronize()
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for o, p in zip(outs, pick):
            assert torch.equal(o, want[p])
    got = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 2]):
            got.append(ops.paged_decode(q, k, v, table, torch.tensor(lens[i % 3], dtype=torch.int32, device="cuda")))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 3])


# ------------------------------------------------------------------ reader
READS = [([1], 1, 16, 64, {}), ([0, 1, 15, 16, 17, 64, 100], 3, 16, 64, {}), ([130, 0, 64, 5], 2, 64, 128, {}), ([130, 0, 64, 5], 1, 48, 256, dict(width=9)),
         ([0, 0], 2, 64, 128, {}), ([40 + 3 * i for i in range(50)], 2, 32, 64, {})]


def read_case(lens, hkv, page, hd, dtype, width=None, device="cpu"):
    k, v, table, sl = paged(lens, hkv, page, hd, dtype, 5, device, width=width)
    held = [-(-n // page) for n in lens]
    for num in (sum(held), None):
        kd, vd, t = ops.paged_read(k, v, table, sl, num_pages=num)
        assert kd.shape[0] == (sum(held) if num is not None else table.numel())
        at = 0
        for i, (n, m) in enumerate(zip(lens, held)):
            assert t[i].tolist() == list(range(at, at + m)) + [0] * (table.shape[1] - m)
            for got, cache in ((kd, k), (vd, v)):
                rows = got[at:at + m].reshape(m * page, hkv, hd)
                assert torch.equal(rows[:n].double(), sequence64(cache, table[i], n))          # exact: they are bf16 numbers
                assert not bool(rows[n:].any())
            at += m


@DTYPES
@pytest.mark.parametrize("case", READS, ids=str)
def test_reader_cpu(case, dtype):
    *sizes, more = case
    read_case(*sizes, dtype, **more)


@gpu
@DTYPES
@pytest.mark.parametrize("case", READS + [([5000, 3, 900], 8, 64, 128, {})], ids=str)
def test_reader(case, dtype):
    *sizes, more = case
    read_case(*sizes, dtype, device="cuda", **more)
    ops.raise_on_status()


@gpu
def test_reader_leaves_what_does_not_fit():
    k, v, table, sl = paged([100, 100], 1, 64, 64, E4M3, 5, "cuda")
    kd, _, t = ops.paged_read(k, v, table, sl, num_pages=3)
    with pytest.raises(ops.KernelError):
        ops.raise_on_status()
    assert t.tolist() == [[0, 1], [2, 0]]
    assert torch.equal(kd[2].double().transpose(0, 1), values64(ops.QuantKV(k.codes[int(table[1, 0])][None], k.exponents[int(table[1, 0])][None]))[0])


@gpu
@DTYPES
def test_every_code_reads_as_what_it_is(dtype):
    codes = torch.arange(256, dtype=torch.uint8).view(1, 1, 4, 64).repeat(1, 1, 4, 1).contiguous()
    exps = torch.tensor([27, 119, 127, 200], dtype=torch.uint8).view(1, 1, 4).repeat_interleave(4, 2).contiguous()
    kv = ops.QuantKV(codes.view(dtype).cuda(), exps.cuda())
    kd, _, _ = ops.paged_read(kv, kv, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([16], dtype=torch.int32, device="cuda"))
    want = values64(kv)[0, 0].cpu()
    assert torch.equal(kd[0, :, 0].double().cpu().nan_to_num(-1.0), want.nan_to_num(-1.0))


# ------------------------------------------------------------------ prompts
PREFILLS = [
    # (new, past) of every sequence, hq, hkv, hd, page, window
    ([(1, 0)], 4, 2, 64, 16, 0),
    ([(5, 0), (64, 0), (1, 30), (70, 63)], 4, 2, 64, 64, 0),
    ([(100, 40), (3, 500)], 8, 2, 128, 64, 0),
    ([(100, 40), (3, 500)], 8, 2, 256, 64, 0),
    ([(100, 40), (3, 500)], 6, 2, 128, 32, 50),
    ([(300, 0)], 5, 1, 64, 48, 17),
]


def prefill_case(parts, hq, hkv, hd, page, window, dtype, device="cpu", **more):
    lens = [a + b for a, b in parts]
    k, v, table, sl = paged(lens, hkv, page, hd, dtype, 5, device)
    starts = [0]
    for n, _ in parts:
        starts.append(starts[-1] + n)
    g = torch.Generator().manual_seed(2)
    q = torch.randn(starts[-1], hq, hd, generator=g).bfloat16().to(device)
    out = ops.paged_prefill(q, k, v, table, sl, torch.tensor(starts, dtype=torch.int32, device=device), window=window, **more)
    check_attention(out, q, k, v, table, sl, starts, 1 / math.sqrt(hd), window)


@DTYPES
@pytest.mark.parametrize("case", PREFILLS, ids=str)
def test_prefill_cpu(case, dtype):
    prefill_case(*case, dtype)


@gpu
@DTYPES
@pytest.mark.parametrize("case", PREFILLS, ids=str)
def test_prefill(case, dtype):
    lens = [a + b for a, b in case[0]]
    prefill_case(*case, dtype, device="cuda")
    prefill_case(*case, dtype, device="cuda", max_seq_len=max(lens), kv_pages=sum(-(-n // case[4]) for n in lens))
    ops.raise_on_status()


# ------------------------------------------------------------------ how a decode call is shared out
def shared_out(lens, hq, hkv, hd, bound=None):
    """"cluster", "warp" or "chunks" (zb_kv8_decode_plan): a cluster or a CTA for each pair of a sequence and a key head, a warp, or chunks."""
    parts, _ = kv8._plan(0, len(lens), hq, hkv, hd, max(lens) if bound is None else bound)
    return "chunks" if parts > 0 else "warp" if parts == 0 else "cluster"


MANY = [(i * 37) % 90 for i in range(310)]                       # 0 .. 89 keys
UNEVEN = [3000 if i % 9 == 0 else 5 * i for i in range(100)]
SHARED = [
    # kind, lens, hq, hkv, hd, page, more
    ("warp", MANY, 2, 2, 64, 16, {}),
    ("warp", MANY, 6, 2, 128, 64, {}),
    ("warp", MANY, 6, 2, 256, 32, {}),
    ("warp", MANY, 26, 2, 64, 64, dict(window=20)),
    ("warp", MANY, 36, 2, 128, 48, dict(window=64)),
    ("warp", MANY, 24, 2, 256, 16, dict(window=1)),
    ("chunks", UNEVEN, 4, 2, 64, 64, {}),
    ("chunks", UNEVEN, 12, 2, 128, 16, dict(window=1500)),
    ("chunks", UNEVEN, 32, 2, 128, 64, {}),
    ("chunks", UNEVEN, 16, 2, 256, 48, dict(window=2047)),
    ("chunks", [9000, 0, 2500, 1, 20000, 64], 5, 5, 64, 64, {}),
    ("chunks", [9000, 0, 2500, 1, 20000, 64], 16, 4, 256, 64, {}),
    ("cluster", [700, 64, 0, 1], 4, 2, 128, 64, {}),
    ("cluster", [1000] + [900 - i for i in range(199)], 2, 1, 128, 64, {}),
    ("cluster", [5000, 300, 4999, 0], 4, 2, 64, 64, {}),
    ("cluster", [5000, 300, 4999, 0], 10, 2, 128, 48, dict(window=3000)),
    ("cluster", [5000, 300, 4999, 0], 10, 2, 256, 16, {}),
]


@gpu
@DTYPES
@pytest.mark.parametrize("case", SHARED, ids=lambda c: f"{c[0]}-{len(c[1])}x{c[2]}-{c[3]}x{c[4]}")
def test_decode_however_it_is_shared_out(case, dtype):
    kind, lens, hq, hkv, hd, page, more = case
    assert shared_out(lens, hq, hkv, hd) == kind
    decode_case(lens, hq, hkv, hd, page, dtype, device="cuda", max_seq_len=max(lens), **more)
    ops.raise_on_status()


@gpu
@DTYPES
@pytest.mark.parametrize("kind,lens,hkv", [("warp", [33] * 310, 1), ("chunks", [40, 20000, 33, 2500], 2), ("cluster", [300, 40], 2)])
def test_decode_rows_that_are_nan_however_it_is_shared_out(kind, lens, hkv, dtype):
    """One key, and one value, of one sequence each: NaN there, in no other sequence or head, and nowhere when the window hides them."""
    k, v, table, sl = paged(lens, hkv, 64, 128, dtype, 5, "cuda")
    q = torch.randn(len(lens), 4 * hkv, 128, device="cuda").bfloat16()
    assert shared_out(lens, 4 * hkv, hkv, 128) == kind
    for cache, seq in ((k, 0), (v, 1)):
        page = int(table[seq, 0])
        cache.exponents[page, 0, 3] = 255
        cache.codes.view(torch.uint8)[page, 0, 3] = 0
    got = ops.paged_decode(q, k, v, table, sl, max_seq_len=max(lens)).isnan().view(len(lens), hkv, -1)
    want = torch.zeros(len(lens), hkv, 1, dtype=torch.bool, device="cuda")
    want[:2, 0] = True
    assert torch.equal(got, want.expand_as(got))
    assert not bool(ops.paged_decode(q, k, v, table, sl, window=29, max_seq_len=max(lens)).isnan().any())


@gpu
def test_decode_of_more_sequences_than_are_cut():
    """8200 sequences: none is cut, however long."""
    lens = [4000 if i == 8000 else i % 6 for i in range(8200)]
    assert shared_out(lens, 2, 1, 64) == "warp"
    k, v, table, sl = paged(lens, 1, 16, 64, INT8, 5, "cuda")
    q = torch.randn(len(lens), 2, 64, device="cuda").bfloat16()
    out = ops.paged_decode(q, k, v, table, sl)
    at = torch.tensor([0, 1, 5, 4095, 4096, 7999, 8000, 8001, 8199], device="cuda")
    check_attention(out[at], q[at], k, v, table[at], sl[at], None, 0.125, 0)
    for n in range(0, len(lens), 1000):
        part = slice(n, n + 1000)
        few = ops.paged_decode(q[part], k, v, table[part], sl[part]).float()
        assert float((few - out[part].float()).abs().max()) <= 2.0 ** -7 * float(few.abs().max())      # a rounding to bf16 on each side


@gpu
@pytest.mark.parametrize("stock", ["stock", "none", "at its end"])
def test_decode_of_cut_pairs_in_graphs_and_streams(stock, monkeypatch):
    """Captured calls that draw tickets: of a stock, or of an allocation of their own.  Lengths change on the device between replays, two graphs run on
    two streams at once, and eager calls run beside them."""
    lens = [[9000, 40, 2000, 64], [1, 33, 500, 0], [0, 8999, 64, 4000]]
    assert shared_out(lens[0], 16, 4, 128) == "chunks"
    k, v, table, _ = paged([9000, 9000, 9000, 9000], 4, 64, 128, E4M3, 5, "cuda")
    q = torch.randn(4, 16, 128, device="cuda").bfloat16()
    sls = [torch.tensor(n, dtype=torch.int32, device="cuda") for n in lens]
    want = [ops.paged_decode(q, k, v, table, n) for n in sls]
    for i, n in enumerate(lens):
        check_attention(want[i], q, k, v, table, sls[i], None, 1 / math.sqrt(128), 0)
    if stock == "none":
        monkeypatch.setattr(kv8, "_CAPTURED", {})
    elif stock == "at its end":
        monkeypatch.setattr(kv8, "CAPTURED_TICKETS", 1)
    graphs, outs, now = [], [], []
    for _ in range(2):
        n = sls[0].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([ops.paged_decode(q, k, v, table, n) for _ in range(2)])
        graphs.append(g)
        now.append(n)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for i in range(9):
        pick = [i % 3, (i + 1) % 3]
        for n, p in zip(now, pick):
            n.copy_(sls[p])
        torch.cuda.synchronize()
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        with torch.cuda.stream(streams[2]):
            eager = [ops.paged_decode(q, k, v, table, sls[j]) for j in range(3)]
        torch.cuda.synchronize()
        for o, p in zip(outs, pick):
            assert torch.equal(o[0], want[p]) and torch.equal(o[1], want[p])
        for j in range(3):
            assert torch.equal(eager[j], want[j])


# ------------------------------------------------------------------ prompts over pages of any size
@gpu
@pytest.mark.parametrize("page", [16, 48, 64, 112, 128, 320])
def test_prompts_over_pages_of_any_size(page):
    """The reader's pages for prompts hold 64 tokens: the same rows whatever the cache's pages hold, zeros behind a sequence's end."""
    lens = [0, 1, 63, 64, 65, 700, 129]
    k, v, table, sl = paged(lens, 2, page, 128, INT8, 5, "cuda")
    width = -(-table.shape[1] * page // 64)
    held = [-(-n // 64) for n in lens]
    kd, vd, t = kv8._read(k, v, table, sl, 64, width, sum(held))
    at = 0
    for i, (n, m) in enumerate(zip(lens, held)):
        assert t[i].tolist() == list(range(at, at + m)) + [0] * (width - m)
        for got, cache in ((kd, k), (vd, v)):
            rows = got[at:at + m].reshape(m * 64, 2, 128)
            assert torch.equal(rows[:n].double(), sequence64(cache, table[i], n)) and not bool(rows[n:].any())
        at += m
    ops.raise_on_status()
    parts = [(1, 0), (63, 1), (64, 200), (65, 0), (130, 570)]
    for more in ({}, dict(max_seq_len=700, kv_pages=sum(-(-(a + b) // page) for a, b in parts)), dict(max_seq_len=700)):
        prefill_case(parts, 8, 2, 128, page, 0, E4M3, "cuda", **more)
    prefill_case(parts, 8, 2, 64, page, 100, INT8, "cuda")
    ops.raise_on_status()


@gpu
def test_prompts_report_a_page_that_is_none():
    k, v, table, sl = paged([100], 2, 16, 64, E4M3, 5, "cuda")
    q = torch.randn(3, 4, 64, device="cuda").bfloat16()
    for bad in (-1, k.codes.shape[0]):
        table[0, 5] = bad
        ops.paged_prefill(q, k, v, table, sl, torch.tensor([0, 3], dtype=torch.int32, device="cuda"))
        with pytest.raises(ops.KernelError):
            ops.raise_on_status()


def check_prompt_edges(device):
    """Lengths that reach beyond the table count as far as it goes, and below zero as none; sequences without keys, a table without columns, and rows
    behind the last sequence, which are left as they are."""
    k, v, table, _ = paged([128, 128, 128], 2, 64, 64, E4M3, 5, device)
    q = torch.randn(9, 4, 64, generator=torch.Generator().manual_seed(4)).bfloat16().to(device)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)
    starts = ints(0, 3, 3, 6)
    want = ops.paged_prefill(q[:6], k, v, table, ints(128, 0, 128), starts)
    assert torch.equal(ops.paged_prefill(q[:6], k, v, table, ints(10 ** 6, -5, 129), starts), want)
    check_attention(want, q, k, v, table, ints(128, 0, 128), starts.tolist(), 0.125, 0)
    if device != "cpu":
        out = torch.full((9, 4, 64), 7.0, dtype=torch.bfloat16, device=device)
        assert ops.paged_prefill(q, k, v, table, ints(128, 0, 128), starts, out=out) is out
        assert torch.equal(out[:6], want) and bool((out[6:] == 7).all())
        ops.raise_on_status()
    for bt, more in ((table, dict(max_seq_len=0, kv_pages=0)), (table, {}), (table[:, :0].contiguous(), {})):
        none = ops.paged_prefill(q[:0], k, v, bt, ints(0, 0, 0), ints(0, 0, 0, 0), **more)
        assert none.shape == (0, 4, 64)
        assert ops.paged_read(k, v, bt, ints(0, 0, 0), num_pages=0)[0].shape == (0, 64, 2, 64)
        assert not bool(ops.paged_decode(q[:3], k, v, bt, ints(0, 0, 0)).any())
    if device != "cpu":
        ops.raise_on_status()


def test_prompt_edges_cpu():
    check_prompt_edges("cpu")


@gpu
def test_prompt_edges():
    check_prompt_edges("cuda")


@gpu
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_outputs_at_any_address(shift):
    """Outputs that start on 2, 4 or 8 bytes."""
    lens = [70, 200]
    k, v, table, sl = paged(lens, 2, 64, 128, E4M3, 5, "cuda")
    q = torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(6)).bfloat16().cuda()
    at = lambda *shape: torch.full((math.prod(shape) + 8,), 7.0, dtype=torch.bfloat16, device="cuda")
    flat = at(2, 8, 128)
    out = flat[shift:shift + 2048].view(2, 8, 128)
    assert ops.paged_decode(q, k, v, table, sl, out=out) is out
    assert torch.equal(out, ops.paged_decode(q, k, v, table, sl)) and bool((flat[:shift] == 7).all()) and bool((flat[shift + 2048:] == 7).all())
    qkv = torch.randn(5, 12 * 128, generator=torch.Generator().manual_seed(7)).bfloat16().cuda()
    pos, freq = torch.arange(5, dtype=torch.int32, device="cuda"), torch.ones(64, device="cuda")
    flat = at(5, 8, 128)
    out = flat[shift:shift + 5 * 8 * 128].view(5, 8, 128)
    assert ops.rope_kvwrite(qkv, pos, pos, freq, k, v, 8, 2, 128, q_out=out) is out
    want = ops.rope_kvwrite(qkv, pos, pos, freq, k, v, 8, 2, 128)
    err = (out.double() - want.double()).abs()                # two kernels: each rounds once to bf16, fp32 before that
    assert bool((err <= 2 * 2.0 ** -8 * want.double().abs() + 2.0 ** -17).all())
    assert bool((flat[:shift] == 7).all()) and bool((flat[shift + 5 * 8 * 128:] == 7).all())
    ops.raise_on_status()
