"""Attention behind a shared prefix where lengths, scores and sizes are at their ends, against softmax attention in 64 bits."""
import math

import pytest
import torch

from test_shared_attention import call, check, make
from zml_b200 import ops

gpu = pytest.mark.gpu

HEADS = [(8, 2, 64), (32, 2, 128), (20, 1, 128), (8, 2, 256)]              # 4, 16 and 20 heads to a key head; heads of 64, 128 and 256


def shortened(lens, heads=(8, 2, 64), behind=None, prefix=700, page=64):
    """A group of len(lens) members behind `prefix` shared keys, shortened to `lens` keys, the members in this order; keys from `behind` (the longest
    member's end) on hold NaN and infinities.  The table's row of a member without keys is zero.  One sequence is in no group."""
    hq, hkv, hd = heads
    s = make([(prefix, [page] * len(lens))], (90,), hq, hkv, hd, page, seed=len(lens) + hd, nan_behind=False)
    rows = s["shared"].rows.tolist()
    behind = max(lens) if behind is None else behind
    for row, n in zip(rows, lens):
        for at in range(behind // page, s["table"].shape[1]):
            first = max(behind - at * page, 0)
            mine = int(s["table"][row, at])
            if at < prefix // page + 1:
                s["k"][mine, first:], s["v"][mine, first:] = math.nan, math.inf
        s["lens"][row] = n
        if n == 0:
            s["table"][row] = 0
    return {**{n: t.cuda() for n, t in s.items() if n != "shared"}, "shared": ops.SharedPrefix.of([(rows, prefix)], "cuda")}


@gpu
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("lens", [(500, 300, 1), (0, 500, 640), (0, 0, 699), (65, 65, 65), (0, 0, 0), (700, 0, 10), (764, 3, 700), (1, 64, 128)])
def test_members_that_end_inside_of_the_prefix(lens, heads):
    s = shortened(lens, heads)
    got = call(s)
    ops.raise_on_status()
    check(got, s)
    assert not got[s["lens"] == 0].any()


@gpu
@pytest.mark.parametrize("heads", HEADS)
def test_a_member_does_not_see_what_only_longer_ones_do(heads):
    s = shortened((640, 300, 0, 301), heads, behind=301)
    got, few = call(s), [i for i, n in enumerate(s["lens"].tolist()) if n <= 301]
    assert len(few) == 4
    check(got[few], {**s, "q": s["q"][few], "table": s["table"][few], "lens": s["lens"][few]})
    assert not got[s["lens"] == 0].any()
    ops.raise_on_status()


@gpu
def test_a_captured_call_whose_first_member_ends():
    s = shortened((764, 720, 701, 710))
    rows = s["shared"].rows.tolist()
    call(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(s)
    for dead in (rows[:1], rows[:3], rows):           # the groups stay as they are
        for row in dead:
            s["lens"][row] = 0
            s["table"][row] = 0
        s["k"][0], s["v"][0] = math.nan, math.nan     # nobody's page, where the ended ones' rows of the table point
        graph.replay()
        live = [i for i, n in enumerate(s["lens"].tolist()) if n > 0 and 0 not in s["table"][i, :-(-n // 64)].tolist()]
        check(out[live], {**s, "q": s["q"][live], "table": s["table"][live], "lens": s["lens"][live]})
        assert not out[s["lens"] == 0].any()
    ops.raise_on_status()


@gpu
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 15, 2.0 ** 16, 2.0 ** 25, 2.0 ** 40])
def test_scores_that_are_whole_numbers_in_fp32(size, heads):
    """Scores of size^2, where fp32 has no fractions: all of the weight is on the largest one, which is further from the second than sums of hd
    products are off (hd 2^-23 of their magnitudes' sum)."""
    hq, hkv, hd = heads
    s = make([(900, [0, 100, 300])], (65,), hq, hkv, hd, 64, seed=hd, device="cuda")
    s["q"], s["k"] = s["q"] * size, s["k"] * size
    got = call(s).cpu()
    ops.raise_on_status()
    q, k, v, table = (s[n].cpu() for n in ("q", "k", "v", "table"))
    told = 0
    for i, n in enumerate(s["lens"].tolist()):
        at = table[i, :-(-n // 64)].long()
        kk, vv = (c[at].flatten(0, 1)[:n].double().permute(1, 0, 2) for c in (k, v))
        qq = q[i].double().unflatten(0, (hkv, -1))
        score, mag = qq @ kk.mT, (qq.abs() @ kk.abs().mT).amax(-1)
        top = score.topk(2, -1)
        far = top.values[..., 0] - top.values[..., 1] > 2 * hd * 2.0 ** -23 * mag + 200 * hd ** 0.5
        want = vv.gather(1, top.indices[..., :1].expand(-1, -1, hd)).flatten(0, 1)
        far = far.flatten()
        told += int(far.sum())
        assert bool(got[i].isfinite().all())
        assert bool(((got[i].double() - want)[far].abs() <= 2.0 ** -7 * want[far].abs()).all())
    assert told >= 3 * hq
