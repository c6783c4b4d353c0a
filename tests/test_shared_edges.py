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


@gpu
@pytest.mark.parametrize("batch,hq,hkv,hd", [(1, 128, 1, 128), (8, 66, 1, 64), (64, 34, 2, 256), (64, 32, 8, 128), (8, 32, 2, 64)])
def test_the_workspace_has_room_for_the_parts_and_little_else(batch, hq, hkv, hd):
    """A row of fp32 sums and two numbers for each head of a sequence, in its prefix and behind it, and again for each piece that the keys are cut into: at most
    two CTAs an SM of 128 rows in front, and of a key head's rows behind - six of these a CTA up to 16 heads, whose keys single warps read."""
    lib = ops._lib.lib()
    group, ctas = hq // hkv, 2 * lib.zb_num_sms()
    most = 32 * batch + 4 * (hd + 2) * (2 * batch * hq + ctas * 128 + ctas * (6 if group <= 16 else 1) * group + 1)
    assert 4 * (hd + 2) * 2 * batch * hq < lib.zb_shared_decode_workspace(batch, batch, 1, hq, hkv, hd, 64) <= most


@gpu
@pytest.mark.parametrize("hq,hkv,hd", [(128, 1, 128), (66, 1, 64), (34, 2, 256), (17, 1, 128)])
def test_parts_of_many_heads_to_a_key_head_stay_in_the_workspace(hq, hkv, hd):
    """Long keys of few and of many sequences, so that every CTA has a piece of either line; what lies behind the workspace is left as it was."""
    for groups, alone in (([(3000, [2500, 1])], (4000,)), ([(64, [700] * 40)], ()), ([], (9000,)), ([(9000, [0])], ()), ([(130, [1] * 150)], (1,) * 50)):
        s = make(groups, alone, hq, hkv, hd, 64, seed=hq, device="cuda")
        guard, new_empty = [], torch.Tensor.new_empty

        class Q(torch.Tensor):
            def new_empty(self, shape, **kw):
                if kw.get("dtype") is not torch.uint8:
                    return new_empty(self.as_subclass(torch.Tensor), shape, **kw)
                whole = torch.full((shape[0] + 4096,), 77, dtype=torch.uint8, device="cuda")
                guard.append(whole[shape[0]:])
                return whole[:shape[0]]
        got = call({**s, "q": s["q"].as_subclass(Q)})
        check(got, s)
        assert len(guard) == 1 and bool((guard[0] == 77).all())
    ops.raise_on_status()
