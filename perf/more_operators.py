"""Timed cases of answering one prompt many times: attention of single tokens that share a prefix, and the draw of the next tokens.

"shared": one query token for each sequence over all of its keys.  Sequences come in groups whose first keys are the same pages of the cache (the
answers to one prompt, the users of one long instruction); behind them every sequence has keys of its own.  Caches are [pages, page, heads, hd] in
bfloat16; `lens` are keys per sequence, those shared among them; a sequence without keys (a row that pads a batch) gives zeros.

"sample": one token a row of logits.  With weights w_i = exp((x_i - max x) / temperature), in this order:
* only the `top_k` largest logits stay (0: all; of equal logits those of lower index);
* of these, from the largest down, a token stays while the weights in front of it are less than `top_p` of the sum of all (1 or more: all stay);
* and while w_i >= `min_p`;
* the token is the first one, in the vocabulary's order, up to which the weights that stayed sum to more than `uniform` times their whole sum.
A temperature of zero takes the first of the largest logits.  The second output is the logarithm of the probability that the token was drawn with.

Head layouts and vocabularies are those of the presets in `zml_b200.models`.  Lengths of a batch are spread evenly over [shortest, longest] in a
shuffled order that the case alone decides; block tables are shuffled, and the rows of a group lie anywhere in the batch.
"""
from __future__ import annotations

import math
import random

import torch

own = False
DEVICE = "cuda"
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16}


def _shared(name, hq, hkv, hd, page, groups, members, prefix, suffix, empty=0):
    """`groups` groups of members[0] to members[1] sequences; keys that a group shares, and that a sequence has of its own: [shortest, longest]."""
    return {"name": name, "do": "shared", "hq": hq, "hkv": hkv, "hd": hd, "page": page, "groups": groups, "fewest": members[0], "most": members[1],
            "prefix_shortest": prefix[0], "prefix_longest": prefix[1], "suffix_shortest": suffix[0], "suffix_longest": suffix[1], "empty": empty}


def _sample(name, rows, vocab, temperature, top_k=0, top_p=1.0, min_p=0.0, dtype="f32", spread=2.5, peak=5.0, masked=0.0, mixed=False, pad=0):
    """Logits N(0, spread), some of them raised by about `peak`; a part `masked` of the vocabulary is forbidden; `mixed`: every row has settings of
    its own; rows of the logits lie vocab + pad apart."""
    return {"name": name, "do": "sample", "rows": rows, "vocab": vocab, "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p,
            "dtype": dtype, "spread": spread, "peak": peak, "masked": masked, "mixed": mixed, "pad": pad}


def listed():
    return [
        # eight answers to one question, at their beginning: latency
        _shared("shared-8-answers", 32, 8, 128, 64, 1, (8, 8), (2000, 2000), (1, 40)),
        # 32 attempts at one problem with a long statement, heads of 64
        _shared("shared-32-attempts", 32, 8, 64, 64, 1, (32, 32), (8192, 8192), (1, 512)),
        # three prompts with some answers each, heads of 256; rows that pad the batch
        _shared("shared-3-prompts", 16, 4, 256, 64, 3, (3, 7), (1500, 5000), (100, 700), 1),
        # small pages, five query heads to a key head, many small groups of unequal size
        _shared("shared-9-groups", 40, 8, 128, 16, 9, (1, 9), (100, 2500), (0, 300), 3),
        # 128 users behind one instruction, eight query heads to a key head
        _shared("shared-128-users", 32, 4, 128, 64, 1, (128, 128), (4133, 4133), (64, 1500)),
        # 64 questions about one book
        _shared("shared-64-of-65536", 32, 8, 128, 64, 1, (64, 64), (65536, 65536), (16, 256)),
        # one user's chat: latency
        _sample("sample-1-chat", 1, 128256, 0.7, top_p=0.9),
        # a batch of users, every one with settings of their own
        _sample("sample-32-mixed", 32, 128256, 1.0, mixed=True),
        # half-precision logits, answers held to a grammar, high temperature
        _sample("sample-16-grammar", 16, 65536, 1.5, min_p=0.05, dtype="bf16", spread=2.0, peak=3.0, masked=0.6, pad=8),
        # rollouts: the whole distribution
        _sample("sample-64-rollouts", 64, 151936, 1.0),
        # what many models' generation settings say
        _sample("sample-128-top-k", 128, 248320, 0.6, top_k=50, top_p=0.95),
        # a large batch, and a nucleus of very many tokens where logits are flat
        _sample("sample-256-nucleus", 256, 151936, 1.0, top_p=0.95, spread=1.5, peak=4.0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """Any of the above with other heads, sizes and settings, at most as much as the largest listed one of its kind."""
    case = _drawn_shared(rng) if rng.random() < 0.5 else _drawn_sample(rng)
    del case["name"]
    return case


def _drawn_shared(rng):
    hd = rng.choice([64, 128, 128, 256])
    hkv = rng.choice([1, 2, 3, 4, 5, 8, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 8, 12, 16])
    groups = rng.choice([1, 1, 1, 2, 3, 5, 8, 13, 21])
    most = _log_int(rng, 1, max(1, 160 // groups))
    fewest = _log_int(rng, max(1, most // 4), most)
    rows = groups * most
    suffix = _log_int(rng, 1, max(1, min(16000, 128 * 1500 * 512 // (rows * hkv * hd)))) - 1
    room = 65536 * 1024 - rows * suffix * hkv * hd // 2
    longest = min(room // (groups * hkv * hd), 64 * 4096 * 65536 // (rows * hq * hd))              # keys that may be shared
    prefix = _log_int(rng, 1, max(1, min(65536, longest)))
    return _shared("", hq, hkv, hd, rng.choice([16, 32, 64, 64, 64, 128]), groups, (fewest, most), (_log_int(rng, max(1, prefix // 8), prefix), prefix),
                   (rng.randint(0, suffix), suffix), rng.choice([0, 0, 0, 1, 2, 5]))


def _drawn_sample(rng):
    vocab = rng.choice([128256, 151936, 248320, 65536, _log_int(rng, 1000, 262144), _log_int(rng, 1000, 262144)])
    rows = _log_int(rng, 1, min(256, 256 * 151936 // vocab))
    flat = rng.random() < 0.25
    return _sample("", rows, vocab, round(rng.choice([1.0, 1.0, rng.uniform(0.3, 2.0)]), 3), rng.choice([0, 0, 1, 20, 50, _log_int(rng, 2, vocab)]),
                   rng.choice([1.0, 0.9, 0.95, round(rng.uniform(0.05, 0.999), 4)]), rng.choice([0.0, 0.0, 0.05, round(rng.uniform(0.001, 0.5), 4)]),
                   rng.choice(["f32", "f32", "f32", "bf16"]), round(rng.uniform(0.2, 1.5) if flat else rng.uniform(1.5, 3.5), 2),
                   0.0 if flat else round(rng.uniform(0.0, 8.0), 2), rng.choice([0.0, 0.0, 0.3, 0.9]), rng.random() < 0.25, rng.choice([0, 0, 1, 8, 64]))


# ------------------------------------------------------------------------------------------ sizes
def _spread(n, lo, hi, salt):
    out = [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]
    random.Random(1000003 * n + 1009 * lo + hi + salt).shuffle(out)
    return out


def _layout(case):
    """(group of every row or -1, keys that each group shares, keys of every row)."""
    members = _spread(case["groups"], case["fewest"], case["most"], 1)
    prefix = _spread(case["groups"], case["prefix_shortest"], case["prefix_longest"], 2)
    group = [g for g, n in enumerate(members) for _ in range(n)]
    own_keys = _spread(len(group), case["suffix_shortest"], case["suffix_longest"], 3)
    rows = [(g, prefix[g] + n) for g, n in zip(group, own_keys)] + [(-1, 0)] * case["empty"]
    random.Random(17 + len(rows)).shuffle(rows)
    return [g for g, _ in rows], prefix, [n for _, n in rows]


def work(case):
    if case["do"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["dtype"] == "f32" else 2) + case["rows"] * 12, "flops": 4 * n}
    group, prefix, lens = _layout(case)
    keys = sum(prefix) + sum(n - prefix[g] for g, n in zip(group, lens) if g >= 0)
    return {"bytes": keys * 4 * case["hkv"] * case["hd"] + len(lens) * 4 * case["hq"] * case["hd"], "flops": 4 * case["hq"] * case["hd"] * sum(lens)}


# ------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    return _prepare_sample(case, g) if case["do"] == "sample" else _prepare_shared(case, seed, g)


def _prepare_shared(case, seed, g):
    group, prefix, lens = _layout(case)
    page, hkv, hd = case["page"], case["hkv"], case["hd"]
    common = [p // page for p in prefix]                                         # whole pages are shared
    # a page that a prefix fills in part belongs to each sequence, which holds the same tokens in it
    held = [-(-n // page) for n in lens]
    pages = 1 + sum(common) + sum(h - common[i] for i, h in zip(group, held) if i >= 0)
    order = torch.randperm(pages - 1, generator=torch.Generator().manual_seed(seed)).add(1).tolist()
    table = torch.zeros((len(lens), max(1, max(held))), dtype=torch.int32)
    first, at = [], 0
    for n in common:
        first.append(order[at:at + n])
        at += n
    for i, (j, n) in enumerate(zip(group, held)):
        if j >= 0:
            mine = first[j] + order[at:at + n - common[j]]
            at += n - common[j]
            table[i, :n] = torch.tensor(mine, dtype=torch.int32)
    channel = torch.empty((1, 1, hkv, hd), device=DEVICE).normal_(0.0, 0.5, generator=g).exp_()
    k = torch.empty((pages, page, hkv, hd), device=DEVICE).normal_(generator=g).mul_(channel).bfloat16()
    v = torch.empty((pages, page, hkv, hd), device=DEVICE).normal_(generator=g).bfloat16()
    table = table.to(DEVICE)
    rows = [[i for i, j in enumerate(group) if j == n] for n in range(case["groups"])]
    for n, members in enumerate(rows):                                           # the rest of a prefix, in each member's own page
        rest = prefix[n] - common[n] * page
        if rest:
            mine = table[torch.tensor(members, device=DEVICE), common[n]].long()
            for cache in (k, v):
                cache[mine[1:], :rest] = cache[mine[0], :rest]
    starts = [0]
    for members in rows:
        starts.append(starts[-1] + len(members))
    i32 = dict(dtype=torch.int32, device=DEVICE)
    return {"case": case, "k": k, "v": v, "table": table, "lens": torch.tensor(lens, **i32), "longest": max(lens), "longest_prefix": max(prefix),
            "longest_suffix": max(n - prefix[j] for j, n in zip(group, lens) if j >= 0), "most": max(len(m) for m in rows),
            "rows": torch.tensor([i for m in rows for i in m], **i32), "starts": torch.tensor(starts, **i32), "shared": torch.tensor(prefix, **i32),
            "q": torch.empty((len(lens), case["hq"], hd), device=DEVICE).normal_(generator=g).bfloat16()}


def _prepare_sample(case, g):
    n, vocab = case["rows"], case["vocab"]
    x = torch.empty((n, vocab + case["pad"]), device=DEVICE).normal_(0.0, case["spread"], generator=g)
    some = torch.randint(0, vocab, (n, 64), device=DEVICE, generator=g)
    x.scatter_add_(1, some, torch.empty((n, 64), device=DEVICE).exponential_(1.0, generator=g).mul_(case["peak"]))
    if case["masked"]:
        x.masked_fill_(torch.rand(x.shape, device=DEVICE, generator=g) < case["masked"], -math.inf)
        x[:, 0] = 0.0                                                            # the end of the text is allowed everywhere
    settings = {name: case[name] for name in ("temperature", "top_k", "top_p", "min_p")}
    if case["mixed"]:
        def choose(values, dtype):
            at = torch.randint(0, len(values), (n,), device=DEVICE, generator=g)
            return torch.tensor(values, dtype=dtype, device=DEVICE)[at]
        settings = {"temperature": choose([0.0, 0.3, 0.7, 1.0, 1.0, 1.4], torch.float32), "top_k": choose([0, 0, 1, 20, 50, 1000], torch.int32),
                    "top_p": choose([1.0, 1.0, 0.9, 0.95, 0.5], torch.float32), "min_p": choose([0.0, 0.0, 0.05, 0.2], torch.float32)}
    return {"case": case, "logits": x.to(DTYPE[case["dtype"]])[:, :vocab], "uniforms": torch.rand(n, device=DEVICE, generator=g), **settings}


# ------------------------------------------------------------------------------------------ a pass
def run(state):
    if own:
        return _own(state)
    return _plain_sample(state) if state["case"]["do"] == "sample" else _plain_shared(state)


def _own(s):
    from zml_b200 import ops
    if s["case"]["do"] == "sample":
        token, logprob = ops.sample(s["logits"], s["uniforms"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], return_logprobs=True)
        return {"token": token, "logprob": logprob}
    shared = ops.SharedPrefix(s["rows"], s["starts"], s["shared"])
    return ops.paged_decode(s["q"], s["k"], s["v"], s["table"], s["lens"], max_seq_len=s["longest"], shared=shared)


# ------------------------------------------------------------------------------------------ plain form
def _plain_shared(s):
    """Scores of a group's queries over the keys that they share and of every query over its own, one softmax over both, in 32 bits."""
    c = s["case"]
    hkv, hd, page = c["hkv"], c["hd"], c["page"]
    count = (s["starts"][1:] - s["starts"][:-1]).long()
    nth = torch.arange(s["most"], device=DEVICE)
    at = (s["starts"][:-1].long()[:, None] + nth).clamp_max(s["rows"].shape[0] - 1)
    row = s["rows"].long()[at]                                                   # [groups, most]; those past a group's end are left out below
    valid = nth < count[:, None]
    q = s["q"].float()[row].unflatten(2, (hkv, -1)).transpose(1, 2) / math.sqrt(hd)      # [groups, hkv, most, heads, hd]
    place = torch.arange(s["longest_prefix"], device=DEVICE)
    page_of = s["table"].long()[row[:, 0]][:, place // page]
    k, v = (s[n][page_of, place % page].float().transpose(1, 2) for n in ("k", "v"))     # [groups, hkv, prefix, hd]
    front = (q.flatten(2, 3) @ k.transpose(-1, -2)).unflatten(2, (s["most"], -1))
    front = front.masked_fill((place >= s["shared"][:, None])[:, None, None, None], -math.inf)
    more = s["shared"].long()[:, None, None] + torch.arange(max(1, s["longest_suffix"]), device=DEVICE)      # [groups, 1, suffix]
    seen = (more < s["lens"].long()[row][:, :, None])
    near = more.clamp_max(s["longest"] - 1).expand(seen.shape)
    page_of = s["table"].long()[row[:, :, None], near // page]
    k_own, v_own = (s[n][page_of, near % page].float().permute(0, 3, 1, 2, 4) for n in ("k", "v"))          # [groups, hkv, most, suffix, hd]
    back = (q @ k_own.transpose(-1, -2)).masked_fill(~seen[:, None, :, None], -math.inf)
    top = torch.maximum(front.amax(-1, keepdim=True), back.amax(-1, keepdim=True)).clamp_min(-1e30)
    p, p_own = torch.exp(front - top), torch.exp(back - top)
    total = p.sum(-1, keepdim=True) + p_own.sum(-1, keepdim=True)
    o = ((p.flatten(2, 3) @ v).unflatten(2, (s["most"], -1)) + p_own @ v_own) / total.clamp_min(1e-30)
    out = torch.zeros(s["q"].shape, device=DEVICE)
    out[row[valid]] = o.transpose(1, 2).flatten(2, 3)[valid]
    return out.bfloat16()


def _column(value, like):
    return value.double()[:, None] if isinstance(value, torch.Tensor) else torch.full((like.shape[0], 1), float(value), dtype=torch.float64, device=like.device)


def _plain_sample(s):
    """By sorting, in 64 bits: the sums are long, and a token lies next to a border."""
    x = s["logits"]
    temperature, top_k, top_p, min_p = (_column(s[n], x) for n in ("temperature", "top_k", "top_p", "min_p"))
    x, index = torch.sort(x, dim=-1, descending=True, stable=True)
    x = x.double()
    place = torch.arange(x.shape[1], device=x.device)
    w = torch.exp((x - x[:, :1]) / torch.where(temperature > 0, temperature, 1.0))
    w = w.masked_fill((place >= top_k) & (top_k > 0) | (place > 0) & (temperature <= 0), 0.0)
    upto = w.cumsum(-1)
    keep = ((upto - w < top_p * upto[:, -1:]) | (top_p >= 1.0)) & (w >= min_p)
    w = torch.zeros_like(w).scatter_(1, index, w.masked_fill(~keep, 0.0))
    upto = w.cumsum(-1)
    total = upto[:, -1:]
    token = torch.searchsorted(upto, s["uniforms"].double()[:, None] * total, right=True)
    return {"token": token[:, 0].int(), "logprob": torch.log(w.gather(1, token) / total)[:, 0].float()}


# ------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return _exact_sample(state) if case["do"] == "sample" else _exact_shared(state)


def _exact_shared(state):
    """Sequence after sequence, each over all of its keys."""
    case, lens = state["case"], state["lens"].tolist()
    if sum(lens) * case["hq"] * case["hd"] > 3 << 33:
        return None
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device=DEVICE)
    for i, n in enumerate(lens):
        if n == 0:
            continue
        pages = state["table"][i, :-(-n // case["page"])].long()
        k, v = (state[name][pages].flatten(0, 1)[:n].double().permute(1, 0, 2) for name in ("k", "v"))
        q = state["q"][i].double().reshape(case["hkv"], -1, case["hd"])
        out[i] = torch.bmm(torch.softmax(torch.bmm(q, k.mT) * case["hd"] ** -0.5, dim=-1), v).reshape(case["hq"], case["hd"])
    return out


def _exact_sample(state):
    """Row after row: a threshold on the logits and a number of ties that stay, then the weights in the vocabulary's order."""
    rows = state["logits"].shape[0]
    setting = lambda name, i: float(state[name][i]) if isinstance(state[name], torch.Tensor) else float(state[name])  # noqa: E731
    tokens, logprobs = [], []
    for i in range(rows):
        x = state["logits"][i].double()
        best, temperature = x.max(), setting("temperature", i)
        if temperature <= 0:
            tokens.append(int((x == best).nonzero()[0]))
            logprobs.append(0.0)
            continue
        w = ((x - best) / temperature).exp()
        stays = torch.ones_like(x, dtype=torch.bool)
        k, p, m = int(setting("top_k", i)), setting("top_p", i), setting("min_p", i)
        if 0 < k < x.numel():
            last = torch.topk(x, k).values[-1]
            stays = (x > last) | ((x == last) & ((x == last).cumsum(0) <= k - (x > last).sum()))
        if p < 1.0:
            goes = torch.where(stays, w, 0.0)
            values, ties = torch.unique(x[stays], return_counts=True)
            values, ties = values.flip(0), ties.flip(0)
            each = ((values - best) / temperature).exp()
            mass = (each * ties).cumsum(0)
            need = p * goes.sum()
            j = int((mass < need).sum().clamp_max(values.numel() - 1))
            before = mass[j - 1] if j else mass.new_zeros(())
            left = max(1, int(torch.ceil((need - before) / each[j]))) if float(each[j]) > 0 else 1
            stays = stays & ((x > values[j]) | ((x == values[j]) & ((stays & (x == values[j])).cumsum(0) <= left)))
        stays = stays & (w >= m)
        upto = torch.where(stays, w, 0.0).cumsum(0)
        token = int((upto <= float(state["uniforms"][i]) * upto[-1]).sum())
        tokens.append(token)
        logprobs.append(float((x[token] - best) / temperature - upto[-1].log()))
    return {"token": torch.tensor(tokens, dtype=torch.int32), "logprob": torch.tensor(logprobs, dtype=torch.float64)}
