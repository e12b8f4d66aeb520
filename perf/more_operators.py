"""Performance cases of the operators around a KV cache that requests share and shrink.

Requests of a step often begin with the same cached tokens (a system prompt, samples
of one prompt, turns of one conversation), and long contexts keep only the tokens
that attention looks at.

* ``shared`` cases call ``shared_prefix_attention``: the shared tokens' keys and values
  are read once for all requests of a group;
* ``scored`` cases call ``scored_attention``: attention that also sums up the weight
  that every cached token gets;
* ``evict`` cases call ``evict_tokens``: the tokens of the least weight leave the
  request's row of the slot table.

``own`` False computes the operators from elementary torch operations in fp32.
"""
from __future__ import annotations

import math
import random

import torch

own = False

E4M3_MAX = 448.0


def _shared(name, groups, members, prefix, suffix, loose=0, new=1, heads=(24, 4), dim=256,
            fp8=False):
    return _named(name, dict(kind="shared", groups=groups, members=members, prefix=prefix,
                             suffix=suffix, loose=loose, new=new, hq=heads[0], hkv=heads[1],
                             dim=dim, fp8=fp8))


def _scored(name, requests, lo, hi, new=1, window=32, add=True, heads=(24, 4), dim=256, fp8=False):
    return _named(name, dict(kind="scored", requests=requests, lo=lo, hi=hi, new=new,
                             window=window, add=add, hq=heads[0], hkv=heads[1], dim=dim, fp8=fp8))


def _evict(name, requests, lo, hi, keep, first=0, recent=64, prefixes=False):
    return _named(name, dict(kind="evict", requests=requests, lo=lo, hi=hi, keep=keep, first=first,
                             recent=recent, prefixes=prefixes))


def _named(name, case):
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # Three samples of one short prompt, a token each: latency.
        _shared("shared_samples", 1, 3, 300, 40, heads=(16, 2)),
        # Turns of four conversations' branches beside other requests, verify steps of up to 4 tokens.
        _shared("shared_turns", 4, 4, 4096, 2048, loose=5, new=4),
        # A decode batch behind one long system prompt.
        _shared("shared_system", 1, 64, 8192, 1024),
        # The same with narrower heads and a shorter prompt.
        _shared("shared_heads128", 1, 96, 2000, 700, heads=(32, 8), dim=128),
        # A large decode batch on a long document in an fp8 pool.
        _shared("shared_document", 1, 256, 32768, 2048, fp8=True),
        # One user's token.
        _scored("scored_one", 1, 900, 900),
        # A decode batch that adds up its weights.
        _scored("scored_decode", 64, 1024, 8192),
        # Long contexts of an fp8 pool, weights of the last token alone.
        _scored("scored_long", 8, 32768, 32768, add=False, fp8=True),
        # Prompts: the last 32 tokens say what the prompt's cache keeps.
        _scored("scored_prompt", 4, 2048, 10240, new=2048, add=False),
        # A few requests that outgrow a small budget.
        _evict("evict_few", 3, 1100, 1500, 1024, first=4),
        # A decode batch behind shared prefixes, which stay.
        _evict("evict_batch", 64, 2048, 8192, 2048, first=1000, prefixes=True),
        # Long prompts cut to an eighth.
        _evict("evict_long", 8, 131072, 131072, 16384, first=4, recent=1024),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    """(query heads, kv heads), head dim"""
    return rng.choice([((24, 4), 256), ((24, 4), 256), ((16, 2), 256), ((6, 1), 256),
                       ((32, 8), 128), ((8, 8), 64)])


def draw(rng):
    kind = rng.choice(["shared", "shared", "scored", "scored", "evict"])
    heads, dim = _heads(rng)
    fp8 = rng.random() < 0.3
    if kind == "shared":
        groups = rng.choice([1, 1, 2, 5])
        members = _log_int(rng, 2, 200 // groups)
        return _shared(None, groups, members, _log_int(rng, 100, 16384), _log_int(rng, 4, 2000),
                       loose=rng.choice([0, 0, 1, 7]), new=rng.choice([1, 1, 2, 6]), heads=heads,
                       dim=dim, fp8=fp8)
    if kind == "scored":
        if rng.random() < 0.3:
            new = _log_int(rng, 2, 1500)
            hi = new + _log_int(rng, 1, 6000)
            return _scored(None, rng.randint(1, 4), max(new, hi // 2), hi, new=new,
                           window=rng.choice([1, 16, 32, 57]), add=rng.random() < 0.5, heads=heads,
                           dim=dim, fp8=fp8)
        hi = _log_int(rng, 20, 16384)
        return _scored(None, _log_int(rng, 1, 48), 1 + hi // rng.choice([1, 2, 10]), hi,
                       add=rng.random() < 0.5, heads=heads, dim=dim, fp8=fp8)
    hi = _log_int(rng, 60, 60000)
    keep = _log_int(rng, 16, hi)
    first = rng.randint(0, keep // 2)
    return _evict(None, _log_int(rng, 1, 16), 1 + hi // 3, hi, keep, first=first,
                  recent=rng.randint(0, keep - first), prefixes=rng.random() < 0.5)


def _sizes(case):
    """The case's lengths: spread over its range, the same for every seed."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    if case["kind"] != "shared":
        return [rng.randint(case["lo"], case["hi"]) for _ in range(case["requests"])]
    several = case["groups"] > 1
    prefixes = [rng.randint(case["prefix"] // 4, case["prefix"]) if several else case["prefix"]
                for _ in range(case["groups"])]
    # (group or -1, tokens of its own, of them new) of every request, in a batch's order
    reqs = [(g, rng.randint(1, case["suffix"]), rng.randint(1, case["new"]))
            for g in list(range(case["groups"])) * case["members"] + [-1] * case["loose"]]
    rng.shuffle(reqs)
    return prefixes, [(g, max(n, e), e) for g, n, e in reqs]


def _pool(slots, hkv, dim, fp8, gen):
    x = torch.randn((slots, hkv, dim), generator=gen, device="cuda")
    if not fp8:
        return x.to(torch.bfloat16), None
    scale = (x.abs().amax() / E4M3_MAX).reshape(1)
    return (x / scale).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def _ints(values):
    return torch.tensor(values, dtype=torch.int64, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "evict":
        return _prepare_evict(case, gen)
    st = dict(case=case)
    prefixes, shared = [], []
    if case["kind"] == "shared":
        prefixes, reqs = _sizes(case)
        st["groups"] = [([b for b, r in enumerate(reqs) if r[0] == g], n)
                        for g, n in enumerate(prefixes)]
        lens = [n + (prefixes[g] if g >= 0 else 0) for g, n, _ in reqs]
        new = [e for _, _, e in reqs]
    else:
        reqs = [(-1, n, case["new"]) for n in _sizes(case)]
        lens, new = [n for _, n, _ in reqs], [e for _, _, e in reqs]
    total = sum(prefixes) + sum(n for _, n, _ in reqs)
    slots = total + total // 4 + 8
    perm = torch.randperm(slots - 1, generator=gen, device="cuda") + 1
    table = torch.full((2 * len(reqs), max(lens) + 16), -1, dtype=torch.int64, device="cuda")
    rows = torch.randperm(2 * len(reqs), generator=gen, device="cuda")[:len(reqs)]
    at = 0
    for n in prefixes:
        shared.append(perm[at:at + n])
        at += n
    for row, (g, n, _) in zip(rows.tolist(), reqs):
        p = len(shared[g]) if g >= 0 else 0
        if p:
            table[row, :p] = shared[g]
        table[row, p:p + n] = perm[at:at + n]
        at += n
    hkv, dim = case["hkv"], case["dim"]
    st["k"], st["k_scale"] = _pool(slots, hkv, dim, case["fp8"], gen)
    st["v"], st["v_scale"] = _pool(slots, hkv, dim, case["fp8"], gen)
    st["q"] = (1.5 * torch.randn((sum(new), case["hq"], dim), generator=gen,
                                 device="cuda")).to(torch.bfloat16)
    st.update(table=table, rows=rows, seq=_ints(lens), lens=lens, new=new, row_list=rows.tolist())
    if case["kind"] == "scored":
        # what earlier steps added up
        st["scores"] = torch.rand(table.shape, generator=gen, device="cuda").pow(8)
    if own:
        from tokenfactory_amd import ForwardBatch, SharedPrefixes
        starts = _ints([n - e for n, e in zip(lens, new)])
        st["batch"] = ForwardBatch(
            batch_size=len(lens), req_pool_indices=rows, seq_lens=st["seq"], prefix_lens=starts,
            extend_lens=new, out_cache_loc=_ints([0] * sum(new)), req_to_token=table,
            is_prefill=max(new) > 1, max_seq_len=max(lens))
        if case["kind"] == "shared":
            st["shared"] = SharedPrefixes(st["groups"])
    return st


def _prepare_evict(case, gen):
    lens = _sizes(case)
    n = len(lens)
    table = torch.full((2 * n, max(lens) + 16), -1, dtype=torch.int64, device="cuda")
    perm = torch.randperm(2 * n, generator=gen, device="cuda")
    for b, (row, length) in enumerate(zip(perm[:n].tolist(), lens)):
        table[row, :length] = torch.randperm(length, generator=gen, device="cuda") + 1 + b * length
    # A few tokens hold most of the weight; some were never looked at.
    scores = torch.randn(table.shape, generator=gen, device="cuda").mul_(2.5).exp_().mul_(1e-3)
    scores[scores < 2e-5] = 0.0
    first = case["first"]
    if case["prefixes"]:
        first = torch.randint(0, first + 1, (n,), generator=gen, device="cuda")
    # The full rows stay for the prefix cache; decoding goes on with the short ones.
    return dict(case=case, table=table, scores=scores, rows=perm[:n].contiguous(),
                out_rows=perm[n:].contiguous(), seq=_ints(lens), max_len=max(lens), first=first)


def run(st):
    kind = st["case"]["kind"]
    if kind == "shared":
        return _run_shared(st)
    return _run_scored(st) if kind == "scored" else _run_evict(st)


def _run_shared(st):
    if own:
        from tokenfactory_amd import shared_prefix_attention
        return shared_prefix_attention(st["q"], st["k"], st["v"], st["batch"], st["shared"],
                                       k_scale=st["k_scale"], v_scale=st["v_scale"])
    out = torch.empty_like(st["q"])
    starts = _starts(st["new"])
    loose = set(range(len(st["lens"])))
    for members, n in st["groups"]:
        loose -= set(members)
        tokens = [t for b in members for t in range(starts[b], starts[b] + st["new"][b])]
        rows = _by_kv_head(st, st["q"][_ints(tokens)])
        k, v = _keys(st, st["row_list"][members[0]], 0, n)
        shared = rows @ k.transpose(1, 2)          # every row sees the whole prefix
        own_parts, at = [], 0
        for b in members:
            width = st["new"][b] * st["case"]["hq"] // st["case"]["hkv"]
            ko, vo = _keys(st, st["row_list"][b], n, st["lens"][b])
            s = _causal(st, b, rows[:, at:at + width] @ ko.transpose(1, 2), n)
            own_parts.append((at, at + width, s, vo))
            at += width
        top = shared.amax(dim=2, keepdim=True)
        for lo, hi, s, _ in own_parts:
            top[:, lo:hi] = torch.maximum(top[:, lo:hi], s.amax(dim=2, keepdim=True))
        p = torch.exp(shared - top)
        norm, o = p.sum(dim=2, keepdim=True), p @ v
        for lo, hi, s, vo in own_parts:
            p = torch.exp(s - top[:, lo:hi])
            norm[:, lo:hi] += p.sum(dim=2, keepdim=True)
            o[:, lo:hi] += p @ vo
        out[_ints(tokens)] = _by_token(st, o / norm)
    for b in loose:
        out[starts[b]:starts[b] + st["new"][b]] = _request(st, b, starts[b])[0]
    return out


def _starts(new):
    at = [0]
    for e in new:
        at.append(at[-1] + e)
    return at


def _by_kv_head(st, q):
    """[tokens, Hq, D] -> fp32 [Hkv, tokens x group, D], scaled"""
    case = st["case"]
    group = case["hq"] // case["hkv"]
    q = q.float() * case["dim"] ** -0.5
    return q.view(-1, case["hkv"], group, case["dim"]).transpose(0, 1).reshape(
        case["hkv"], -1, case["dim"])


def _by_token(st, o):
    case = st["case"]
    group = case["hq"] // case["hkv"]
    o = o.view(case["hkv"], -1, group, case["dim"]).transpose(0, 1)
    return o.reshape(-1, case["hq"], case["dim"]).to(torch.bfloat16)


def _keys(st, row, lo, hi):
    """fp32 [Hkv, keys, D] of K and V"""
    slots = st["table"][row, lo:hi]
    k, v = st["k"][slots].float(), st["v"][slots].float()
    if st["case"]["fp8"]:
        k, v = k * st["k_scale"], v * st["v_scale"]
    return k.transpose(0, 1).contiguous(), v.transpose(0, 1).contiguous()


def _causal(st, b, s, first_key):
    """Masks what the request's new tokens do not see yet."""
    e = st["new"][b]
    if e == 1:
        return s
    group = st["case"]["hq"] // st["case"]["hkv"]
    token = torch.arange(e, device="cuda").repeat_interleave(group)
    key = torch.arange(first_key, first_key + s.shape[2], device="cuda")
    last = st["lens"][b] - e + token
    return s.masked_fill_(key[None, :] > last[:, None], -math.inf)


def _request(st, b, start):
    """(outputs, weights [Hkv, rows, keys]) of one request over all of its keys"""
    rows = _by_kv_head(st, st["q"][start:start + st["new"][b]])
    k, v = _keys(st, st["row_list"][b], 0, st["lens"][b])
    s = _causal(st, b, rows @ k.transpose(1, 2), 0)
    s = torch.exp(s - s.amax(dim=2, keepdim=True))
    s /= s.sum(dim=2, keepdim=True)
    return _by_token(st, s @ v), s


def _run_scored(st):
    case = st["case"]
    scores = st["scores"].clone() if case["add"] else st["scores"]
    if own:
        from tokenfactory_amd import scored_attention
        out = scored_attention(st["q"], st["k"], st["v"], st["batch"], scores,
                               window=case["window"], add=case["add"], k_scale=st["k_scale"],
                               v_scale=st["v_scale"])
        return out, scores
    out = torch.empty_like(st["q"])
    group = case["hq"] // case["hkv"]
    starts = _starts(st["new"])
    for b, length in enumerate(st["lens"]):
        out[starts[b]:starts[b] + st["new"][b]], p = _request(st, b, starts[b])
        weight = p[:, -group * min(case["window"], st["new"][b]):].sum(dim=(0, 1))
        row = st["row_list"][b]
        scores[row, :length] = scores[row, :length] + weight if case["add"] else weight
    return out, scores


def _run_evict(st):
    case = st["case"]
    if own:
        from tokenfactory_amd import evict_tokens
        lens, freed = evict_tokens(st["table"], st["scores"], st["rows"], st["seq"], case["keep"],
                                   max_seq_len=st["max_len"], first=st["first"],
                                   recent=case["recent"], out_rows=st["out_rows"])
        return lens, freed, st["table"], st["scores"]
    pos = torch.arange(st["max_len"], device="cuda")[None, :]
    n = st["seq"][:, None]
    first = st["first"][:, None] if case["prefixes"] else torch.full_like(n, case["first"])
    first = torch.minimum(first, n)
    last = torch.maximum(n - case["recent"], first)
    budget = torch.clamp(first + case["recent"], min=case["keep"])
    slots = st["table"][st["rows"], :st["max_len"]]
    weight = st["scores"][st["rows"], :st["max_len"]]
    # Kept whatever their weight, then by weight, the first of equal ones first.
    order = torch.where((pos < first) | (pos >= last), torch.full_like(weight, math.inf), weight)
    order = torch.where(pos < n, order, torch.full_like(weight, -math.inf))
    rank = torch.sort(order, dim=1, descending=True, stable=True)[1]
    kept = torch.zeros_like(pos < n).scatter_(1, rank, pos < torch.minimum(budget, n))
    lens = kept.sum(dim=1)
    front = torch.sort((~kept).to(torch.int8), dim=1, stable=True)[1]     # kept ones, in order
    there = pos < lens[:, None]
    new_slots = torch.where(there, slots.gather(1, front), torch.full_like(slots, -1))
    new_weight = torch.where(there, weight.gather(1, front), torch.zeros_like(weight))
    inside = (pos < n).expand_as(slots)
    for table, value in ((st["table"], new_slots), (st["scores"], new_weight)):
        rows = table[st["out_rows"], :st["max_len"]]
        table[st["out_rows"], :st["max_len"]] = torch.where(inside, value, rows)
    gone = (pos < n) & ~kept
    back = torch.sort((~gone).to(torch.int8), dim=1, stable=True)[1]
    freed = torch.where(pos < gone.sum(dim=1, keepdim=True), slots.gather(1, back),
                        torch.full_like(slots, -1))
    return lens, freed[:, :max(0, st["max_len"] - case["keep"])], st["table"], st["scores"]


def work(case):
    """Keys and values of a shared prefix, and of every request's own tokens, read once;
    with weights, a score per cached token written (and read where it is added to)."""
    if case["kind"] == "evict":
        lens = _sizes(case)
        gone = sum(max(0, n - case["keep"]) for n in lens)
        return {"bytes": sum(lens) * (12 + 12) + 8 * gone, "flops": 0}
    per_key = 2 * case["hkv"] * case["dim"] * (1 if case["fp8"] else 2)
    per_pair = 4 * case["hq"] * case["dim"]
    if case["kind"] == "shared":
        prefixes, reqs = _sizes(case)
        tokens = sum(e for _, _, e in reqs)
        keys = sum(prefixes) + sum(n for _, n, _ in reqs)
        pairs = sum(e * ((prefixes[g] if g >= 0 else 0) + n) - e * (e - 1) // 2
                    for g, n, e in reqs)
        return {"bytes": keys * (per_key + 8) + 4 * tokens * case["hq"] * case["dim"],
                "flops": per_pair * pairs}
    lens, e = _sizes(case), case["new"]
    pairs = sum(e * n - e * (e - 1) // 2 for n in lens)
    return {"bytes": sum(lens) * (per_key + 8 + (8 if case["add"] else 4))
            + 4 * len(lens) * e * case["hq"] * case["dim"], "flops": per_pair * pairs}


# The operators in 64 bits.

def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "evict":
        return _exact_evict(st)
    out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    scores = st["scores"].double() if case["kind"] == "scored" else None
    group, at = case["hq"] // case["hkv"], 0
    ks = st["k_scale"].double() if case["fp8"] else 1.0
    vs = st["v_scale"].double() if case["fp8"] else 1.0
    for row, length, e in zip(st["row_list"], st["lens"], st["new"]):
        slots = st["table"][row, :length]
        weight = torch.zeros((length,), dtype=torch.float64, device="cuda")
        seen = torch.arange(length, device="cuda") <= torch.arange(length - e, length,
                                                                   device="cuda")[:, None]
        for h in range(case["hkv"]):
            k, v = st["k"][slots, h].double() * ks, st["v"][slots, h].double() * vs
            for i in range(h * group, (h + 1) * group):
                s = torch.mm(st["q"][at:at + e, i].double(), k.t()) / math.sqrt(case["dim"])
                p = torch.softmax(torch.where(seen, s, -math.inf), dim=1)
                out[at:at + e, i] = torch.mm(p, v)
                if scores is not None:
                    weight += p[-case["window"]:].sum(dim=0)
        if scores is not None:
            scores[row, :length] = weight + (scores[row, :length] if case["add"] else 0.0)
        at += e
    return out if scores is None else (out, scores)


def _exact_evict(st):
    """Row by row on the host: whole numbers, and scores that are moved."""
    case = st["case"]
    table, scores = st["table"].cpu(), st["scores"].cpu()
    width = max(0, st["max_len"] - case["keep"])
    lens, freed = [], torch.full((len(st["rows"]), width), -1, dtype=torch.int64)
    for b, (row, to, n) in enumerate(zip(st["rows"].tolist(), st["out_rows"].tolist(),
                                         st["seq"].tolist())):
        first = min(n, int(st["first"][b]) if case["prefixes"] else case["first"])
        end = max(first, n - case["recent"])
        room = max(case["keep"], first + case["recent"]) - first - (n - end)
        values = scores[row, first:end].tolist()
        best = sorted(range(len(values)), key=lambda i: (-values[i], i))[:max(0, room)]
        stay = list(range(first)) + sorted(first + i for i in best) + list(range(end, n))
        out = sorted(set(range(n)) - set(stay))
        freed[b, :len(out)] = table[row, out]
        slots, weight = table[row, stay].clone(), scores[row, stay].clone()
        table[to, :n], scores[to, :n] = -1, 0.0
        table[to, :len(stay)], scores[to, :len(stay)] = slots, weight
        lens.append(len(stay))
    dev = st["table"].device
    return _ints(lens), freed.to(dev), table.to(dev), scores.double().to(dev)
