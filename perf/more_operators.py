"""Operators of serving from a paged cache whose requests share a prompt's start and whose keys are dropped by their attention weight, as cases
timed one by one.

  * "shared":  attention of a step's new tokens where groups of requests have their first keys in common, read once for all of a group
               (ops.shared_prefix_attention): single tokens or a few of each request, and with key weights accumulated in the same call;
  * "observe": attention weight of every cached key under a prompt's last queries (ops.paged_key_weights);
  * "evict":   the heaviest keys of every kv head moved to the front of a request's pages, the others dropped (ops.paged_evict).

Head shapes are those of perf/cases.py: 32 / 8 and 28 / 4 heads of 128 channels, 32 / 8 and 14 / 2 of 64.  Pools bf16, weights fp32.
With `own` false the operators are computed by elementary torch operations in 32 bits, rounded once at the end.
"""

import math
import random

import torch

own = False

HEADS = ((32, 8, 128), (28, 4, 128), (32, 8, 64), (14, 2, 64))


def _heads(i):
    hq, hkv, d = HEADS[i]
    return {"hq": hq, "hkv": hkv, "d": d}


def _shared(name, page, groups, members, prefix, own_len, new=1, weigh=False, alone=0, heads=0):
    """`groups` groups of `members` requests with `prefix` keys in common, up to own_len keys of their own and `new` new tokens each (of the first
    request of a group; 1 to `new` of the others), and `alone` requests that share nothing."""
    return {"name": name, "op": "shared", "page": page, "groups": groups, "members": members, "prefix": prefix, "own_len": own_len, "new": new,
            "weigh": weigh, "alone": alone, **_heads(heads)}


def _observe(name, page, batch, length, queries, accumulate=False, first=0, heads=0):
    return {"name": name, "op": "observe", "page": page, "batch": batch, "length": length, "queries": queries, "accumulate": accumulate,
            "first": first, **_heads(heads)}


def _evict(name, page, batch, length, budget, recent, first=0, heads=0):
    return {"name": name, "op": "evict", "page": page, "batch": batch, "length": length, "budget": budget, "recent": recent, "first": first,
            **_heads(heads)}


def listed():
    return [
        # eight chats under a system prompt, the next token of each: latency
        _shared("shared_8x1k", 16, 1, 8, 1024, 200),
        # a serving batch over one long instruction, ragged answers
        _shared("shared_64x8k", 64, 1, 64, 8192, 2000),
        # four documents, sixteen questions about each and three requests about none, key weights kept; groups of seven heads
        _shared("shared_4x16_weighed", 16, 4, 16, 4000, 701, weigh=True, alone=3, heads=1),
        # drafted tokens of thirty-two requests checked over a shared document, a small model's heads
        _shared("shared_verify_32", 32, 1, 32, 16001, 1000, new=5, heads=2),
        # many short answers about one long document
        _shared("shared_128x32k", 128, 1, 128, 32768, 600),
        # chats that share nothing and have their keys weighed at every token
        _shared("weighed_16x4k", 64, 0, 0, 0, 4001, weigh=True, alone=16),
        # the last queries of one short prompt
        _observe("observe_16_of_1k", 16, 1, 1025, 16),
        # the last queries of a long prompt
        _observe("observe_32_of_32k", 64, 1, 32768, 32, heads=1),
        # ragged prompts behind a shared start, on top of what earlier queries gave
        _observe("observe_8x64_of_8k", 32, 8, 8001, 64, accumulate=True, first=512, heads=2),
        # a short cache made shorter
        _evict("evict_1x2k", 16, 1, 2000, 256, 64),
        # a ragged batch, groups of seven heads
        _evict("evict_16x8k", 64, 16, 8001, 1900, 100, first=64, heads=1),
        # a long document cut to a sixteenth
        _evict("evict_128k", 128, 1, 131072, 8000, 192),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("shared", "shared", "shared", "observe", "evict"))
    page = rng.choice((16, 32, 64, 128, 256))
    heads = rng.randrange(4)
    if op == "shared":
        groups = rng.choice((0, 1, 1, 1, 2, 3, 5))
        members = _log_int(rng, 2, 96 // groups) if groups else 0
        alone = _log_int(rng, 1, 32) if not groups else rng.choice((0, 0, 1, 5))
        new = rng.choice((1, 1, 1, 2, 4, 9))
        prefix = _log_int(rng, 16, min(32768 // groups, (1 << 22) // (groups * members * new))) if groups else 0
        weigh = new == 1 and (rng.random() < 0.5 or not groups)
        own_len = max(_log_int(rng, 10, 60000 // max(groups * members + alone, 8)), new)
        c = _shared("", page, groups, members, prefix, own_len, new, weigh, alone, heads)
    elif op == "observe":
        batch = rng.choice((1, 1, 2, 4, 8))
        length = _log_int(rng, 20, 65536 // batch)
        queries = min(_log_int(rng, 1, 64), length)
        c = _observe("", page, batch, length, queries, rng.random() < 0.5, rng.choice((0, 0, rng.randrange(1, 600))), heads)
    else:
        batch = _log_int(rng, 1, 32)
        length = _log_int(rng, 30, 131072 // batch)
        c = _evict("", page, batch, length, _log_int(rng, 4, max(length // 2, 5)), rng.randrange(0, 200), rng.choice((0, 4, rng.randrange(0, 300))), heads)
    del c["name"]
    return c


# ---- sizes that a case's seedless description leaves open: they are the same whatever the inputs ----------------------------
def _ceil(a, b):
    return -(-a // b)


def _requests(case):
    """-> (lens, new, prefix of every request, [first request, one past the last] of every group): by the case alone."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    if case["op"] != "shared":
        n = case["length"]
        lens = [n if i == 0 else rng.randrange(max(n // 4, 1), n + 1) for i in range(case["batch"])]
        q = case.get("queries", 0)
        new = [min(q, lens[i]) if i == 0 else rng.randrange(1, min(q, lens[i]) + 1) for i in range(case["batch"])] if q else [0] * case["batch"]
        return lens, new, [0] * case["batch"], []
    lens, new, prefix, spans = [], [], [], []

    def one(shared, first):
        t = case["new"] if first else rng.randrange(1, case["new"] + 1)
        n = case["own_len"] if first else rng.randrange(max(case["own_len"] // 4, 1), case["own_len"] + 1)
        new.append(t)
        lens.append(shared + max(n, t))
        prefix.append(shared)

    for g in range(case["groups"]):
        shared = case["prefix"] if g == 0 else rng.randrange(max(case["prefix"] // 2, 1), case["prefix"] + 1)
        spans.append((len(lens), len(lens) + case["members"]))
        for i in range(case["members"]):
            one(shared, i == 0)
    for i in range(case["alone"]):
        one(0, i == 0)
    return lens, new, prefix, spans


# ---- inputs -----------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).to(torch.bfloat16)
    ints = lambda values: torch.tensor(values, dtype=torch.int32, device=dev)
    page, hq, hkv, d = case["page"], case["hq"], case["hkv"], case["d"]
    lens, new, prefix, spans = _requests(case)
    width = max(_ceil(n, page) for n in lens)
    # pages in any order; those that hold nothing but shared keys are named by every request of a group
    need, rows = 0, []
    holder = {b: first for first, end in spans for b in range(first, end)}
    for b, n in enumerate(lens):
        first = holder.get(b, b)
        whole = prefix[b] // page if first != b else 0
        rows.append((rows[first][:whole] if whole else []) + list(range(need, need + _ceil(n, page) - whole)))
        need += _ceil(n, page) - whole
    order = torch.randperm(need + 7, generator=gen, device=dev).to(torch.int32)
    places = torch.tensor([r + [need] * (width - len(r)) for r in rows], dtype=torch.int64, device=dev)
    table = torch.where(places < need, order[places], torch.full((), -1, dtype=torch.int32, device=dev)).contiguous()
    k, v = (rand(need + 7, hkv, page, d) for _ in range(2))
    for first, end in spans:  # a page that holds the last shared keys and some of a request's own: everyone has a copy
        part, at = prefix[first] % page, prefix[first] // page
        if part:
            ids = table[first:end, at].long()
            for pool in (k, v):
                pool[ids, :, :part] = pool[ids[:1], :, :part]
    state = {"case": case, "k": k, "v": v, "table": table, "lens": ints(lens), "scale": d ** -0.5, "host": (lens, new, prefix, spans)}
    # what softmax weights summed over many queries look like: a few heavy keys, many light ones, some that have vanished
    heavy = torch.exp(2.0 * torch.randn(need + 7, hkv, page, generator=gen, device=dev)) * 0.01
    heavy[torch.rand(need + 7, hkv, page, generator=gen, device=dev) < 0.01] = 0.0
    if case["op"] == "evict":
        state["weights"], state["first"] = heavy, ints([min(case["first"], n) for n in lens])
        return state
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    state["q"] = rand(starts[-1], hq, d).transpose(0, 1)  # as a model's projections leave it, token by token
    if case["op"] == "observe":
        state["weights"], state["cu"] = heavy, ints(starts)
        state["first"] = ints([min(case["first"], n) for n in lens]) if case["first"] else None
        return state
    state["cu"] = ints(starts) if case["new"] > 1 else None
    state["weights"] = heavy if case["weigh"] else None
    state["groups"] = ints([s[0] for s in spans] + [spans[-1][1] if spans else 0])
    state["prefix"] = ints([prefix[s[0]] for s in spans])
    return state


# ---- one pass ---------------------------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    from shareprefill_amd import ops

    case = state["case"]
    if case["op"] == "evict":
        lens = ops.paged_evict(state["k"], state["v"], state["weights"], state["table"], state["lens"], case["budget"], case["recent"],
                               first=state["first"])
        return state["k"], state["v"], state["weights"], lens
    if case["op"] == "observe":
        return ops.paged_key_weights(state["q"], state["k"], state["table"], state["lens"], state["scale"], state["weights"], cu_q=state["cu"],
                                     first=state["first"], accumulate=case["accumulate"])
    out = ops.shared_prefix_attention(state["q"], state["k"], state["v"], state["table"], state["lens"], state["prefix"], state["groups"],
                                      state["scale"], cu_q=state["cu"], weights=state["weights"])
    return (out, state["weights"]) if case["weigh"] else out


def _scores(q, k, scale, first):
    """q [Hq, n, D], the last of which is at position first + n - 1, over k [Hkv, len, D] -> masked fp32 logits [Hkv, g n, len]"""
    hq, n, d = q.shape
    hkv, total, _ = k.shape
    s = torch.matmul(q.float().reshape(hkv, hq // hkv * n, d), k.float().transpose(1, 2).contiguous()) * scale
    if first + 1 < total:  # some query does not see all keys
        hidden = torch.arange(total, device=q.device)[None, :] > torch.arange(first, first + n, device=q.device)[:, None]
        s.view(hkv, hq // hkv, n, total).masked_fill_(hidden, -math.inf)
    return s


def _cached(pool, ids, lo, hi, page):
    """rows lo .. hi of a request, [Hkv, hi - lo, D]"""
    p0 = lo // page
    x = pool[ids[p0:_ceil(hi, page)].long()].transpose(0, 1)
    return x.reshape(x.shape[0], -1, x.shape[3])[:, lo - p0 * page:hi - p0 * page]


def _run_plain(state):
    case = state["case"]
    if case["op"] == "evict":
        return _evict_plain(state)
    q, table, page, scale = state["q"], state["table"], case["page"], state["scale"]
    lens, new, prefix, spans = state["host"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    g = hq // hkv
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    if case["op"] == "observe":
        weights = state["weights"]
        for b, (total, n) in enumerate(zip(lens, new)):
            k = _cached(state["k"], table[b], 0, total, page)
            s = _scores(q[:, starts[b]:starts[b + 1]], k, scale, total - n)
            e = torch.exp(s - s.amax(-1, keepdim=True))
            w = (e / e.sum(-1, keepdim=True)).sum(1)
            lo = min(case["first"], total)
            j = torch.arange(lo, total, device=q.device)
            ids, at = table[b].long()[j // page], j % page
            w = w[:, lo:].t()
            if case["accumulate"]:
                w = w + torch.where((j < total - n)[:, None], weights[ids, :, at], torch.zeros_like(w))
            weights[ids, :, at] = w
        return weights
    out = torch.empty(starts[-1], hq, d, dtype=torch.bfloat16, device=q.device)
    weights = state["weights"]
    groups = list(spans) + [(b, b + 1) for b in range(len(lens)) if prefix[b] == 0]
    for first, end in groups:
        shared, t0, t1 = prefix[first], starts[first], starts[end]
        if shared:
            kp, vp = (_cached(pool, table[first], 0, shared, page) for pool in (state["k"], state["v"]))
            sp = _scores(q[:, t0:t1], kp, scale, shared).view(hkv, g, t1 - t0, shared)
            vp = vp.float()
        for b in range(first, end):
            total, n, r0 = lens[b], new[b], starts[b] - t0
            ko, vo = (_cached(pool, table[b], shared, total, page) for pool in (state["k"], state["v"]))
            s = _scores(q[:, starts[b]:starts[b + 1]], ko, scale, total - n - shared)
            top = s.amax(-1, keepdim=True)
            if shared:
                mine = sp[:, :, r0:r0 + n].reshape(hkv, g * n, shared)
                top = torch.maximum(top, mine.amax(-1, keepdim=True))
            e = torch.exp(s - top)
            total_e, o = e.sum(-1, keepdim=True), torch.matmul(e, vo.float())
            if shared:
                ep = torch.exp(mine - top)
                total_e, o = total_e + ep.sum(-1, keepdim=True), o + torch.matmul(ep, vp)
            out[starts[b]:starts[b + 1]] = (o / total_e).view(hq, n, d).transpose(0, 1).to(torch.bfloat16)
            if weights is not None:
                w = (e / total_e).sum(1).t()
                j = torch.arange(shared, total, device=q.device)
                ids, at = table[b].long()[j // page], j % page
                weights[ids, :, at] = w + torch.where((j < total - 1)[:, None], weights[ids, :, at], torch.zeros_like(w))
    return (out, weights) if case["weigh"] else out


def _evict_plain(state):
    case, k, v, weights, table = state["case"], state["k"], state["v"], state["weights"], state["table"]
    page, hkv, recent, budget = case["page"], case["hkv"], case["recent"], case["budget"]
    lens = state["host"][0]
    heads = torch.arange(hkv, device=table.device)[:, None]
    out = []
    for b, total in enumerate(lens):
        first = min(case["first"], total)
        mid = max(total - recent - first, 0)
        keep = min(mid, budget)
        if keep < mid:
            j = torch.arange(first, total, device=table.device)
            ids, at = table[b].long()[j // page], j % page
            w = weights[ids, :, at].t()  # [Hkv, len - first]
            chosen = torch.sort(w[:, :mid], dim=1, descending=True, stable=True).indices[:, :keep].sort(dim=1).values
            src = torch.cat((chosen, torch.arange(mid, total - first, device=table.device).expand(hkv, -1)), 1)
            n = src.shape[1]
            to = (ids[:n], at[:n])
            moved = [x[ids[src], heads, at[src]] for x in (k, v, weights)]  # [Hkv, n, ...]
            for x, m in zip((k, v, weights), moved):
                x[to[0], :, to[1]] = m.transpose(0, 1)
        out.append(total - mid + keep)
    return k, v, weights, torch.tensor(out, dtype=torch.int32, device=table.device)


# ---- what a pass cannot do without --------------------------------------------------------------------------------
def work(case):
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    lens, new, prefix, spans = _requests(case)
    moved = flops = 0.0
    if case["op"] == "evict":
        for total in lens:
            first = min(case["first"], total)
            mid = max(total - case["recent"] - first, 0)
            keep = min(mid, case["budget"])
            if keep < mid:
                # the weights of what may go, and every kept key's row, value and weight read and written
                moved += hkv * (4.0 * mid + 2.0 * (total - first - mid + keep) * (4.0 * d + 4.0))
        return {"bytes": moved + 8.0 * len(lens), "flops": 0.0}
    for total, n, shared in zip(lens, new, prefix):
        own_keys = total - shared
        pairs = n * total - n * (n - 1) // 2
        if case["op"] == "observe":
            moved += 2.0 * d * (n * hq + total * hkv) + 4.0 * hkv * (total - min(case["first"], total)) * (2 if case["accumulate"] else 1)
            flops += 2.0 * d * hq * pairs
            continue
        moved += 2.0 * d * (2 * n * hq + 2 * own_keys * hkv) + (8.0 * hkv * own_keys if case["weigh"] else 0.0) + 4.0 * _ceil(total, page)
        flops += 4.0 * d * hq * pairs
    for first, _ in spans:
        moved += 4.0 * d * hkv * prefix[first]
    return {"bytes": moved, "flops": flops}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    lens, new, prefix, _ = state["host"]
    page, hkv, d = case["page"], case["hkv"], case["d"]
    g = case["hq"] // hkv
    table = state["table"].long()
    if case["op"] == "evict":
        return _evict_exact(state)
    out = torch.empty(sum(new), case["hq"], d, dtype=torch.float64, device=table.device)
    weights = state["weights"].double() if state["weights"] is not None else None
    at = 0
    for b, (total, n) in enumerate(zip(lens, new)):
        j = torch.arange(total, device=table.device)
        pages, rows = table[b][j // page], j % page
        hidden = j[None, :] > torch.arange(total - n, total, device=table.device)[:, None]
        sums = torch.empty(hkv, total, dtype=torch.float64, device=table.device)
        for h in range(hkv):
            keys = state["k"][pages, h, rows].double()
            queries = state["q"][h * g:(h + 1) * g, at:at + n].double()
            logits = (queries.reshape(g * n, d) @ keys.t().contiguous()).mul_(state["scale"]).view(g, n, total).masked_fill_(hidden, -math.inf)
            p = torch.softmax(logits, -1).view(g * n, total)
            sums[h] = p.sum(0)
            if case["op"] == "shared":
                out[at:at + n, h * g:(h + 1) * g] = (p @ state["v"][pages, h, rows].double()).view(g, n, d).transpose(0, 1)
        if weights is not None:
            # a key of a new token starts from nothing, and so does every key unless earlier sums are to be kept
            keep_from = prefix[b] if case["op"] == "shared" else min(case["first"], total)
            adds = case["op"] == "shared" or case["accumulate"]
            old = weights[pages, :, rows].t() * (j < total - n if adds else torch.zeros_like(j, dtype=torch.bool))
            live = j >= keep_from
            weights[pages[live], :, rows[live]] = (sums + old).t()[live]
        at += n
    if case["op"] == "observe":
        return weights
    return (out, weights) if case["weigh"] else out


def _evict_exact(state):
    case, table = state["case"], state["table"].tolist()
    page, hkv = case["page"], case["hkv"]
    pools = [state[x].cpu() for x in ("k", "v", "weights")]
    before = [x.clone() for x in pools]
    w = before[2].numpy()
    new_lens = []
    for b, total in enumerate(state["host"][0]):
        first = min(case["first"], total)
        mid = list(range(first, max(total - case["recent"], first)))
        kept = min(len(mid), case["budget"])
        new_lens.append(total - len(mid) + kept)
        if kept == len(mid):
            continue
        places = torch.tensor([table[b][j // page] * page + j % page for j in range(total)])
        for h in range(hkv):
            flat = w[:, h].reshape(-1)
            weight = flat[places[first:first + len(mid)].numpy()].tolist()
            heaviest = sorted(range(len(mid)), key=lambda i: (-weight[i], i))[:kept]
            src = sorted(heaviest) + list(range(len(mid), total - first))
            to, come = places[first:first + len(src)], places[[first + i for i in src]]
            for pool, old in zip(pools, before):
                pool[to // page, h, to % page] = old[come // page, h, come % page]
    dev = state["table"].device
    return (*(x.to(torch.float64).to(dev) for x in pools), torch.tensor(new_lens, dtype=torch.int32, device=dev))
