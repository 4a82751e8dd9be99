"""The operators of serving from a paged key / value cache, and attention with a sliding window, as cases timed one by one.

  * "tables": block tables, slots and positions of a step's new tokens, from the requests' lengths (ops.page_tables);
  * "write":  a step's new keys and values into their pages (ops.paged_cache_write);
  * "paged":  attention of the new tokens of a batch of requests over everything cached (ops.paged_attention): prompts in
              chunks, single tokens, and batches of both, with a window and sinks or without;
  * "window": the same mask over contiguous keys and values (ops.window_attention): whole prompts and single tokens.

Head shapes are those of perf/cases.py: 32 / 8 and 28 / 4 heads of 128 channels, 32 / 8 and 14 / 2 of 64.  bf16.
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


def _tables(name, batch, cached, new, page):
    return {"name": name, "op": "tables", "batch": batch, "cached": cached, "new": new, "page": page}


def _write(name, tokens, page, heads=0, token_major=True):
    return {"name": name, "op": "write", "tokens": tokens, "page": page, "token_major": token_major, **_heads(heads)}


def _paged(name, page, singles, single_len, chunks, chunk, chunk_len, heads=0, window=0, sinks=0):
    """`singles` requests with one new token each and up to single_len keys, `chunks` with `chunk` new tokens and chunk_len keys."""
    return {"name": name, "op": "paged", "page": page, "singles": singles, "single_len": single_len, "chunks": chunks, "chunk": chunk,
            "chunk_len": chunk_len, "window": window, "sinks": sinks, **_heads(heads)}


def _window(name, batch, n, nk, window, sinks, heads=0):
    return {"name": name, "op": "window", "batch": batch, "n": n, "nk": nk, "window": window, "sinks": sinks, **_heads(heads)}


def listed():
    return [
        # a decode step of eight chats: one new token each, now and then a page
        _tables("tables_8_chats", 8, 1500, 1, 16),
        # a step of a full server: many requests, most with one token, some with a chunk of their prompt
        _tables("tables_256_mixed", 256, 4000, 512, 16),
        # the new keys and values of a decode step
        _write("write_8", 8, 16),
        # those of a large chunk
        _write("write_16k", 16384, 64),
        # one chat, the next token: latency
        _paged("paged_token_1x1k", 16, 1, 1025, 0, 0, 0),
        # a serving batch of ragged caches, groups of seven heads
        _paged("paged_tokens_64x8k", 64, 64, 8001, 0, 0, 0, heads=1),
        # a chunk of a prompt over what is cached of it
        _paged("paged_chunk_512_of_8k", 16, 0, 0, 1, 512, 8192),
        # chunks of two prompts beside the next tokens of thirty chats, a small model's heads
        _paged("paged_mixed_32", 32, 30, 3001, 2, 999, 5000, heads=2),
        # a large chunk of a long document
        _paged("paged_chunk_2k_of_64k", 128, 0, 0, 1, 2048, 65001),
        # a prompt in a sliding window with the first tokens kept
        _window("window_8k", 1, 8192, 8192, 1024, 4, heads=1),
        # a long prompt, ragged, a wide window
        _window("window_30k_wide", 1, 30001, 30001, 4096, 64),
        # the next tokens of eight long chats in a window
        _window("window_tokens_8x32k", 8, 1, 32768, 4096, 4),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("tables", "write", "paged", "paged", "paged", "window", "window"))
    page = rng.choice((16, 32, 64, 128, 256))
    heads = rng.randrange(4)
    if op == "tables":
        return {k: v for k, v in _tables("", _log_int(rng, 1, 1024), _log_int(rng, 1, 20000), _log_int(rng, 1, 512), page).items() if k != "name"}
    if op == "write":
        c = _write("", _log_int(rng, 1, 16384), page, heads, rng.random() < 0.5)
    elif op == "paged":
        window = rng.choice((0, 0, _log_int(rng, 1, 8192)))
        sinks = rng.choice((0, 4, rng.randrange(1, 200))) if window else 0
        kind = rng.choice(("singles", "chunks", "both"))
        singles = chunks = 0
        single_len = chunk = chunk_len = 0
        if kind != "chunks":
            singles = _log_int(rng, 1, 128)
            single_len = _log_int(rng, 1, 500000 // singles if kind == "singles" else 8000)
            single_len = min(single_len, 131072)
        if kind != "singles":
            chunks = rng.choice((1, 1, 2, 3, 5))
            chunk_len = _log_int(rng, 10, 60000 if chunks == 1 else 12000)
            chunk = min(_log_int(rng, 2, 2048 if chunks == 1 else 1024), chunk_len)
        c = _paged("", page, singles, single_len, chunks, chunk, chunk_len, heads, window, sinks)
    else:
        window, sinks = _log_int(rng, 16, 8192), rng.choice((0, 4, rng.randrange(1, 200)))
        if rng.random() < 0.4:
            batch = _log_int(rng, 1, 32)
            c = _window("", batch, 1, _log_int(rng, 1, 400000 // batch), window, sinks, heads)
        else:
            batch = rng.choice((1, 1, 2, 3))
            nk = _log_int(rng, 2, 30000 // batch)
            n = nk if rng.random() < 0.7 else rng.randrange(1, nk + 1)
            c = _window("", batch, n, nk, window, sinks, heads)
    del c["name"]
    return c


# ---- sizes that a case's seedless description leaves open: they are the same whatever the inputs ----------------------------
def _lengths(case):
    """-> (cached, new) per request, ragged: by the case alone, since the work has to be known without the inputs."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    if case["op"] == "tables":
        # half the requests or so are chats with one new token, some stand still, the others bring a part of their prompt
        cached = [rng.randrange(0, case["cached"] + 1) for _ in range(case["batch"])]
        new = [rng.choice((0, 1, 1, 1, 1, rng.randrange(1, case["new"] + 1))) if case["new"] > 1 else 1 for _ in range(case["batch"])]
        return cached, new
    cached, new = [], []
    for i in range(case["singles"]):
        n = case["single_len"] if i == 0 else rng.randrange(case["single_len"] // 4, case["single_len"] + 1)
        cached.append(max(n, 1) - 1)
        new.append(1)
    for i in range(case["chunks"]):
        n = case["chunk"] if i == 0 else rng.randrange(1, case["chunk"] + 1)
        total = case["chunk_len"] if i == 0 else rng.randrange(n, case["chunk_len"] + 1)
        cached.append(total - n)
        new.append(n)
    order = list(range(len(new)))
    rng.shuffle(order)
    return [cached[i] for i in order], [new[i] for i in order]


def _ceil(a, b):
    return -(-a // b)


# ---- inputs -----------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).to(torch.bfloat16)
    ints = lambda values: torch.tensor(values, dtype=torch.int32, device=dev)
    page = case.get("page")
    if case["op"] == "tables":
        cached, new = _lengths(case)
        width = max(_ceil(c + n, page) for c, n in zip(cached, new)) + 1
        used = sum(_ceil(c, page) for c in cached)
        total = used + sum(new) + 5
        pages = torch.randperm(total, generator=gen, device=dev).to(torch.int32)  # a cache that has been in use: pages in any order
        have = ints([_ceil(c, page) for c in cached])
        table = torch.full((case["batch"], width), -1, dtype=torch.int32, device=dev)
        table[torch.arange(width, device=dev)[None, :] < have[:, None]] = pages[:used]
        return {"case": case, "lens": ints(cached), "new": ints(new), "table": table, "free": pages[used:].contiguous(),
                "free_count": ints([total - used]), "pages": total, "tokens": max(sum(new), 1)}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "write":
        n = case["tokens"]
        pages = _ceil(n, page) + 3
        slots = torch.randperm(pages * page, generator=gen, device=dev)[:n]
        if n > 8:
            slots[n - 3:] = -1  # the end of a padded step
        kv = [rand(n, hkv, d).transpose(0, 1) if case["token_major"] else rand(hkv, n, d) for _ in range(2)]
        pools = [torch.zeros(pages, hkv, page, d, dtype=torch.bfloat16, device=dev) for _ in range(2)]
        return {"case": case, "kv": kv, "pools": pools, "slots": slots}
    if case["op"] == "window":
        b, n, nk = case["batch"], case["n"], case["nk"]
        # as a model's projections leave them, token by token; a cache is kept head by head
        q = rand(b, n, hq, d).transpose(1, 2)
        k, v = (rand(b, hkv, nk, d) if n < nk else rand(b, nk, hkv, d).transpose(1, 2) for _ in range(2))
        return {"case": case, "q": q, "k": k, "v": v, "scale": d ** -0.5}
    cached, new = _lengths(case)
    lens = [c + n for c, n in zip(cached, new)]
    width = max(_ceil(n, page) for n in lens)
    need = sum(_ceil(n, page) for n in lens)
    order = torch.randperm(need + 7, generator=gen, device=dev).to(torch.int32)
    have = ints([_ceil(n, page) for n in lens])
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=dev)
    table[torch.arange(width, device=dev)[None, :] < have[:, None]] = order[:need]
    pools = [rand(need + 7, hkv, page, d) for _ in range(2)]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = rand(starts[-1], hq, d).transpose(0, 1)
    return {"case": case, "q": q, "k": pools[0], "v": pools[1], "table": table, "lens": ints(lens), "scale": d ** -0.5,
            "cu": ints(starts) if case["chunks"] else None, "host": (lens, new)}


# ---- one pass ---------------------------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    from shareprefill_amd import ops

    case = state["case"]
    if case["op"] == "tables":
        t = ops.page_tables(state["lens"], state["new"], state["table"], state["free"], state["free_count"], case["page"], state["pages"],
                            state["tokens"])
        return state["table"], t.seq_lens, t.cu_new, t.slots, t.positions, t.free_left
    if case["op"] == "write":
        ops.paged_cache_write(*state["kv"], *state["pools"], state["slots"])
        return state["pools"]
    if case["op"] == "window":
        return ops.window_attention(state["q"], state["k"], state["v"], state["scale"], window=case["window"], sinks=case["sinks"])
    return ops.paged_attention(state["q"], state["k"], state["v"], state["table"], state["lens"], state["scale"], cu_q=state["cu"],
                               window=case["window"] or None, sinks=case["sinks"])


def _softmax_rows(scores, seen):
    """softmax over the last axis of what is seen; rows that see nothing are zero"""
    scores = torch.where(seen, scores, torch.full_like(scores, -math.inf))
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _attend_plain(q, k, v, scale, first, window, sinks):
    """q [Hq, n, D] at positions first .. first + n - 1 over k, v [Hkv, len, D] -> fp32 [n, Hq, D]"""
    hq, n, d = q.shape
    hkv, total, _ = k.shape
    g = hq // hkv
    out = torch.empty(n, hq, d, dtype=torch.float32, device=q.device)
    rows = max(1, min(n, (1 << 31) // (hq * max(min(total, window + 1024 if window else total), 1))))
    rows = min(rows, 1024) if window else rows
    for r0 in range(0, n, rows):
        r1 = min(n, r0 + rows)
        lo, hi = 0, min(total, first + r1)
        if window:
            lo = max(0, first + r0 - window + 1)
        s = min(sinks, lo)
        keys = torch.cat((torch.arange(s, device=q.device), torch.arange(lo, max(hi, lo), device=q.device)))
        if keys.numel() == 0:
            out[r0:r1] = 0
            continue
        pick = (lambda x: x[:, lo:hi].float()) if s == 0 else (lambda x: torch.cat((x[:, :s], x[:, lo:hi]), 1).float())
        kf, vf = pick(k), pick(v)
        qf = q[:, r0:r1].float().reshape(hkv, g * (r1 - r0), d)
        scores = torch.matmul(qf, kf.transpose(1, 2).contiguous()).view(hkv, g, r1 - r0, -1) * scale
        pos = torch.arange(first + r0, first + r1, device=q.device)[:, None]
        seen = keys[None, :] <= pos
        if window:
            seen = seen & ((keys[None, :] > pos - window) | (keys[None, :] < sinks))
        p = _softmax_rows(scores, seen)
        o = torch.matmul(p.view(hkv, g * (r1 - r0), -1), vf)
        out[r0:r1] = o.view(hq, r1 - r0, d).transpose(0, 1)
    return out


def _run_plain(state):
    case = state["case"]
    if case["op"] == "tables":
        return _tables_plain(state)
    if case["op"] == "write":
        slots, page = state["slots"], case["page"]
        ok = slots >= 0
        at = slots[ok]
        for x, pool in zip(state["kv"], state["pools"]):
            pool[at // page, :, at % page] = x[:, ok].transpose(0, 1)
        return state["pools"]
    if case["op"] == "window":
        q, k, v = state["q"], state["k"], state["v"]
        n, nk = case["n"], case["nk"]
        outs = [_attend_plain(q[b], k[b], v[b], state["scale"], nk - n, case["window"], case["sinks"]) for b in range(case["batch"])]
        return torch.stack(outs).to(torch.bfloat16)
    q, table, page = state["q"], state["table"], case["page"]
    lens, new = state["host"]
    hkv, d = case["hkv"], case["d"]
    if state["cu"] is None:
        # one token each: the caches side by side, padded to the longest
        b, width = table.shape
        hq = case["hq"]
        ids = table.clamp(min=0).long()
        k, v = (pool[ids].permute(0, 2, 1, 3, 4).reshape(b, hkv, width * page, d).float() for pool in (state["k"], state["v"]))
        pos = (state["lens"].long() - 1)[:, None]
        keys = torch.arange(width * page, device=q.device)[None, :]
        seen = keys <= pos
        if case["window"]:
            seen = seen & ((keys > pos - case["window"]) | (keys < case["sinks"]))
        v = torch.where((keys <= pos)[:, None, :, None], v, torch.zeros_like(v))
        qf = q.transpose(0, 1).float().reshape(b, hkv, hq // hkv, d)
        scores = torch.matmul(qf, k.transpose(2, 3).contiguous()) * state["scale"]
        p = _softmax_rows(scores, seen[:, None, None, :])
        return torch.matmul(p, v).reshape(b, hq, d).to(torch.bfloat16)
    outs, at = [], 0
    for i, (total, n) in enumerate(zip(lens, new)):
        ids = table[i, :_ceil(total, page)].long()
        k, v = (pool[ids].transpose(0, 1).reshape(hkv, -1, d)[:, :total] for pool in (state["k"], state["v"]))
        outs.append(_attend_plain(q[:, at:at + n], k, v, state["scale"], total - n, case["window"], case["sinks"]))
        at += n
    return torch.cat(outs).to(torch.bfloat16)


def _tables_plain(state):
    page, tokens, pages = state["case"]["page"], state["tokens"], state["pages"]
    lens, new, table, free = state["lens"].long(), state["new"].long(), state["table"], state["free"].long()
    b, width = table.shape
    dev = table.device
    count = state["free_count"].long()
    zero = torch.zeros(1, dtype=torch.int64, device=dev)
    have = torch.clamp((lens + page - 1) // page, max=width)
    need = torch.clamp((lens + new + page - 1) // page, max=width) - have
    page_end, token_end = torch.cumsum(need, 0), torch.cumsum(new, 0)
    cu = torch.cat((zero, token_end))
    page_at = page_end - need
    # the new entries of every row: the stack's top goes to the first request that opens a page
    col = torch.arange(width, device=dev)[None, :]
    fresh = (col >= have[:, None]) & (col < (have + need)[:, None])
    order = count - 1 - (page_at[:, None] + col - have[:, None])
    ids = torch.where(order >= 0, free[order.clamp(min=0, max=max(free.numel() - 1, 0))], torch.full_like(order, -1))
    table.copy_(torch.where(fresh, ids.to(torch.int32), table))
    # the new tokens
    t = torch.arange(tokens, device=dev)
    row = (t[:, None] >= token_end[None, :]).sum(1)
    real = row < b
    row = row.clamp(max=b - 1)
    pos = torch.where(real, lens[row] + t - cu[row], torch.zeros_like(t))
    entry = table[row, (pos // page).clamp(max=width - 1)].long()
    ok = real & (pos // page < width) & (entry >= 0) & (entry < pages)
    slots = torch.where(ok, entry * page + pos % page, torch.full_like(pos, -1))
    left = (count - page_end[-1:]).to(torch.int32)
    return table, (lens + new).to(torch.int32), cu.to(torch.int32), slots, pos.to(torch.int32), left


# ---- what a pass cannot do without --------------------------------------------------------------------------------
def _pairs(first, n, window, sinks):
    """-> (pairs of query and key that are seen, keys that any query sees) for queries at first .. first + n - 1"""
    if not window:
        return n * first + n * (n + 1) // 2, first + n
    pairs = 0
    # rows whose window still reaches the first key see p + 1 keys; the others the window and what sinks lie in front of it
    whole = min(max(window - first, 0), n)
    pairs += whole * first + whole * (whole + 1) // 2
    for_sinks = [(p - window + 1) for p in (first + whole, first + n - 1)]
    rest = n - whole
    pairs += rest * window
    if rest and sinks:
        a, z = for_sinks  # keys in front of the window, from a up to z
        short = max(0, min(z, sinks - 1) - a + 1)
        pairs += short * (2 * a + short - 1) // 2 + (rest - short) * sinks
    lo = max(0, first - window + 1)
    return pairs, first + n - lo + min(sinks, lo)


def work(case):
    if case["op"] == "tables":
        cached, new = _lengths(case)
        b, t, page = len(new), max(sum(new), 1), case["page"]
        opened = sum(_ceil(c + n, page) - _ceil(c, page) for c, n in zip(cached, new))
        return {"bytes": 4.0 * (2 * b + b + b + 1 + 2 * opened) + 12.0 * t, "flops": 0.0}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "write":
        t = case["tokens"]
        return {"bytes": 8.0 * t * hkv * d + 8.0 * t, "flops": 0.0}
    if case["op"] == "window":
        pairs, keys = _pairs(case["nk"] - case["n"], case["n"], case["window"], case["sinks"])
        b = case["batch"]
        return {"bytes": 2.0 * b * d * (2 * case["n"] * hq + 2 * keys * hkv), "flops": 4.0 * b * d * hq * pairs}
    total_bytes = flops = 0.0
    for c, n in zip(*_lengths(case)):
        pairs, keys = _pairs(c, n, case["window"], case["sinks"])
        total_bytes += 2.0 * d * (2 * n * hq + 2 * keys * hkv) + 4.0 * _ceil(c + n, case["page"])
        flops += 4.0 * d * hq * pairs
    return {"bytes": total_bytes, "flops": flops}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "tables":
        return _tables_exact(state)
    if case["op"] == "write":
        page = case["page"]
        slots = state["slots"].tolist()
        pools = [pool.cpu() for pool in state["pools"]]
        for x, pool in zip(state["kv"], pools):
            x = x.cpu()
            flat = pool.permute(0, 2, 1, 3).reshape(-1, pool.shape[1], pool.shape[3]).clone()
            for t, s in enumerate(slots):
                if s >= 0:
                    flat[s] = x[:, t]
            pool.copy_(flat.view(pool.shape[0], page, pool.shape[1], pool.shape[3]).permute(0, 2, 1, 3))
        return [pool.to(torch.float64).cuda() for pool in pools]
    q, hq, g = state["q"], case["hq"], case["hq"] // case["hkv"]
    if case["op"] == "window":
        out = torch.empty(case["batch"], case["n"], hq, case["d"], dtype=torch.float64, device=q.device)
        for b in range(case["batch"]):
            for h in range(hq):
                out[b, :, h] = _head_exact(q[b, h], state["k"][b, h // g], state["v"][b, h // g], state["scale"], case["window"], case["sinks"])
        return out
    lens, new = state["host"]
    out = torch.empty(sum(new), hq, case["d"], dtype=torch.float64, device=q.device)
    at = 0
    for i, (total, n) in enumerate(zip(lens, new)):
        where = torch.arange(total, device=q.device)
        pages, rows = state["table"][i].long()[where // case["page"]], where % case["page"]
        for h in range(hq):
            out[at:at + n, h] = _head_exact(q[h, at:at + n], state["k"][pages, h // g, rows], state["v"][pages, h // g, rows], state["scale"],
                                            case["window"], case["sinks"])
        at += n
    return out


def _head_exact(q, k, v, scale, window, sinks):
    """one head: q [n, D] the last n of k's positions"""
    n, total = q.shape[0], k.shape[0]
    k64, v64 = k.double().t().contiguous(), v.double()
    out = torch.empty(n, q.shape[1], dtype=torch.float64, device=q.device)
    j = torch.arange(total, device=q.device)
    for r in range(0, n, 2048):
        i = torch.arange(r, min(n, r + 2048), device=q.device)[:, None] + (total - n)
        hidden = j > i
        if window:
            hidden |= (i - j >= window) & (j >= sinks)
        logits = (q[r:r + 2048].double() @ k64).mul_(scale).masked_fill_(hidden, -math.inf)
        weights = torch.softmax(logits, dim=-1)
        out[r:r + 2048] = weights @ v64
    return out


def _tables_exact(state):
    page = state["case"]["page"]
    lens, new, free = state["lens"].tolist(), state["new"].tolist(), state["free"].tolist()
    table = state["table"].tolist()
    stack = free[:state["free_count"].item()]
    slots, positions, cu = [], [], [0]
    for i, (length, n) in enumerate(zip(lens, new)):
        for p in range(length, length + n):
            if p % page == 0:
                table[i][p // page] = stack.pop()
            slots.append(table[i][p // page] * page + p % page)
            positions.append(p)
        cu.append(cu[-1] + n)
    pad = state["tokens"] - len(slots)
    make = lambda x, t: torch.tensor(x, dtype=t, device=state["table"].device)
    return (make(table, torch.int32), make([a + b for a, b in zip(lens, new)], torch.int32), make(cu, torch.int32),
            make(slots + [-1] * pad, torch.int64), make(positions + [0] * pad, torch.int32), make([len(stack)], torch.int32))
