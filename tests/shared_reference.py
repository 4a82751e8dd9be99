"""Inputs and the 64-bit reference of the operators of caches whose requests share a start: the mask and bounds are paged_reference's, request by request."""

import torch

from paged_reference import reference


def make_shared(groups, alone, hkv, d, page, gen, slack=4, fill=float("nan")):
    """groups: [(shared keys, [own keys of every request])], alone: [keys of requests that share nothing], which come last.
    -> (pools, table, lens, shared_lens, cu_groups, [(k, v)] of every request [Hkv, len, D], [shared keys of every request]); `fill` stands where no key does.
    Whole pages of shared keys are named by all requests of a group; a page that is shared in part is copied."""
    rows, lens, prefix, need, kv = [], [], [], 0, []
    draw = lambda n: torch.randn(hkv, n, d, generator=gen).to(torch.bfloat16)
    for shared, owns in list(groups) + [(0, [n]) for n in alone]:
        common, first = (draw(shared), draw(shared)), None
        for own in owns:
            total, whole = shared + own, shared // page if first is not None else 0
            pages = -(-total // page)
            rows.append((first[:whole] if whole else []) + list(range(need, need + pages - whole)))
            need += pages - whole
            first = first if first is not None else rows[-1]
            lens.append(total)
            prefix.append(shared)
            kv.append(tuple(torch.cat((c, draw(own)), 1) for c in common))
    order = torch.randperm(need + slack, generator=gen)
    width = max(max(len(r) for r in rows), 1)
    table = torch.full((len(rows), width), -1, dtype=torch.int32)
    pools = [torch.full((need + slack, hkv, page, d), fill, dtype=torch.bfloat16) for _ in range(2)]
    for b, r in enumerate(rows):
        ids = order[torch.tensor(r, dtype=torch.int64)]
        table[b, :len(r)] = ids.to(torch.int32)
        for pool, x in zip(pools, kv[b]):
            for i, page_id in enumerate(ids.tolist()):
                part = x[:, i * page:(i + 1) * page]
                pool[page_id, :, :part.shape[1]] = part
    cu = [0]
    for _, owns in groups:
        cu.append(cu[-1] + len(owns))
    return pools, table, lens, [g[0] for g in groups], cu, kv, prefix


def references(q, kv, new, scale):
    """q [Hq, T, D] of the requests one behind the other -> (out [T, Hq, D], bound)"""
    outs, bounds, at = [], [], 0
    for (k, v), n in zip(kv, new):
        out, bound = reference(q[:, at:at + n], k, v, scale, 0, 0)
        outs.append(out), bounds.append(bound)
        at += n
    return torch.cat(outs), torch.cat(bounds)


def key_weights(q, k, scale):
    """[Hkv, len]: the sums of the softmax weights of the last n keys' queries q [Hq, n, D], in 64 bits"""
    hq, n, d = q.shape
    hkv, total, _ = k.shape
    out = torch.zeros(hkv, total, dtype=torch.float64)
    for i in range(n):
        seen = total - n + i + 1
        if seen <= 0:
            continue
        for h in range(hq):
            out[h // (hq // hkv), :seen] += torch.softmax(k[h // (hq // hkv), :seen].double() @ q[h, i].double() * scale, 0)
    return out


def weight_bound(q, k, scale):
    """How far a weight may be from that, relative to it: a logit is off by (D + 4) 2^-24 of its largest term, the row's maximum and sum by as much again, an
    exponential by 2^-21, and a sum of n terms by n 2^-24."""
    d = q.shape[2]
    largest = scale * k.double().abs().sum(2).max().item() * q.double().abs().max().item()
    return 3 * (d + 4) * 2.0 ** -24 * largest + 2.0 ** -20 + (k.shape[1] + q.shape[0] * q.shape[1]) * 2.0 ** -24
