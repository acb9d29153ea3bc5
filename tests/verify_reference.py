"""Drafted trees against given random numbers, in 64 bits, from the definition: every rest is normalised before the next child is tried."""
import math

import torch


def distribution(x, temperature, top_p):
    """fp64 probabilities of one row of logits; None for a row that is no distribution."""
    x = x.double().cpu()
    if bool(torch.isnan(x).any()) or x.max() == math.inf or x.max() == -math.inf:
        return None
    p = torch.softmax(x / temperature, 0)
    if top_p < 1:
        order = torch.sort(x, descending=True)
        mass = p[order.indices]
        before = torch.cumsum(mass, 0) - mass
        first = torch.searchsorted(-order.values, -x, right=False)  # (the first place of an entry's equals: their mass does not count)
        p = torch.where(before[first] <= top_p, p, 0.0)
    return p / p.sum()


def pick(p, u):
    run = torch.cumsum(p, 0)
    at = int((run <= u * run[-1]).sum())
    return at if at < len(p) else int(torch.nonzero(p)[-1])


def judge(logits, tokens, parents, row0, n, uniforms, draft, temperature, top_p, draft_temperature, draft_top_p):
    """(path, next token) of one entry."""
    walk = [0]
    while True:
        v = walk[-1]
        row = row0 + v
        p = distribution(logits[row], temperature, top_p)
        kids = [i for i in range(v + 1, n) if parents[row0 + i] == v]
        if p is None:
            return walk, -1
        if uniforms is None or draft is None:
            t = int((logits[row] == logits[row].max()).nonzero()[0]) if uniforms is None else pick(p, float(uniforms[row, 1]))
            same = [i for i in kids if tokens[row0 + i] == t]
            if not same:
                return walk, t
            walk.append(same[0])
            continue
        rest, ahead = p, None
        if kids:
            q = distribution(draft[row], draft_temperature, draft_top_p)
            if q is None:
                return walk, -1
            for i in kids:
                x = tokens[row0 + i]
                if not 0 <= x < len(p):
                    continue
                if float(uniforms[row0 + i, 0]) * float(q[x]) < float(rest[x]):
                    ahead = i
                    break
                less = (rest - q).clamp(min=0)
                if float(less.sum()) <= 0:
                    rest = p
                    break
                rest = less / less.sum()
        if ahead is None:
            return walk, pick(rest, float(uniforms[row, 1]))
        walk.append(ahead)
