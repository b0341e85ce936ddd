"""
CPU oracle for the key-value cache's operators — TEST INFRASTRUCTURE ONLY (imported by tests/ alone; the product package never imports it).

Dense float64 statements (integers: loops over lists) of what a layer of pithtrain/models/qwen3_30b_a3b.py:413-438 computes for tokens whose predecessors lie
in a cache, one sequence and one token at a time. Inputs are taken at the values they hold; nothing is rounded on the way.

  plan        pages of a pool and rows of requests, a request after the other
  append      :417-421 (q_norm, k_norm, rotation), the values as they are
  attention   softmax over the rows that a token sees, sums of absolute values for error bounds beside it
  bounds      least and largest features of a page
  select      every page's score, the best by a sort
"""

import math

import torch

from oracle.latent_oracle import sees  # noqa: F401  (the same rule of who sees what)
from oracle.prologue_oracle import rope


def plan(counts, lengths, table, free, count, page, tokens):
    """Lists in, lists out: a dict of cu_q, position_ids, slots, granted, lengths, free_count, page_table, free."""
    lengths, table, free = list(lengths), [list(r) for r in table], list(free)
    width = len(table[0]) if table else 0
    for i, c in enumerate(counts):
        if c < 0:
            for p in table[i][: -(-lengths[i] // page)]:
                if count < len(free):
                    free[count] = p
                    count += 1
            lengths[i] = 0
    cu, positions, slots, granted, refused = [0], [], [], [], False
    for i, c in enumerate(counts):
        n = min(max(c, 0), tokens - cu[-1])
        held = -(-lengths[i] // page)
        fits = c >= 0 and lengths[i] + n <= width * page
        need = -(-(lengths[i] + n) // page) - held if fits else 0
        served = fits and (need == 0 or (not refused and need <= count))
        refused = refused or (fits and not served)
        for j in range(need if served else 0):
            count -= 1
            table[i][held + j] = free[count]
        for at in range(lengths[i], lengths[i] + n):
            positions.append(at)
            slots.append(table[i][at // page] * page + at % page if served else -1)
        granted.append(n if served else 0)
        lengths[i] += granted[-1]
        cu.append(cu[-1] + n)
    positions += [0] * (tokens - len(positions))
    slots += [-1] * (tokens - len(slots))
    return dict(cu_q=cu, position_ids=positions, slots=slots, granted=granted, lengths=lengths, free_count=[count], page_table=table, free=free)


def norm_rope(x, weight, cos, sin, positions, eps):
    """(rot(norm(x)), the same sum with absolute values) of x [T, heads, d] at the given positions of the tables."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    c, s = cos.double()[positions], sin.double()[positions]
    half = x.shape[-1] // 2
    mass = (x * c[:, None]).abs() + (torch.cat((x[..., half:], x[..., :half]), -1) * s[:, None]).abs()
    return rope(x.unsqueeze(0), c.unsqueeze(0), s.unsqueeze(0))[0], mass


def attention(q, k, v, seen, scale):
    """(o, lse in bits, sum of P |v|, largest sum of |q k| in bits) of q [n, h, d] against k, v [hkv, rows, d]; seen [n, rows]."""
    n, h, _ = q.shape
    group = h // k.shape[0]
    o, lse, mass, spread = [], [], [], []
    for i in range(h):
        kk, vv, qq = k[i // group].double(), v[i // group].double(), q[:, i].double()
        s = (qq @ kk.T) * (scale / math.log(2))
        s = torch.where(seen, s, -math.inf)
        top = s.max(-1, keepdim=True).values if s.shape[1] else torch.full((n, 1), -math.inf, dtype=torch.double)
        p = torch.exp2(s - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        p = torch.where(total == 0, 0.0, p / total)
        vv = torch.where(seen.any(0)[:, None], vv, 0.0)  # what nobody sees may hold anything
        o.append(p @ vv)
        mass.append(p @ vv.abs())
        lse.append((top + torch.log2(total))[:, 0])
        a = (qq.abs() @ kk.abs().T) * (abs(scale) / math.log(2))
        spread.append(torch.where(seen, a, 0.0).amax(-1) if s.shape[1] else torch.zeros(n, dtype=torch.double))
    return torch.stack(o, 1), torch.stack(lse), torch.stack(mass, 1), torch.stack(spread, 1)


def bounds(rows):
    """[hkv, 2, d] of a page's rows [hkv, page, d]."""
    return torch.stack((rows.double().min(1).values, rows.double().max(1).values), 1)


def scores(q, lo_hi):
    """[hkv, pages] in fp32 (the operator's definition) of one token's q [h, d] against bounds [pages, hkv, 2, d]."""
    pages, hkv, _, d = lo_hi.shape
    q = q.double().view(hkv, -1, 1, d)
    x = lo_hi.double().transpose(0, 1)[:, None]  # [hkv, 1, pages, 2, d]
    return torch.maximum(q * x[..., 0, :], q * x[..., 1, :]).sum(-1).amax(1).float()


def select(q, lo_hi, visible, page, keep):
    """Per key-value head the kept pages (numbers within the sequence), of one token that sees `visible` rows; lo_hi: bounds of its pages."""
    pages = -(-visible // page)
    hkv = lo_hi.shape[1]
    if pages <= keep:
        return [list(range(pages))] * hkv
    s = scores(q, lo_hi[: pages - 1])
    keys = [[math.inf if math.isnan(x) else x for x in row] for row in s.tolist()]
    nan = torch.isnan(s).tolist()
    return [sorted(sorted(range(pages - 1), key=lambda j: (not nan[g][j], -keys[g][j], j))[: keep - 1]) + [pages - 1] for g in range(hkv)]
