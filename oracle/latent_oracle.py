"""
CPU oracle for the latent cache's operators — TEST INFRASTRUCTURE ONLY (imported by tests/ alone; the product package never imports it).

Dense float64 statements of what a layer of pithtrain/models/deepseek_v2_lite.py:420-470 computes for tokens whose predecessors lie in a cache, one
sequence and one token at a time. Inputs are taken at the values they hold; nothing is rounded on the way.

  append_rows     :430-435 (kv_a_layernorm), :173-187 and :446-447 (rotation of k_pe)
  absorb_query    :437-445 with kv_b_proj's W_uk moved to the query's side
  absorb_value    the same for W_uv
  attention       softmax over the rows that a token sees, sums of absolute values for error bounds beside it
  expanded        the layer as the reference writes it (keys and values of every head), which pins the absorbed form: tests/test_latent.py
"""

import math

import torch

from oracle.prologue_oracle import deinterleave, rope

LATENT, ROPE, NOPE, VALUE = 512, 64, 128, 128


def rotate(pe, cos, sin, positions):
    """pe [T, h, 64] (pairs interleaved) at the given positions of the tables."""
    return rope(deinterleave(pe.double()).unsqueeze(0), cos.double()[positions].unsqueeze(0), sin.double()[positions].unsqueeze(0))[0]


def append_rows(kv_a, weight, cos, sin, positions, eps):
    x = kv_a.double()
    c = x[:, :LATENT]
    n = c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps) * weight.double()
    return n, rotate(x[:, None, LATENT:], cos, sin, positions)[:, 0]


def absorb_query(q, weight):
    t, h, _ = q.shape
    w = weight.double().reshape(h, NOPE + VALUE, LATENT)[:, :NOPE]
    q = q.double()[..., :NOPE]
    return torch.stack([q[:, i] @ w[i] for i in range(h)], 1), torch.stack([q[:, i].abs() @ w[i].abs() for i in range(h)], 1)


def absorb_value(o_latent, weight):
    t, h, _ = o_latent.shape
    w = weight.double().reshape(h, NOPE + VALUE, LATENT)[:, NOPE:]
    x = o_latent.double()
    return torch.stack([x[:, i] @ w[i].T for i in range(h)], 1), torch.stack([x[:, i].abs() @ w[i].abs().T for i in range(h)], 1)


def sees(n, length, words=None):
    """[n, length] truth values: which of its sequence's cached rows each of the n newest tokens sees."""
    before = length - n
    j = torch.arange(length)
    if words is None:
        return j[None] <= before + torch.arange(n)[:, None]
    seen = torch.zeros(n, length, dtype=torch.bool)
    for t in range(n):
        for key in range(length):
            seen[t, key] = key < before or (key - before < 64 and (int(words[t]) >> (key - before)) & 1 == 1)
    return seen


def attention(q_latent, q_pe, latent, k_pe, seen, scale):
    """q_latent [n, h, 512], q_pe [n, h, 64], latent [L, 512], k_pe [L, 64], seen [n, L]. Returns o [n, h, 512], lse [h, n] in bits, sum_j P_j |c_j|
    [n, h, 512] and the largest sum of absolute products behind a score of each row [n, h], in bits. Rows that see nothing: 0, -inf, 0, 0."""
    n, h, _ = q_latent.shape
    ql, qp, c, p = q_latent.double(), q_pe.double(), latent.double(), k_pe.double()
    kappa = scale * math.log2(math.e)
    o, mass = torch.zeros(n, h, LATENT, dtype=torch.float64), torch.zeros(n, h, LATENT, dtype=torch.float64)
    lse, spread = torch.full((h, n), -math.inf, dtype=torch.float64), torch.zeros(n, h, dtype=torch.float64)
    for t in range(n):
        keys = seen[t].nonzero()[:, 0]
        if keys.numel() == 0:
            continue
        ck, pk = c[keys], p[keys]
        s = (ql[t] @ ck.T + qp[t] @ pk.T) * kappa
        lse[:, t] = torch.logsumexp(s * math.log(2), -1) / math.log(2)
        w = torch.exp2(s - lse[:, t, None])
        o[t], mass[t] = w @ ck, w @ ck.abs()
        spread[t] = ((ql[t].abs() @ ck.abs().T + qp[t].abs() @ pk.abs().T) * abs(kappa)).amax(-1)
    return o, lse, mass, spread


def expanded(q, n_latent, rotated_pe, weight, cos, sin, positions, scale):
    """The layer over one sequence with keys and values of every head: q [S, h, 192] (rope part not rotated yet), causal; o [S, h, 128]."""
    s, h, _ = q.shape
    kv = (n_latent.double() @ weight.double().T).reshape(s, h, NOPE + VALUE)
    k = torch.cat((kv[..., :NOPE], rotated_pe.double()[:, None].expand(s, h, ROPE)), -1)
    qq = torch.cat((q.double()[..., :NOPE], rotate(q[..., NOPE:], cos, sin, positions)), -1)
    score = torch.einsum("qhd,khd->hqk", qq, k) * scale
    score = score.masked_fill(torch.ones(s, s).triu(1).bool(), -math.inf)
    return torch.einsum("hqk,khv->qhv", score.softmax(-1), kv[..., NOPE:])
