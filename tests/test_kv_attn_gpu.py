"""Attention to the key-value cache: what the weights of few rows keep, against the fp64 oracle. The bounds are test_kv_gpu.py's, where not said otherwise."""

import math

import pytest
import test_kv_gpu as G
import torch

from oracle import kv_oracle as O

pytestmark = pytest.mark.gpu
U = G.U


# ---------------------------------------------------------------------------------------------
# Weights


@G.BOTH
@pytest.mark.parametrize("heads", [(8, 2, 128), (32, 4, 128), (16, 1, 64), (5, 1, 64)], ids=str)
@pytest.mark.parametrize("counts, lengths, tree", [([1], [20], None), ([1, 1, 1], [517, 1, 1301], None), ([1], [20011], None), ([1, 1, 0, 1, 1, 1], [40, 130, 3, 1000, 64, 2], None), ([1], [77], "tree")], ids=str)
def test_weights_of_few_rows_lose_no_more_than_a_score_does(gpu, counts, lengths, tree, heads, fp8):
    """Calls that take blocks of 16 rows: a weight goes into the products as the sum of two bf16 numbers, the first cut off (2^-7 of it is left at most), the second
    rounded (2^-8 of that), with 2^-20 of the weight on top: (2^-15 + 2^-20) sum P |v| instead of u."""
    b = G.Batch(gpu, counts, lengths, heads, page=16, fp8=fp8, tree=tree, seed=heads[0] + len(lengths))
    assert G._rows_of(b) == 16
    o, _ = b.attention()
    first = 0
    for i, (n, length) in enumerate(zip(counts, lengths)):
        sl = slice(first, first + n)
        first += n
        if n == 0:
            continue
        seen = O.sees(n, length, None if b.words is None else b.words[sl].tolist())
        want, _, mass, spread = O.attention(b.q[sl].cpu(), *b.rows(b.table[i], length), seen, b.scale)
        e = (b.d + 8) * 2.0**-24 * spread
        G._within(o[sl], want, U * want.abs() + (2.0**-15 + 2.0**-20 + 2 * (e[..., None] * math.log(2) + 2.0**-16)) * mass, f"sequence {i}")


@pytest.mark.parametrize("heads", [(8, 2, 128), (16, 1, 64), (40, 1, 128)], ids=str)
@pytest.mark.parametrize("lengths", [[200], [1], [33, 20011, 64]], ids=str)
def test_infinite_values_that_are_seen_make_infinite_results(gpu, heads, lengths):
    """Whatever their weights: none is so small that it is 0, and the rest of one that is a bf16 number (the largest, 1) is not either."""
    b = G.Batch(gpu, [1] * len(lengths), lengths, heads, page=16, seed=23)
    v = b.kv[1]
    v[..., 3], v[..., 40] = math.inf, -math.inf
    o, lse = b.attention()
    assert (o[..., 3] == math.inf).all() and (o[..., 40] == -math.inf).all() and torch.isfinite(lse).all()
    v[..., 3], v[..., 40] = 1.0, 0.5
    want, _ = b.attention()
    others = torch.tensor([i not in (3, 40) for i in range(b.d)])
    assert torch.equal(o[..., others], want[..., others])
