"""Attention to the key-value cache: what the weights of few rows keep, that calls take the kernels that they are meant for, which rows are written whatever tables,
lengths and offsets hold, and steps that attend to selected pages, against the fp64 oracle. The bounds are test_kv_gpu.py's, where not said otherwise."""

import math

import pytest
import test_kv_gpu as G
import torch

from oracle import kv_oracle as O
from pithtrain_amd.operators import paging
from pithtrain_amd.operators.gqa import kv_cache as K
from pithtrain_amd.operators.mla import latent as L

pytestmark = pytest.mark.gpu
BF, I32, I64, U = G.BF, G.I32, G.I64, G.U


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


# ---------------------------------------------------------------------------------------------
# Which kernel a call takes


@G.BOTH
@pytest.mark.parametrize("heads", [(74, 2, 128), (80, 2, 64)], ids=str)
@pytest.mark.parametrize("name", ["none", "few_tokens", "prompt", "contradiction"])
def test_every_set_of_lengths_reaches_the_blocks_of_more_rows(gpu, monkeypatch, name, heads, fp8):
    """64 rows of bf16 heads of 128, 32 of the others."""
    taken = G._wide(monkeypatch, 64)
    counts, lengths = G.LENGTH_SETS[name]
    b = G.Batch(gpu, counts, lengths, heads, page=16 if name == "prompt" else 64, fp8=fp8, seed=len(name))
    taken(b)
    b.check(*b.attention(), name)


def test_blocks_of_64_rows_where_there_is_that_much_to_read(gpu):
    """Keys and values of 200 MB and more, in tables no wider than they need be."""
    lengths = [8192 - 37 * i for i in range(13)]
    b = G.Batch(gpu, [8] * 13, lengths, (32, 4, 128), seed=22)
    assert G._rows_of(b) == 64
    b.check(*b.attention())


# ---------------------------------------------------------------------------------------------
# What is written


BAD = {
    "pages": (2**31 - 1, None, None, 4),
    "pages_below": (-(2**31), None, None, 4),
    "lengths": (None, [2**31 - 1, -5, -(2**31)], None, 4),
    "offsets": (None, None, [-7, 3, 2, 2**31 - 1], 6),
    "offsets_beyond": (None, None, [9, 9, 9, 9], 0),
}


@pytest.mark.parametrize("width", [20, 300])
@pytest.mark.parametrize("name", BAD)
def test_bad_tables_lengths_and_offsets_write_their_tokens_and_nothing_else(gpu, name, width):
    page, lens, offsets, written = BAD[name]
    b = G.Batch(gpu, [2, 1, 1], [40, 70, 300], extra_tokens=2, seed=10, page=16)
    table = torch.full((3, width), 1 if page is None else page, dtype=I32, device=gpu)
    if page is None:
        table[:, : b.table.shape[1]] = torch.where(b.table == -1, 3, b.table)
    lens = b.lens if lens is None else torch.tensor(lens, dtype=I32, device=gpu)
    cu_q = b.cu_q if offsets is None else torch.tensor(offsets, dtype=I32, device=gpu)
    o, lse = torch.full_like(b.q, 7.0), torch.full((b.h, 6), 8.0, device=gpu)
    K.kv_attention_into(b.q, b.cache, table, lens, cu_q, b.scale, None, o, lse)
    assert (o[:written] != 7).flatten(1).any(1).all() and (lse[:, :written] != 8).all()
    assert (o[written:] == 7).all() and (lse[:, written:] == 8).all()
    bounds = torch.zeros(b.kv[0].shape[0], b.hkv, 2, b.d, dtype=BF, device=gpu)
    chosen, rows = K.kv_select_pages(b.q, bounds, table, lens, cu_q, 16, 3)
    assert (rows[written:] == 0).all() and (chosen[written:] == -1).all() and (0 <= rows).all() and (rows <= 3 * 16).all()
    if page is None:
        named = (rows + 15) // 16  # pages that were chosen, the first ones of their row
        assert torch.equal(chosen != -1, torch.arange(3, device=gpu) < named[..., None])
    K.kv_page_bounds(b.cache, bounds, table, lens, cu_q, 6)
    if written == 0:
        assert not bounds.any()


# ---------------------------------------------------------------------------------------------
# Steps that attend to selected pages


@G.BOTH
def test_steps_that_attend_to_some_of_their_pages(gpu, fp8):
    """Requests of up to 12 pages of which a token keeps 4: every result is the attention to the pages that the oracle chooses, for the queries as they were rounded, by the
    bounds of the keys that the cache holds."""
    h, hkv, d, page, pages, b, keep, width = 8, 2, 128, 16, 40, 3, 4, 12
    g = torch.Generator().manual_seed(60)
    cache = K.KVCache.empty(pages, hkv, d, page, L.FP8 if fp8 else BF, gpu)
    for x in cache:
        if x is not None:
            x.view(torch.uint8).fill_(0x7F)  # NaN
    bounds = cache.empty_bounds().fill_(math.nan)
    pool, table, lengths = paging.PagePool.full(pages, gpu), torch.full((b, width), -1, dtype=I32, device=gpu), torch.zeros(b, dtype=I32, device=gpu)
    cos, sin = (x.to(gpu) for x in G._tables(d, 300))
    w = [(1 + 0.2 * torch.randn(d, generator=g)).to(BF).to(gpu) for _ in range(2)]
    scale, dropped = d**-0.5, 0
    for new in [[70, 33, 0], [1, 1, 90], [1, 1, 1], [30, -1, 1], [1, 80, 1], [3, 1, 2], [16, 16, 16], [1, 1, 1]]:
        tokens = sum(max(c, 0) for c in new) + 3
        qkv = torch.randn(tokens, h + 2 * hkv, d, generator=g).to(BF).to(gpu)
        plan = paging.plan_step(torch.tensor(new, dtype=I32, device=gpu), lengths, table, pool, page, tokens)
        lengths, pool = plan.lengths, paging.PagePool(pool.free, plan.free_count)
        assert plan.granted.tolist() == [max(c, 0) for c in new]
        parts = qkv.split((h, hkv, hkv), 1)
        out = K.kv_decode(*parts, *w, cos, sin, plan.position_ids, plan.slots, cache, table, lengths, plan.cu_q, scale, bounds=bounds, keep=keep)
        other = K.KVCache(*(None if x is None else x.clone() for x in cache))
        q = K.kv_cache_append(*parts, *w, cos, sin, plan.position_ids, plan.slots, other)  # the queries as the step had them
        first = 0
        for i, c in enumerate(new):
            length, entries = int(lengths[i]), table[i]
            j = torch.arange(length, device=gpu)
            at, row = entries[j // page].long(), j % page
            keys, values = (
                (x.to(torch.float32)[at, :, row].double() * (1.0 if s is None else s[at, :, row].double()[..., None])).transpose(0, 1).cpu()
                for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))
            )
            whole = entries[: length // page].long()
            of_pages = cache.k[whole].float() * (1.0 if cache.k_scale is None else cache.k_scale[whole][..., None])
            assert torch.equal(bounds[whole], torch.stack((of_pages.amin(2), of_pages.amax(2)), 2).to(BF)), "bounds of full pages"
            known = torch.cat((bounds[whole].cpu(), torch.zeros(1, hkv, 2, d, dtype=BF)))  # (a last page that is not full is not scored)
            for k in range(max(c, 0)):
                visible = length - c + k + 1
                kept = O.select(q[first + k].cpu(), known, visible, page, keep)
                dropped += -(-visible // page) > keep
                for head in range(hkv):
                    mine = slice(head * (h // hkv), (head + 1) * (h // hkv))
                    mask = torch.tensor([[m < visible and m // page in kept[head] for m in range(length)]])
                    want, _, mass, spread = O.attention(q[first + k : first + k + 1, mine].cpu(), keys[head : head + 1], values[head : head + 1], mask, scale)
                    e = (d + 8) * 2.0**-24 * spread
                    G._within(out[first + k : first + k + 1, mine], want, U * want.abs() + (U + 2 * (e[..., None] * math.log(2) + 2.0**-16)) * mass, f"{new} request {i} token {k} head {head}")
            first += max(c, 0)
        assert (out[first:] == 0).all()
    assert dropped > 100
