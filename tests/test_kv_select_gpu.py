"""Selection of pages on the GPU where many pages are close to the border of the choice, where one has bounds of another size than the rest, for more tokens than
are taken at a time, and with token offsets that do not begin at 0 or that fall. The choice is exact: it has to be the oracle's. test_kv_gpu.py has the ordinary calls."""

import pytest
import test_kv_gpu as G
import torch

from oracle import kv_oracle as O
from pithtrain_amd.operators.gqa import kv_cache as K

pytestmark = pytest.mark.gpu
BF, I32 = G.BF, G.I32


# ---------------------------------------------------------------------------------------------
# Many pages in question


def _close(pages, heads, values, seed):
    """Bounds whose scores differ by less than a sum of 32 bits over the features is known to: 1 (or -1) in all features but the last, which is one of `values`."""
    g = torch.Generator().manual_seed(seed)
    bounds = torch.ones(pages, heads, 2, 64) * (-1 if max(values) < 0 else 1)
    last = torch.tensor(values)[torch.randint(0, len(values), (pages, heads), generator=g)]
    bounds[..., 0, 63], bounds[..., 1, 63] = last, last
    return bounds.to(BF)


def _ones(monkeypatch):
    made = G.Batch.__init__

    def of_ones(self, *args, **kw):
        made(self, *args, **kw)
        self.q.fill_(1.0)

    monkeypatch.setattr(G.Batch, "__init__", of_ones)


# sums of absolute values are 63 and a little: scores that lie 2^-8 apart, E, may stand in either order
VALUES = {"equal": [0.5], "two": [0.0, 2.0**-17], "many": [2.0**-9 * (1 + i / 128) for i in range(128)], "below": [-(2.0**-9) * (1 + i / 128) for i in range(128)]}
# tables of one launch, of up to 2048 pages and of more
WIDTHS = [(250, 200), (250, 3), (254, 129), (1999, 700), (1999, 5), (16381, 4000), (9001, 77)]


@pytest.mark.parametrize("values", VALUES)
@pytest.mark.parametrize("pages, keep", WIDTHS, ids=str)
def test_choices_among_many_pages_in_question(gpu, monkeypatch, pages, keep, values):
    _ones(monkeypatch)
    lengths = [16 * pages, 16 * (pages - 7) + 3]
    _selection_of(gpu, lengths, keep, _close(2 * (pages + 2), 2, VALUES[values], pages))


@pytest.mark.parametrize("pages, keep", WIDTHS, ids=str)
def test_choices_among_pages_without_anything_in_them(gpu, pages, keep):
    """A cache of zeros: all scores are 0 exactly."""
    _selection_of(gpu, [16 * pages - 5], keep, torch.zeros(pages + 2, 2, 2, 64, dtype=BF))


def _selection_of(gpu, lengths, keep, bounds):
    G._selection(gpu, lengths, (4, 2, 64), keep, seed=3, bounds=bounds)


@pytest.mark.parametrize("pages, keep", [(250, 60), (2000, 64), (16000, 64)])
@pytest.mark.parametrize("size", [30.0, 1000.0, 1e30])
def test_choices_beside_a_page_with_bounds_of_another_size(gpu, pages, keep, size):
    g = torch.Generator().manual_seed(pages)
    x = torch.randn(pages + 2, 2, 2, 64, generator=g)
    x[::97] *= size
    bounds = torch.stack((x.amin(2), x.amax(2)), 2).to(BF)
    _selection_of(gpu, [16 * pages - 3], keep, bounds)
    bounds[:, :, 1] = bounds[:, :, 0]  # and of scores on both sides of the others'
    _selection_of(gpu, [16 * pages - 3], keep, bounds)


def _us(call, calls=20):
    call()
    first, last = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    first.record()
    for _ in range(calls):
        call()
    last.record()
    torch.cuda.synchronize()
    return first.elapsed_time(last) * 1000 / calls


@pytest.mark.parametrize("pages", [2000, 16000])
def test_one_page_of_another_size_or_equal_scores_do_not_take_a_call_out_of_proportion(gpu, pages):
    """Only pages whose own sums may be off by what separates them from the border are summed anew: one page with bounds ten thousand times as large as the rest makes no more
    of them. Equal scores do, and a page is summed and counted, not compared with all others: the time grows like the pages, not like their square. (us measured: 2000 pages 18,
    21 and 370, 16000 pages 70, 90 and 2450, for eight tokens.)"""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(pages, 4, 2, 64, generator=g)
    ordinary = torch.stack((x.amin(2), x.amax(2)), 2).to(BF).to(gpu)
    outlying, equal = ordinary.clone(), torch.ones_like(ordinary)
    outlying[pages // 2] *= 10000
    q = torch.randn(2, 8, 64, generator=g).to(BF).to(gpu)
    table, lens = torch.arange(pages, dtype=I32, device=gpu).repeat(2, 1), torch.tensor([16 * pages - 1] * 2, dtype=I32, device=gpu)
    us = {name: _us(lambda: K.kv_select_pages(q, bounds, table, lens, None, 16, 64)) for name, bounds in (("ordinary", ordinary), ("outlying", outlying), ("equal", equal))}
    print(us)
    assert us["outlying"] < 10 * us["ordinary"], us
    assert us["equal"] < 10 * us["ordinary"] + 0.5 * pages, us


# ---------------------------------------------------------------------------------------------
# Offsets


@pytest.mark.parametrize("width", [40, 300])
@pytest.mark.parametrize("offsets, same", [([2, 4, 3, 6], [2, 4, 4, 6]), ([-3, 2, 2, 5], [0, 2, 2, 5]), ([0, 3, 5, 99], [0, 3, 5, 7]), ([5, 1, 6, 6], [5, 5, 6, 6]), ([0, 4, 2, 1], [0, 4, 4, 4]), ([-(2**31), 3, 3, 2**31 - 1], [0, 3, 3, 7])], ids=str)
def test_offsets_count_as_their_maximum_so_far_in_all_operators(gpu, offsets, same, width):
    """As in the attention: tokens in front of the first offset and from the last on are nobody's, falling offsets give no tokens, those beyond the tokens end there."""
    g = torch.Generator().manual_seed(width)
    page, t, pages = 16, 7, 3 * width
    b = G.Batch(gpu, [3, 2, 2], [9, 9, 9], (4, 2, 64), page=page, seed=1)
    k = torch.randn(pages, 2, page, 64, generator=g).to(BF).to(gpu)
    cache = K.KVCache(k, k)
    table = torch.randperm(pages, generator=g).to(I32).view(3, width).to(gpu)
    lens = torch.tensor([page * (width - 1) + 1, page * width, page * (width - 3) + 2], dtype=I32, device=gpu)
    first = torch.stack((k.amin(2), k.amax(2)), 2) + torch.tensor([-1.0, 1.0], device=gpu).to(BF)[:, None]
    results = []
    for cu in (offsets, same):
        cu_q = torch.tensor(cu, dtype=I32, device=gpu)
        bounds = first.clone()
        K.kv_page_bounds(cache, bounds, table, lens, cu_q, t)
        o, lse = torch.full_like(b.q, 7.0), torch.full((4, t), 8.0, device=gpu)
        K.kv_attention_into(b.q, cache, table, lens, cu_q, 0.1, None, o, lse)
        results.append((bounds, *K.kv_select_pages(b.q, first, table, lens, cu_q, page, 5), o, lse))
    for got, want in zip(*results):
        assert torch.equal(got, want)
    bounds, chosen, rows, o, _ = results[0]
    mine = torch.zeros(t, dtype=torch.bool)
    for i in range(3):
        mine[same[i] : same[i + 1]] = True
        for at in range(same[i], same[i + 1]):
            assert (rows[at] == int(lens[i]) - same[i + 1] + at + 1 - page * (-(-(int(lens[i]) - same[i + 1] + at + 1) // page) - 5)).all()
    assert (chosen[~mine] == -1).all() and (rows[~mine] == 0).all() and (o[~mine] == 7).all() and (chosen[mine] >= 0).all() and (o[mine] != 7).any()


@G.BOTH
@pytest.mark.parametrize("b, prompt", [(1, 1500), (700, 1500), (700, 200), (1500, 40)])
def test_bounds_of_a_prompt_among_many_sequences(gpu, b, prompt, fp8):
    """More pages than workgroups of a sequence, behind more sequences than are looked at together."""
    page, at = 16, b - 1
    counts = [1] * b
    counts[at] = prompt
    lengths = [1 + (5 * i) % 40 for i in range(b)]
    lengths[at] = prompt + 21
    x = G.Batch(gpu, counts, lengths, (4, 2, 64), page=page, fp8=fp8, seed=b)
    bounds = torch.full_like(x.cache.empty_bounds(), 3.0)
    K.kv_page_bounds(x.cache, bounds, x.table, x.lens, x.cu_q, sum(counts))
    filled = torch.cat([x.table[i, (n - c) // page : n // page].cpu() for i, (c, n) in enumerate(zip(counts, lengths))]).long()
    keys = x.kv[0][filled.to(gpu)].float() * (1.0 if x.scales[0] is None else x.scales[0][filled.to(gpu)][..., None])
    assert len(filled) > prompt // page and torch.equal(bounds[filled.to(gpu)], torch.stack((keys.amin(2), keys.amax(2)), 2).to(BF))
    others = torch.ones(len(bounds), dtype=torch.bool)
    others[filled] = False
    assert (bounds[others.to(gpu)] == 3).all()


# ---------------------------------------------------------------------------------------------
# Many tokens


def test_many_tokens_are_chosen_for_in_parts(gpu):
    """More tokens than one part of the workspace holds: the choice for each is the one that it gets in a call of few."""
    g = torch.Generator().manual_seed(2)
    pages, page, t = 2048, 16, 2300
    x = torch.randn(pages, 4, 2, 64, generator=g)
    bounds = torch.stack((x.amin(2), x.amax(2)), 2).to(BF).to(gpu)
    q = torch.randn(t, 8, 64, generator=g).to(BF).to(gpu)
    table = torch.randperm(pages, generator=g).to(I32).view(1, pages).repeat(2, 1).to(gpu)
    counts = [1900, 390]  # and ten that are nobody's
    lens, cu_q = [page * 2040 + 7, page * pages], torch.tensor([0, 1900, 2290], dtype=I32, device=gpu)
    chosen, rows = K.kv_select_pages(q, bounds, table, torch.tensor(lens, dtype=I32, device=gpu), cu_q, page, 30)
    for i, (first, n) in enumerate(zip((0, 1900), counts)):
        for at in range(0, n, 100):
            few = min(100, n - at)
            visible = torch.tensor([lens[i] - n + at + few], dtype=I32, device=gpu)
            want = K.kv_select_pages(q[first + at : first + at + few], bounds, table[i : i + 1], visible, torch.tensor([0, few], dtype=I32, device=gpu), page, 30)
            assert torch.equal(chosen[first + at : first + at + few], want.page_table) and torch.equal(rows[first + at : first + at + few], want.lengths), (i, at)
    assert (chosen[2290:] == -1).all() and (rows[2290:] == 0).all()
    some = 1234
    want = O.select(q[some].cpu(), bounds[table[0].long()].cpu(), lens[0] - 1900 + some + 1, page, 30)
    assert all(torch.equal(chosen[some, j].cpu(), table[0].cpu()[want[j]]) for j in range(4))


def test_a_captured_choice_for_many_tokens(gpu):
    g = torch.Generator().manual_seed(4)
    x = torch.randn(700, 16, 2, 64, generator=g)
    bounds = torch.stack((x.amin(2), x.amax(2)), 2).to(BF).to(gpu)
    q, table = torch.randn(1500, 16, 64, generator=g).to(BF).to(gpu), torch.arange(700, dtype=I32, device=gpu).view(1, -1)
    lens, cu_q = torch.tensor([16 * 700], dtype=I32, device=gpu), torch.tensor([0, 1500], dtype=I32, device=gpu)
    call = lambda: K.kv_select_pages(q, bounds, table, lens, cu_q, 16, 9)  # noqa: E731
    call()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        got = call()
    for length in (16 * 700, 1600, 16 * 650 + 5, 16 * 700):
        lens.fill_(length)
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
