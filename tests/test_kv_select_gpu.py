"""Selection of pages on the GPU with token offsets that do not begin at 0 or that fall. test_kv_gpu.py has the ordinary calls."""

import pytest
import test_kv_gpu as G
import torch

from pithtrain_amd.operators.gqa import kv_cache as K

pytestmark = pytest.mark.gpu
BF, I32 = G.BF, G.I32


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
