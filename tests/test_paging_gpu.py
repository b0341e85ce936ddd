"""Planning of a step on the GPU, at the edges of what its arguments may hold; test_kv_gpu.py has the plans of ordinary steps."""

import pytest
import torch

from pithtrain_amd.operators import paging

pytestmark = pytest.mark.gpu
I32 = torch.int32


@pytest.mark.parametrize("b, tokens", [(3, 8100), (70, 8100), (3, 9000), (1100, 8100)])
def test_positions_of_a_request_whose_table_is_full_pass_32_bits(gpu, b, tokens):
    """It gets nothing, but its tokens have the positions that come behind its rows, whatever the number of requests and tokens."""
    page = 4096
    width = (2**31 - 1) // page if b < 1000 else 40000
    full, new = width * page, 8000
    counts, lengths = torch.ones(b, dtype=I32), torch.full((b,), 5, dtype=I32)
    counts[1], lengths[1] = new, full
    counts[2:] = 0
    table = torch.zeros(b, width, dtype=I32, device=gpu)
    plan = paging.plan_step(counts.to(gpu), lengths.to(gpu), table, paging.PagePool.full(9, gpu), page, tokens)
    assert plan.granted.tolist()[:3] == [1, 0, 0] and plan.lengths.tolist() == lengths.add(torch.tensor([1] + [0] * (b - 1))).tolist()
    want = torch.cat((torch.tensor([5]), torch.arange(full, full + new), torch.zeros(tokens - new - 1, dtype=torch.int64)))
    assert torch.equal(plan.position_ids.cpu(), want) and (b > 1000 or want.max() >= 2**31)
    assert plan.slots[0] == 5 and (plan.slots[1:] == -1).all()
