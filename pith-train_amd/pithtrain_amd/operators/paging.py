"""
The bookkeeping of a step of serving, on the device: pages for new rows out of a pool, pages of requests that ended back into it, and the token offsets,
positions and slots that latent_cache_append / kv_cache_append and the attentions to those caches take. One launch (two for many tokens), no host
synchronisation: a captured graph can hold a whole step, bookkeeping included.

 T : tokens of the step, padding included, b : requests.
"""

from typing import NamedTuple

import torch

from pithtrain_amd import _C
from pithtrain_amd._ext import define_op
from pithtrain_amd.operators.mla.latent import _index, _table_args


class PagePool(NamedTuple):
    """Pages that no request holds: the first count[0] entries of free [n] int32, of which the last are taken first. count [1] int32."""

    free: torch.Tensor
    count: torch.Tensor

    @classmethod
    def full(cls, pages: int, device="cuda") -> "PagePool":
        """All of a cache's pages, 0 .. pages - 1; the first to be taken is page 0."""
        return cls(torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=device), torch.tensor([pages], dtype=torch.int32, device=device))


class StepPlan(NamedTuple):
    """What plan_step returns. cu_q [b + 1] int32: offsets of the requests' tokens; lengths [b] int32: cached rows behind the step; position_ids, slots [T]
    int64; granted [b] int32: new rows that have pages; free_count [1] int32: of the pool behind the step. They share one allocation: who keeps one for long clones it."""

    cu_q: torch.Tensor
    lengths: torch.Tensor
    position_ids: torch.Tensor
    slots: torch.Tensor
    granted: torch.Tensor
    free_count: torch.Tensor


def plan_step_into(counts: torch.Tensor, lengths: torch.Tensor, page_table: torch.Tensor, pool: PagePool, page_size: int, plan: StepPlan) -> None:
    """plan_step into tensors of the caller's; plan.lengths may be lengths itself and plan.free_count pool.count itself (a captured step that carries its
    state on), nothing else may overlap."""
    _C.require_device(counts, lengths, page_table, *pool, *plan)
    assert counts.dim() == 1, "counts must be one-dimensional"
    assert plan.position_ids.dim() == 1 and pool.free.dim() == 1, "position_ids and the pool's free pages must be one-dimensional"
    b, t = counts.shape[0], plan.position_ids.shape[0]
    i32, i64 = torch.int32, torch.int64
    args = _C.PlanStepArgs(
        counts=_index(counts, i32, (b,), "counts"), lengths=_index(lengths, i32, (b,), "lengths"),
        free_pages=_index(pool.free, i32, (pool.free.shape[0],), "pool.free"), free_count=_index(pool.count, i32, (1,), "pool.count"),
        cu_q=_index(plan.cu_q, i32, (b + 1,), "plan.cu_q"), position_ids=_index(plan.position_ids, i64, (t,), "plan.position_ids"),
        slots=_index(plan.slots, i64, (t,), "plan.slots"), granted=_index(plan.granted, i32, (b,), "plan.granted"),
        lengths_out=_index(plan.lengths, i32, (b,), "plan.lengths"), free_count_out=_index(plan.free_count, i32, (1,), "plan.free_count"),
        B=b, T=t, pool_size=pool.free.shape[0], page_size=page_size,
    )  # fmt: skip
    args.page_table, args.table_rs, args.table_width = _table_args(page_table, b)
    with torch.cuda.device(counts.device):
        need = max(_C.lib().pith_plan_step_workspace_bytes(_C.byref(args)), 0)
        workspace = torch.empty(need, dtype=torch.uint8, device=counts.device)
        args.workspace, args.workspace_bytes = workspace.data_ptr() if need else None, need
        _C.check(_C.lib().pith_plan_step(_C.byref(args), _C.current_stream(counts)))
    torch.autograd.graph.increment_version((page_table, pool.free, *plan))


def _plan_body(counts, lengths, page_table, free, free_count, page_size, tokens):
    assert tokens >= 0, f"tokens = {tokens}"
    plan = StepPlan(*_plan_fake(counts, lengths, page_table, free, free_count, page_size, tokens))
    plan_step_into(counts, lengths, page_table, PagePool(free, free_count), page_size, plan)
    return tuple(plan)


def _plan_fake(counts, lengths, page_table, free, free_count, page_size, tokens):
    assert counts.dim() == 1, "counts must be one-dimensional"
    b = counts.shape[0]
    mk = lambda n, dtype: counts.new_empty((n,), dtype=dtype)  # noqa: E731
    i32, i64 = torch.int32, torch.int64
    return mk(b + 1, i32), mk(b, i32), mk(tokens, i64), mk(tokens, i64), mk(b, i32), mk(1, i32)


_plan_op = define_op("plan_step", _plan_body, _plan_fake)


def plan_step(counts: torch.Tensor, lengths: torch.Tensor, page_table: torch.Tensor, pool: PagePool, page_size: int, tokens: int) -> StepPlan:
    """Plans a step of b requests. counts [b] int32: new rows of each (0: none), below 0 where a request has ended; lengths [b] int32: rows cached before;
    page_table [b, n] int32: their pages; tokens: T, at least the sum of the counts (what goes beyond is cut off).

    Requests that ended give their ceil(length / page_size) pages back, and have length 0. The others get rows length .. length + count - 1, and the
    pages that these need beyond those they have, from the top of the pool, where ended requests have just laid theirs; or none of them, where the pool does not suffice for
    a request or for one in front of it, or its table is too narrow: then granted is 0, the length stays and its tokens have slots of -1, which an append
    skips (what an attention to their requests gives them is of no use; other requests do not notice). Tokens behind the last request have position 0 and slot -1.
    A request holds the ceil(length / page_size) first pages of its row: where lengths are lowered between steps (drafts that were not taken), the pages
    behind those are the caller's to lay on the pool again, or to keep the length for. A page belongs to one request: one that two tables name would go back to the pool twice. page_table and pool.free are updated in place; lengths and pool.count are not: the
    values behind the step are in the result, and the same call again plans the same step (plan_step_into can write them back)."""
    return StepPlan(*_plan_op(counts, lengths, page_table, pool.free, pool.count, page_size, tokens))


__all__ = ["PagePool", "StepPlan", "plan_step", "plan_step_into"]
