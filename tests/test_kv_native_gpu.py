"""The native host path of the key-value cache's operators and of the planning of a step: ordinary calls never reach an op's Python body, and both give the same bits
(they end in the same kernels)."""

import pytest
import test_kv_gpu as G
import torch

from pithtrain_amd._ext import native
from pithtrain_amd.operators import paging
from pithtrain_amd.operators.gqa import kv_cache as K

pytestmark = pytest.mark.gpu
BF, I32 = G.BF, G.I32
BODIES = {"plan_step": paging._plan_body, "kv_append": K._append_body, "kv_attention": K._attention_body, "kv_bounds": K._bounds_body, "kv_select": K._select_body}


def _plan(gpu, b, tokens):
    counts = torch.full((b,), tokens // b, dtype=I32, device=gpu)
    counts[::5] = -1
    lengths, table = torch.arange(b, dtype=I32, device=gpu) % 50, torch.arange(b * 700, dtype=I32, device=gpu).view(b, 700)
    free, count = torch.arange(4 * b + 2000, dtype=I32, device=gpu), torch.tensor([b + 900], dtype=I32, device=gpu)
    return "plan_step", [counts, lengths, table, free, count, 16, tokens], [2, 3]


def _append(gpu, t, fp8, weight):
    b = G.Batch(gpu, [1], [300], (5, 2, 64), page=16, fp8=fp8, seed=1)
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(t, 9, 64, generator=g).to(BF).to(gpu)
    w = [None, None] if weight is None else [torch.ones(64, dtype=weight, device=gpu)] * 2
    cos, sin = (x.to(gpu) for x in G._tables(64))
    cache = [None if x is None else x.view(torch.uint8).zero_().view(x.dtype) for x in b.cache]
    slots = (torch.arange(t, device=gpu) * 3) % 400 if t < 100 else torch.full((t,), -1, device=gpu)
    return "kv_append", [*qkv.split((5, 2, 2), 1), *w, cos, sin, torch.arange(t, device=gpu) % 50, slots, *cache, 1e-6], [i for i in range(9, 13) if cache[i - 9] is not None]


def _attention(gpu, fp8, tree, heads=(8, 2, 128)):
    b = G.Batch(gpu, [3, 1, 0], [100, 40, 9], heads, page=16, fp8=fp8, tree=tree, seed=3)
    return "kv_attention", [b.q, *b.cache, b.table, b.lens, b.cu_q, b.scale, b.words], []


def _attention_one(gpu, fp8):
    b = G.Batch(gpu, [1, 1], [100, 40], (8, 2, 64), page=16, fp8=fp8, seed=4)
    return "kv_attention", [b.q, *b.cache, b.table, b.lens, None, b.scale, None], []


def _attention_heads(gpu, fp8):
    b = G.Batch(gpu, [1, 1], [100, 80], (8, 2, 128), page=16, fp8=fp8, seed=5)
    return "kv_attention", [b.q, *b.cache, b.table[:, None, :3].repeat(1, 2, 1), torch.tensor([[40, 48], [33, 0]], dtype=I32, device=gpu), None, b.scale, None], []


def _bounds(gpu, fp8):
    b = G.Batch(gpu, [30, 1], [64, 80], (4, 2, 64), page=16, fp8=fp8, seed=6)
    return "kv_bounds", [*b.cache, b.cache.empty_bounds().zero_(), b.table, b.lens, b.cu_q, 31], [4]


def _select(gpu, width):
    g = torch.Generator().manual_seed(7)
    bounds = torch.randn(width, 2, 2, 64, generator=g).sort(dim=2).values.to(BF).to(gpu)
    q, table = torch.randn(3, 4, 64, generator=g).to(BF).to(gpu), torch.arange(width, dtype=I32, device=gpu).repeat(2, 1)
    return "kv_select", [q, bounds, table, torch.tensor([16 * width, 16 * width - 20], dtype=I32, device=gpu), torch.tensor([0, 2, 3], dtype=I32, device=gpu), 16, 9], []


CALLS = {
    "plan": lambda gpu: _plan(gpu, 20, 60), "plan_prompts": lambda gpu: _plan(gpu, 20, 9000), "plan_some": lambda gpu: _plan(gpu, 100, 700), "plan_some_prompts": lambda gpu: _plan(gpu, 100, 9000),
    "plan_many": lambda gpu: _plan(gpu, 1100, 2200), "append": lambda gpu: _append(gpu, 20, False, BF), "append_fp8": lambda gpu: _append(gpu, 20, True, torch.float32),
    "append_many": lambda gpu: _append(gpu, 2100, True, None), "attention": lambda gpu: _attention(gpu, False, None), "attention_fp8": lambda gpu: _attention(gpu, True, None, (6, 1, 64)),
    "tree": lambda gpu: _attention(gpu, False, "tree"), "one": lambda gpu: _attention_one(gpu, True), "of_heads": lambda gpu: _attention_heads(gpu, False), "of_heads_fp8": lambda gpu: _attention_heads(gpu, True),
    "bounds": lambda gpu: _bounds(gpu, False), "bounds_fp8": lambda gpu: _bounds(gpu, True), "select": lambda gpu: _select(gpu, 100), "select_some": lambda gpu: _select(gpu, 700), "select_many": lambda gpu: _select(gpu, 3000),
}  # fmt: skip


@pytest.mark.parametrize("name", CALLS)
def test_native_and_python_bodies_agree(gpu, name):
    """The op, whose body counts its calls, and the body itself, on copies of what either writes."""
    op, args, written = CALLS[name](gpu)
    called = []
    native.set_bodies({n: (lambda *a, n=n: called.append(n) or BODIES[n](*a)) for n in BODIES})
    try:
        results = []
        for run in (getattr(torch.ops.pithtrain_amd, op).default, BODIES[op]):
            mine = [x.clone() if i in written else x for i, x in enumerate(args)]
            out = run(*mine)
            results.append([*(out if isinstance(out, tuple) else [] if out is None else [out]), *(mine[i] for i in written)])
    finally:
        native.set_bodies(BODIES)
    assert not called, f"an ordinary call went through the Python body of {called}"
    for x, y in zip(*results):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)) and x.dtype == y.dtype


@G.BOTH
@pytest.mark.parametrize("made_inside", [False, True])
def test_steps_in_inference_mode(gpu, made_inside, fp8):
    """The same rows and results as under no_grad, with tensors made inside or outside."""
    g = torch.Generator().manual_seed(8)
    qkv = torch.randn(3, 41, 8, 64, generator=g).to(BF).to(gpu)
    cos, sin = (x.to(gpu) for x in G._tables(64))

    def state():
        cache = K.KVCache.empty(9, 2, 64, 16, G.L.FP8 if fp8 else BF, gpu)
        for x in cache:
            if x is not None:
                x.view(torch.uint8).zero_()
        return cache, cache.empty_bounds().zero_(), torch.full((2, 6), -1, dtype=I32, device=gpu), paging.PagePool.full(9, gpu), torch.zeros(2, dtype=I32, device=gpu)

    def steps(cache, bounds, table, pool, lengths):
        results = []
        for i, counts in enumerate(([40, 1], [1, 17], [3, -1])):
            plan = paging.plan_step(torch.tensor(counts, dtype=I32, device=gpu), lengths, table, pool, 16, 41)
            lengths, pool = plan.lengths, paging.PagePool(pool.free, plan.free_count)
            n = sum(max(c, 0) for c in counts)
            o = K.kv_decode(*qkv[i].split((4, 2, 2), 1), None, None, cos, sin, plan.position_ids, plan.slots, cache, table, lengths, plan.cu_q, 0.125, bounds=bounds, keep=2)
            results += [o[:n], *plan]
        return results + [x for x in (*cache, bounds, table, pool.free) if x is not None]

    with torch.no_grad():
        want = steps(*state())
    outside = state()
    with torch.inference_mode():
        got = steps(*(state() if made_inside else outside))
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(got, want))
