"""Append to the key-value cache where a wave takes all of a token (2048 tokens of a call and more), on both sides of that border, and in place;
test_kv_gpu.py has the calls of few tokens."""

import pytest
import test_kv_gpu as G
import torch

from pithtrain_amd import _C
from pithtrain_amd.operators.gqa import kv_cache as K
from pithtrain_amd.operators.mla import latent as L

pytestmark = pytest.mark.gpu
BF, I64 = G.BF, G.I64


@G.BOTH
@pytest.mark.parametrize("weight", [BF, torch.float32, None], ids=str)
@pytest.mark.parametrize("heads", [(32, 4, 128), (5, 1, 64), (3, 3, 128), (9, 9, 64)], ids=str)
@pytest.mark.parametrize("t", [2047, 2048, 2501])
def test_append_of_many_tokens_matches_the_oracle(gpu, t, heads, weight, fp8):
    G.test_append_matches_the_oracle(gpu, t, heads, weight, fp8)


def _new(gpu, t, heads, seed, fp8):
    h, hkv, d = heads
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(t, n, d, generator=g).to(BF).to(gpu) for n in (h, hkv, hkv))
    w = [(1 + 0.2 * torch.randn(d, generator=g)).to(BF).to(gpu) for _ in range(2)]
    cos, sin = (x.to(gpu) for x in G._tables(d))
    pages = -(-t // 16) + 1
    pos, slots = torch.randint(0, 50, (t,), generator=g).to(gpu), torch.randperm(pages * 16, generator=g)[:t].to(gpu)
    slots[::13] = -1
    caches = []
    for _ in range(2):
        cache = K.KVCache.empty(pages, hkv, d, 16, L.FP8 if fp8 else BF, gpu)
        for x in cache:
            if x is not None:
                x.view(torch.uint8).fill_(0x22)
        caches.append(cache)
    return q, k, v, w, cos, sin, pos, slots, caches


@G.BOTH
@pytest.mark.parametrize("heads", [(32, 4, 128), (7, 1, 64), (5, 5, 128)], ids=str)
def test_append_of_many_tokens_gives_the_bits_of_few(gpu, heads, fp8):
    t = 2222
    q, k, v, w, cos, sin, pos, slots, caches = _new(gpu, t, heads, 1, fp8)
    got = K.kv_cache_append(q, k, v, *w, cos, sin, pos, slots, caches[0])
    for a in range(0, t, 500):
        part = slice(a, a + 500)
        assert torch.equal(K.kv_cache_append(q[part], k[part], v[part], *w, cos, sin, pos[part], slots[part], caches[1]), got[part])
    assert all(x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(*caches))


@G.BOTH
@pytest.mark.parametrize("heads", [(32, 4, 128), (7, 1, 64), (5, 5, 128)], ids=str)
@pytest.mark.parametrize("t", [3, 100, 2047, 2048, 2300])
def test_queries_may_be_overwritten_by_their_results(gpu, t, heads, fp8):
    """Through the C interface, whose q_out may be q."""
    h, hkv, d = heads
    q, k, v, w, cos, sin, pos, slots, caches = _new(gpu, t, heads, 2, fp8)
    want = K.kv_cache_append(q, k, v, *w, cos, sin, pos, slots, caches[0])
    wide = torch.full((t, h + 2, d), 3.0, dtype=BF, device=gpu)
    for at in (q, wide[:, 1:-1]):
        at.copy_(q)
        _, hs = at.stride()[:2]
        args = _C.KVAppendArgs(
            q=at.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_weight=w[0].data_ptr(), k_weight=w[1].data_ptr(), cos=cos.data_ptr(), sin=sin.data_ptr(), position_ids=pos.data_ptr(),
            slots=slots.data_ptr(), q_out=at.data_ptr(), T=t, P=cos.shape[0], H=h, eps=1e-6, weight_dtype=_C.PITH_BF16, cache=K._cache_args(q, *caches[1]),
            q_ts=at.stride(0), q_hs=hs, q_out_ts=at.stride(0), q_out_hs=hs, k_ts=hkv * d, k_hs=d, v_ts=hkv * d, v_hs=d,
        )  # fmt: skip
        saved = q.clone()
        _C.check(_C.lib().pith_kv_append(_C.byref(args), _C.current_stream(q)))
        assert torch.equal(at, want)
        q.copy_(saved)
    assert (wide[:, 0] == 3).all() and (wide[:, -1] == 3).all()
    assert all(x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(*caches))
