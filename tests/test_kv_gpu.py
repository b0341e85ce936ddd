"""The key-value cache's operators and the planning of a step on the GPU against the fp64 oracle, through the public entry points.

Bounds are elementwise and come from the arithmetic, u = 2^-8 being bf16's half step relative to the value (torch.finfo(bfloat16).eps / 2):

  a result rounded once from fp32         u |want|; norm and rotation on top 2^-19 of the sum of the absolute values of what the rotation adds (the mean of up to
                                          128 squares, rsqrt, three products and a sum, each off by a few 2^-24)
  e4m3 rows                               2^-4 |want| of the value, but half of its finest step, 2^-10, times the row's scale at least; scales 2^-18
  attention                               the weights P (times the row's scale) are rounded to bf16: u sum P |v|. A score's sum of d products is off by at
                                          most e = (d + 8) 2^-24 (sum of their absolute values, in bits), its exp2, the subtraction of the maximum and the
                                          rescaling by 2^-16 in all: weight and denominator 2 (e ln 2 + 2^-16) sum P |v|. And u |want| for the result.
  lse                                     e + 2^-17 bits (|lse| < 64: its own step is 2^-18)
  plans, bounds of pages and selections   equal
"""

import math

import pytest
import torch

from oracle import kv_oracle as O
from oracle import prologue_oracle as P
from pithtrain_amd import _C
from pithtrain_amd.operators import paging
from pithtrain_amd.operators.gqa import kv_cache as K
from pithtrain_amd.operators.mla import latent as L

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
U = 2.0**-8
I32, I64 = torch.int32, torch.int64


def _within(got, want, bound, what):
    got, want, bound = got.double().cpu(), want.double().cpu(), bound.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)), f"{what}: finite and non-finite values elsewhere than expected"
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine], want[~fine]), f"{what}: other infinities"
    over = ((got - want).abs() - bound)[fine]
    assert over.numel() == 0 or over.max() <= 0, f"{what}: off by {((got - want).abs() / bound.clamp_min(1e-300))[fine].max():.3f} times the bound"


# ---------------------------------------------------------------------------------------------
# Attention


MIN_WIDTH = 0  # of page tables: blocks of more than 16 query rows are for those that are wide


class Batch:
    """Sequences in a cache. counts: new tokens of each, lengths: cached rows of each. Everything that no sequence owns (rows behind the last one of a
    page, pages of nobody, table entries that are not needed) holds NaN or nonsense."""

    def __init__(self, dev, counts, lengths, heads=(8, 2, 128), page=64, fp8=False, tree=None, seed=0, extra_tokens=0, q_std=1.0):
        g = torch.Generator().manual_seed(seed)
        mk = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.h, self.hkv, self.d = heads
        self.counts, self.lengths, self.dev, self.page, self.scale = counts, lengths, dev, page, self.d**-0.5
        t = sum(counts) + extra_tokens
        need = [-(-n // page) for n in lengths]
        pages, width = sum(need) + 3, max(max(need), 1, MIN_WIDTH) + 1
        order = torch.randperm(pages, generator=g)
        table = torch.randint(-5, 2 * pages, (len(counts), width), generator=g).to(I32)  # entries behind a sequence's pages are never followed
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = order[at : at + n]
            at += n
        self.table = table.to(dev)
        self.kv = []
        self.scales = []
        for _ in range(2):
            x = torch.full((pages, page, self.hkv, self.d), math.nan)
            for i, n in enumerate(lengths):
                j = torch.arange(n)
                x[table[i, j // page].long(), j % page] = mk(n, self.hkv, self.d) * (0.5 + torch.rand(self.hkv, self.d, generator=g))
            x = x.transpose(1, 2).contiguous()
            scale = None
            if fp8:
                scale = x.abs().amax(-1) / 448
                x = (x / scale[..., None]).clamp(-448, 448).to(L.FP8)
                scale = scale.to(dev)
            self.kv.append((x if fp8 else x.to(BF)).to(dev))
            self.scales.append(scale)
        self.q = (q_std * mk(t, self.h, self.d)).to(BF).to(dev)
        self.cu_q = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=I32, device=dev)
        self.lens = torch.tensor(lengths, dtype=I32, device=dev)
        self.words = None
        if tree is not None:
            rows = [L.tree_mask_of(torch.tensor([int(torch.randint(max(-1, i - 6), i, (1,), generator=g)) for i in range(n)], dtype=I64)) if n else torch.empty(0, dtype=I64) for n in counts]
            self.words = torch.cat(rows + [torch.zeros(extra_tokens, dtype=I64)])
            if tree == "holes":  # words that leave rows out, and nothing at all for some
                self.words &= torch.randint(-(1 << 62), 1 << 62, self.words.shape, generator=g)
                self.words[::3] = 0
            self.words = self.words.to(dev)

    @property
    def cache(self):
        return K.KVCache(*self.kv, *self.scales)

    def rows(self, table, length):
        """Keys and values of the first rows of a table's pages at the values they hold, [hkv, length, d]."""
        j = torch.arange(length, device=self.dev)
        p, r = table[j // self.page].long(), j % self.page
        out = []
        for x, scale in zip(self.kv, self.scales):
            y = x.to(torch.float32)[p, :, r].double() * (1.0 if scale is None else scale[p, :, r].double()[..., None])
            out.append(y.transpose(0, 1).cpu())
        return out

    def attention(self, words="own"):
        return K.kv_attention(self.q, self.cache, self.table, self.lens, self.cu_q, self.scale, self.words if words == "own" else words)

    def close(self, o, lse, q, k, v, seen, what, slack=0.0):
        want, want_lse, mass, spread = O.attention(q.cpu(), k, v, seen, self.scale)
        e = (self.d + 8) * 2.0**-24 * spread + slack * want_lse.T.abs().nan_to_num(posinf=0.0)
        _within(o, want, U * want.abs() + (U + 2 * (e[..., None] * math.log(2) + 2.0**-16)) * mass, f"{what}: o")
        _within(lse, want_lse, e.T + 2.0**-17, f"{what}: lse")

    def check(self, o, lse, what="", slack=0.0):
        o, lse, first = o.cpu(), lse.cpu(), 0
        for i, (n, length) in enumerate(zip(self.counts, self.lengths)):
            sl = slice(first, first + n)
            first += n
            if n == 0:
                continue
            seen = O.sees(n, length, None if self.words is None else self.words[sl].tolist())
            self.close(o[sl], lse[:, sl], self.q[sl], *self.rows(self.table[i], length), seen, f"{what} sequence {i}", slack)


LENGTH_SETS = {
    "one_row": ([1], [1]),
    "tiny": ([1, 1, 1, 1, 1], [1, 15, 16, 17, 31]),
    "tile_ends": ([1] * 9, [32, 33, 63, 64, 65, 96, 127, 128, 129]),
    "ordinary": ([1, 1, 1], [517, 1, 1301]),
    "none": ([1, 0, 1, 0], [0, 70, 40, 0]),
    "few_tokens": ([2, 3, 1, 5], [2, 64, 700, 37]),
    "prompt": ([70, 33], [70, 129]),
    "contradiction": ([4, 3], [2, 0]),  # more new tokens than rows: the first of them see nothing
}
HEADS = [(32, 4, 128), (8, 2, 64), (5, 1, 128), (3, 3, 64), (40, 2, 128), (16, 1, 64), (70, 1, 128)]
BOTH = pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])


@BOTH
@pytest.mark.parametrize("heads", HEADS[:4], ids=str)
@pytest.mark.parametrize("name", LENGTH_SETS)
def test_attention_matches_the_oracle(gpu, name, heads, fp8):
    counts, lengths = LENGTH_SETS[name]
    b = Batch(gpu, counts, lengths, heads, page=16 if name in ("tiny", "prompt") else 64, fp8=fp8, seed=len(name))
    b.check(*b.attention(), name)


@BOTH
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_attention_of_other_head_counts(gpu, heads, fp8):
    b = Batch(gpu, [1, 2, 9], [333, 90, 200], heads, page=32, fp8=fp8, seed=heads[0])
    b.check(*b.attention())


@BOTH
@pytest.mark.parametrize("page", [16, 32, 128, 1024])
def test_attention_page_sizes(gpu, page, fp8):
    b = Batch(gpu, [1, 3], [page + 5, 2 * page], page=page, fp8=fp8, seed=page)
    b.check(*b.attention())


@BOTH
@pytest.mark.parametrize("heads", [(8, 1, 128), (4, 2, 64)], ids=str)
def test_attention_of_one_long_sequence_is_joined_from_many_parts(gpu, fp8, heads):
    b = Batch(gpu, [1, 1], [20011, 3], heads, fp8=fp8, seed=3, q_std=2.0)
    b.check(*b.attention())


def test_attention_of_more_sequences_than_a_wavefront_scans_at_once(gpu):
    g = torch.Generator().manual_seed(4)
    counts = torch.randint(0, 3, (150,), generator=g).tolist()
    lengths = [max(n, int(x)) for n, x in zip(counts, torch.randint(0, 400, (150,), generator=g))]
    b = Batch(gpu, counts, lengths, (4, 2, 64), page=16, seed=5)
    b.check(*b.attention())


@BOTH
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("b, every, most", [(150, 1, 1), (300, 2, 3), (4300, 9, 1), (4300, 50, 2), (4200, 4150, 1)], ids=str)
def test_attention_of_many_sequences_of_which_few_have_tokens(gpu, monkeypatch, b, every, most, wide, fp8):
    if wide:
        monkeypatch.setitem(globals(), "MIN_WIDTH", 256)
    counts = [1 + i % most if i % every == every - 1 else 0 for i in range(b)]
    x = Batch(gpu, counts, [(7 * i) % 130 for i in range(b)], (4, 2, 64), page=16, fp8=fp8, seed=21, extra_tokens=2)
    x.check(*x.attention())


def test_attention_of_more_row_blocks_than_workgroups(gpu):
    b = Batch(gpu, [1] * 300, [7 + i % 200 for i in range(300)], (8, 4, 64), page=16, seed=6)
    b.check(*b.attention())


def test_large_scores_do_not_overflow(gpu):
    b = Batch(gpu, [1, 2], [300, 65], seed=6, q_std=200.0)
    o, lse = b.attention()
    assert torch.isfinite(o.float()).all() and lse.abs().max() > 500
    b.check(o, lse, slack=2.0**-22)  # lse is in the hundreds here: its bound grows with it (a few more roundings of 2^-24 |lse|)


@BOTH
@pytest.mark.parametrize("kind", ["tree", "holes"])
@pytest.mark.parametrize("counts,lengths,heads", [([1], [1], (8, 2, 128)), ([8, 8], [517, 8], (16, 2, 64)), ([64, 1, 33], [64, 300, 1000], (3, 1, 128)), ([7, 0, 12], [40, 5, 12], (8, 1, 64)), ([64], [63], (2, 2, 128))])
def test_tree_attention_matches_the_oracle(gpu, counts, lengths, heads, kind, fp8):
    b = Batch(gpu, counts, lengths, heads, page=16, fp8=fp8, tree=kind, seed=sum(counts) + heads[0])
    o, lse = b.attention()
    b.check(o, lse, kind)
    if kind == "holes" and lengths == [1]:
        assert (o == 0).all() and (lse == -math.inf).all()


# Blocks of 32 and 64 rows: the same tests with page tables so wide that calls of more than 16 rows a sequence take them.
def _rows_of(b):
    fp8 = b.scales[0] is not None
    c = _C.KVCacheArgs(k=256, v=256, k_scale=256 * fp8, v_scale=256 * fp8, pages=1, page_size=b.page, heads=b.hkv, dim=b.d, dtype=_C.PITH_FP8_E4M3 if fp8 else _C.PITH_BF16)
    args = _C.KVAttnArgs(cache=c, cu_q=256, T=b.q.shape[0], B=len(b.counts), H=b.h, table_width=b.table.shape[1])
    return _C.lib().pith_kv_attn_rows(_C.byref(args))


def _wide(monkeypatch, rows):
    """Page tables that make sure of it (64 rows: only with bf16 heads of 128); returns what checks it."""
    monkeypatch.setitem(globals(), "MIN_WIDTH", 1 << 16)

    def taken(b):
        assert _rows_of(b) == (min(rows, 32) if b.scales[0] is not None or b.d != 128 else rows)

    return taken


@BOTH
@pytest.mark.parametrize("rows, heads", [(32, (16, 2, 128)), (64, (32, 2, 128)), (64, (32, 2, 64)), (32, (16, 2, 64)), (64, (74, 2, 128)), (64, (35, 1, 64))], ids=str)
@pytest.mark.parametrize("name", ["none", "few_tokens", "prompt", "contradiction"])
def test_blocks_of_more_rows_match_the_oracle(gpu, monkeypatch, name, rows, heads, fp8):
    taken = _wide(monkeypatch, rows)
    counts, lengths = LENGTH_SETS[name]
    b = Batch(gpu, counts, lengths, heads, page=16 if name == "prompt" else 64, fp8=fp8, seed=len(name))
    if name == "few_tokens":
        taken(b)
    b.check(*b.attention(), name)


@BOTH
@pytest.mark.parametrize("rows, heads, counts, lengths", [
    (32, (4, 1, 128), [8, 4], [20011, 300]), (64, (8, 1, 64), [63], [9001]), (32, (16, 2, 128), [2, 0, 9] * 40, list(range(7, 127))), (64, (24, 2, 128), [3, 0, 9] * 40, list(range(9, 129))), (32, (3, 1, 64), [8] * 70, list(range(50, 120)))],
    ids=["long", "longer", "many", "many_more", "odd"])  # fmt: skip
def test_work_lists_of_blocks_of_more_rows(gpu, monkeypatch, rows, heads, counts, lengths, fp8):
    taken = _wide(monkeypatch, rows)
    b = Batch(gpu, counts, lengths, heads, page=16, fp8=fp8, seed=15, q_std=1.5)
    taken(b)
    b.check(*b.attention())


@BOTH
@pytest.mark.parametrize("kind", ["tree", "holes"])
@pytest.mark.parametrize("rows, heads", [(32, (4, 2, 128)), (64, (6, 2, 64)), (64, (8, 1, 128))], ids=str)
def test_trees_in_blocks_of_more_rows_match_the_oracle(gpu, monkeypatch, rows, heads, kind, fp8):
    taken = _wide(monkeypatch, rows)
    b = Batch(gpu, [12, 16, 9], [517, 16, 200], heads, page=16, fp8=fp8, tree=kind, seed=rows)
    taken(b)
    b.check(*b.attention(), kind)


@BOTH
@pytest.mark.parametrize("tree", [None, "tree"])
@pytest.mark.parametrize("where", ["key", "value", "scale"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("heads", [(8, 2, 128), (14, 1, 64)], ids=str)
def test_blocks_of_more_rows_are_not_reached_by_rows_that_they_do_not_see(gpu, monkeypatch, bad, where, tree, fp8, heads):
    _wide(monkeypatch, 0)
    test_a_row_that_a_token_does_not_see_cannot_reach_it(gpu, bad, where, tree, fp8, heads)


def test_a_chain_of_drafts_is_the_causal_call(gpu):
    b = Batch(gpu, [5, 9], [200, 60], seed=8)
    words = torch.cat([L.tree_mask_of(torch.arange(-1, n - 1)) for n in b.counts]).to(gpu)
    for x, y in zip(b.attention(), b.attention(words)):
        assert torch.equal(x, y)


@BOTH
@pytest.mark.parametrize("tree", [None, "tree"])
@pytest.mark.parametrize("where", ["key", "value", "scale"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("heads", [(8, 2, 128), (6, 1, 64), (24, 2, 128)], ids=str)
def test_a_row_that_a_token_does_not_see_cannot_reach_it(gpu, bad, where, tree, fp8, heads):
    """The newest row of a sequence holds infinities or NaN: tokens that do not see it are computed as ever, and those that do know of it."""
    if where == "scale" and not fp8:
        pytest.skip("bf16 rows have no scale")
    b = Batch(gpu, [6, 6], [70, 6], heads, page=16, seed=9, tree=tree, fp8=fp8)
    want_o, want_lse = b.attention()
    blind = torch.ones(12, dtype=torch.bool)
    for i in range(2):
        j = b.lengths[i] - 1
        page, row = b.table[i, j // 16].long(), j % 16
        for which in {"key": [0], "value": [1], "scale": [0, 1]}[where]:
            if where == "scale":
                b.scales[which][page, :, row] = bad
            elif fp8:
                b.kv[which].view(torch.uint8)[page, :, row, 20:] = 0x7F
            else:
                b.kv[which][page, :, row, 20:] = bad
        blind[6 * i + 5] = False
        if tree:
            blind[6 * i : 6 * i + 6] = (b.words[6 * i : 6 * i + 6].cpu() >> 5) & 1 == 0
    assert 2 <= blind.sum() < 12
    o, lse = b.attention()
    assert torch.equal(o[blind], want_o[blind]) and torch.equal(lse[:, blind], want_lse[:, blind])
    if where == "value":
        assert torch.equal(lse, want_lse) and torch.equal(o[..., :20], want_o[..., :20])
        got = o[~blind][..., 20:].float()
        assert (torch.isnan(got) if math.isnan(bad) or fp8 else got == bad).all()
    else:
        assert torch.isnan(o[~blind].float()).any()


@BOTH
def test_a_single_draft_that_does_not_see_itself_is_not_reached_by_its_row(gpu, fp8):
    b = Batch(gpu, [1, 1], [90, 1], page=16, fp8=fp8, tree="tree", seed=14)
    b.words.zero_()
    want = b.attention()
    b.check(*want)
    for i in range(2):
        j = b.lengths[i] - 1
        for x in b.kv:
            x[b.table[i, j // 16].long(), :, j % 16] = math.nan
    assert all(torch.equal(x, y) for x, y in zip(b.attention(), want))


def test_tokens_behind_the_last_sequence_keep_what_they_hold(gpu):
    b = Batch(gpu, [2, 1], [40, 70], extra_tokens=3, seed=10)
    o, lse = torch.full_like(b.q, 7.0), torch.full((b.h, 6), 8.0, device=gpu)
    K.kv_attention_into(b.q, b.cache, b.table, b.lens, b.cu_q, b.scale, None, o, lse)
    b.check(o[:3], lse[:, :3])
    assert (o[3:] == 7).all() and (lse[:, 3:] == 8).all()


@BOTH
def test_strides(gpu, fp8):
    """Queries and results as slices, a cache whose layers share an allocation, a page table as a column range, results of heads apart."""
    b = Batch(gpu, [2, 1], [40, 170], seed=11, fp8=fp8, page=32)
    want = b.attention()
    wide = torch.zeros(3, b.h + 3, 2 * b.d, dtype=BF, device=gpu)
    wide[:, 1:-2, b.d :] = b.q
    layers = []
    for x in b.kv + ([] if b.scales[0] is None else b.scales):
        both = torch.zeros((x.shape[0], 2) + tuple(x.shape[1:]), dtype=x.dtype, device=gpu)
        both[:, 1].copy_(x)
        layers.append(both[:, 1])
    table = torch.full((2, b.table.shape[1] + 5), -3, dtype=I32, device=gpu)
    table[:, 2:-3] = b.table
    o, lse = torch.zeros(3, 2 * b.h, b.d, dtype=BF, device=gpu), torch.zeros(b.h, 9, device=gpu)
    K.kv_attention_into(wide[:, 1:-2, b.d :], K.KVCache(*layers), table[:, 2:-3], b.lens, b.cu_q, b.scale, None, o[:, ::2], lse[:, 4:7])
    assert torch.equal(o[:, ::2], want[0]) and torch.equal(lse[:, 4:7], want[1]) and (o[:, 1::2] == 0).all() and (lse[:, :4] == 0).all()
    got = K.kv_attention(wide[:, 1:-2, b.d :], K.KVCache(*layers), table[:, 2:-3], b.lens, b.cu_q, b.scale)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    odd = torch.zeros(3, b.h, b.d + 1, dtype=BF, device=gpu)  # rows off the alignment: copied
    odd[..., 1:] = b.q
    got = K.kv_attention(odd[..., 1:], b.cache, b.table, b.lens, b.cu_q, b.scale)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@BOTH
@pytest.mark.parametrize("heads", [(8, 2, 128), (6, 3, 64), (20, 1, 128)], ids=str)
def test_attention_with_a_table_of_every_head(gpu, fp8, heads):
    """Every token and head attends to rows of its own choice."""
    b = Batch(gpu, [1, 1, 1], [200, 90, 333], heads, page=16, fp8=fp8, seed=12)
    g = torch.Generator().manual_seed(13)
    t, hkv = 3, b.hkv
    table, lengths = torch.full((t, hkv, 7), -1, dtype=I32), torch.zeros(t, hkv, dtype=I32)
    for i in range(t):
        for j in range(hkv):
            n = int(torch.randint(0, 8, (1,), generator=g)) if i else 7
            pages = torch.randint(0, b.lengths[i] // 16, (n,), generator=g)  # whole pages, one more than once perhaps
            table[i, j, :n] = b.table[i].cpu()[pages]
            lengths[i, j] = max(n * 16 - int(torch.randint(0, 16, (1,), generator=g)), 0)
    assert (lengths == 0).any() or hkv == 1
    for width in (7, 60):  # whole, and cut into parts some of which are empty
        wide = torch.full((t, hkv, width), -1, dtype=I32)
        wide[..., :7] = table
        o, lse = (x.cpu() for x in K.kv_attention(b.q, b.cache, wide.to(gpu), lengths.to(gpu), None, b.scale))
        for i in range(t):
            for j in range(hkv):
                n, mine = int(lengths[i, j]), slice(j * (b.h // hkv), (j + 1) * (b.h // hkv))
                k, v = b.rows(table[i, j].to(gpu).clamp(min=0), n)
                b.close(o[i : i + 1, mine], lse[mine, i : i + 1], b.q[i : i + 1, mine], k[j : j + 1], v[j : j + 1], O.sees(1, n), f"token {i} head {j}")
    with pytest.raises(AssertionError, match="no cu_q"):
        K.kv_attention(b.q, b.cache, table.to(gpu), lengths.to(gpu), b.cu_q, b.scale)


def test_bad_tables_lengths_and_offsets_stay_in_memory(gpu):
    """Nonsense in what the kernels index by: wrong rows, but every token of a sequence is written, and nothing else."""
    b = Batch(gpu, [2, 1, 1], [40, 70, 300], extra_tokens=2, seed=10, page=16)
    for table, lens, cu_q in [
        (torch.full_like(b.table, 2**31 - 1), b.lens, b.cu_q),
        (torch.full_like(b.table, -(2**31)), b.lens, b.cu_q),
        (b.table, torch.tensor([2**31 - 1, -5, -(2**31)], dtype=I32, device=gpu), b.cu_q),
        (b.table, b.lens, torch.tensor([-7, 3, 2, 2**31 - 1], dtype=I32, device=gpu)),
        (b.table, b.lens, torch.tensor([9, 9, 9, 9], dtype=I32, device=gpu)),
    ]:
        o, lse = torch.full_like(b.q, 7.0), torch.full((b.h, 6), 8.0, device=gpu)
        K.kv_attention_into(b.q, b.cache, table, lens, cu_q, b.scale, None, o, lse)
        K.kv_select_pages(b.q, torch.zeros(b.kv[0].shape[0], b.hkv, 2, b.d, dtype=BF, device=gpu), table, lens, cu_q, 16, 3)
        K.kv_page_bounds(b.cache, b.cache.empty_bounds(), table, lens, cu_q, 6)
        torch.cuda.synchronize()
    assert (o == 7).all() and (lse == 8).all()  # offsets behind the tokens: nobody's


# ---------------------------------------------------------------------------------------------
# Append


def _tables(d, n=50):
    cos, sin = P.cos_sin_table(torch.arange(n).unsqueeze(0), d, dtype=BF)
    return cos[0], sin[0]


@BOTH
@pytest.mark.parametrize("weight", [BF, torch.float32, None], ids=str)
@pytest.mark.parametrize("heads", [(32, 4, 128), (5, 1, 64), (3, 3, 128)], ids=str)
@pytest.mark.parametrize("t", [1, 13, 130])
def test_append_matches_the_oracle(gpu, t, heads, weight, fp8):
    h, hkv, d = heads
    g = torch.Generator().manual_seed(t + h)
    mk = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    qkv = (2 * mk(t, h + 2 * hkv, d) * (0.2 + torch.rand(t, 1, 1, generator=g))).to(BF)
    qkv[t // 2, h + hkv :] = 0  # a row of zeros
    q, k, v = qkv.split((h, hkv, hkv), 1)
    w = [None, None] if weight is None else [(1 + 0.3 * mk(d)).to(weight) for _ in range(2)]
    cos, sin = _tables(d)
    page = 16
    pages = -(-t // page) + 2
    pos, slots = torch.randint(0, 50, (t,), generator=g), torch.randperm(pages * page, generator=g)[:t]
    if t > 1:
        slots[3], slots[7] = -1, pages * page  # padding
    cache = K.KVCache.empty(pages, hkv, d, page, L.FP8 if fp8 else BF, gpu)
    for x in cache:
        if x is not None:
            x.view(torch.uint8).fill_(0x11)
    before = [None if x is None else x.clone() for x in cache]
    on = lambda x: None if x is None else x.to(gpu)  # noqa: E731
    out = K.kv_cache_append(*qkv.to(gpu).split((h, hkv, hkv), 1), on(w[0]), on(w[1]), on(cos), on(sin), on(pos), on(slots), cache, 1e-6)
    want, mass = O.norm_rope(q, w[0], cos, sin, pos, 1e-6)
    _within(out, want, U * want.abs() + 2.0**-19 * mass, "q")
    kept = (slots >= 0) & (slots < pages * page)
    p, r = slots[kept] // page, slots[kept] % page
    for i, (x, what) in enumerate(((O.norm_rope(k, w[1], cos, sin, pos, 1e-6), "k"), ((v.double(), v.double().abs()), "v"))):
        want, mass = x[0][kept], x[1][kept]
        got = cache[i].cpu().to(torch.float32)[p, :, r].double()
        if fp8:
            scale = cache[2 + i].cpu()[p, :, r].double()
            top = want.abs().amax(-1) / 448
            _within(scale, top, 2.0**-18 * (top + mass.amax(-1) / 448), what + " scale")
            got = got * scale[..., None]
            _within(got, want, 2.0**-4 * want.abs() + 2.0**-10 * scale[..., None] + 2.0**-18 * mass, what)
        else:
            _within(got, want, U * want.abs() + 2.0**-19 * mass, what)
    untouched = torch.ones(pages * page, dtype=torch.bool)
    untouched[slots[kept]] = False
    for x, y in zip(cache, before):
        if x is not None:
            x, y = (z.view(torch.uint8).cpu().transpose(1, 2).reshape(pages * page, -1) if z.dim() == 4 else z.view(I32).cpu().transpose(1, 2).reshape(pages * page, -1) for z in (x, y))
            assert torch.equal(x[untouched], y[untouched]), "rows of nobody were written"


def test_append_is_the_training_prologue(gpu):
    """The same bits as qk_norm_rope, which the layer was trained with."""
    from pithtrain_amd.operators.norm_rope import qk_norm_rope

    g = torch.Generator().manual_seed(20)
    t, h, hkv, d = 37, 32, 4, 128
    q, k, v = (torch.randn(t, n, d, generator=g).to(BF).to(gpu) for n in (h, hkv, hkv))
    w = [(1 + 0.2 * torch.randn(d, generator=g)).to(BF).to(gpu) for _ in range(2)]
    cos, sin = (x.to(gpu) for x in _tables(d))
    with torch.no_grad():
        want_q, want_k = qk_norm_rope(q[None], k[None], *w, cos[None, :t], sin[None, :t], 1e-6)
    cache = K.KVCache.empty(2, hkv, d, 64, device=gpu)
    at = torch.arange(t, device=gpu)
    got = K.kv_cache_append(q, k, v, *w, cos, sin, at, at, cache, 1e-6)
    step = 2.0**-7  # the sums of squares may be added in another order: at most a step of bf16 apart
    _within(got, want_q[0], step * want_q[0].abs(), "q")
    _within(cache.k[0, :, :t].transpose(0, 1), want_k[0], step * want_k[0].abs(), "k")
    assert torch.equal(cache.v[0, :, :t].transpose(0, 1), v)


def test_append_in_place_and_copied(gpu):
    """Rows off the alignment and tables that are not contiguous are copied."""
    g = torch.Generator().manual_seed(21)
    t, h, hkv, d = 6, 4, 2, 64
    q, k, v = (torch.randn(t, n, d, generator=g).to(BF).to(gpu) for n in (h, hkv, hkv))
    cos, sin = (x.to(gpu) for x in _tables(d))
    at = torch.arange(t, device=gpu)
    caches = [K.KVCache.empty(1, hkv, d, 16, device=gpu) for _ in range(2)]
    want = K.kv_cache_append(q, k, v, None, None, cos, sin, at, at, caches[0])
    odd = [torch.zeros(t, x.shape[1], d + 1, dtype=BF, device=gpu) for x in (q, k, v)]
    for x, y in zip(odd, (q, k, v)):
        x[..., 1:] = y
    wide = [torch.cat((x, x), 1)[:, :d] for x in (cos, sin)]
    got = K.kv_cache_append(*(x[..., 1:] for x in odd), None, None, *wide, at, at, caches[1])
    assert torch.equal(got, want) and all(torch.equal(x[:, :, :t], y[:, :, :t]) for x, y in zip(caches[0][:2], caches[1][:2]))


def test_checked_positions_and_slots(gpu, monkeypatch):
    monkeypatch.setenv("PITHTRAIN_AMD_CHECK_POSITIONS", "1")
    z = lambda *s: torch.zeros(*s, dtype=BF, device=gpu)  # noqa: E731
    cos, sin = (x.to(gpu) for x in _tables(64))
    cache = K.KVCache.empty(2, 1, 64, 16, device=gpu)
    call = lambda pos, slots: K.kv_cache_append(z(2, 1, 64), z(2, 1, 64), z(2, 1, 64), None, None, cos, sin, torch.tensor(pos, device=gpu), torch.tensor(slots, device=gpu), cache)  # noqa: E731
    call([0, 49], [-1, 31])
    with pytest.raises(AssertionError, match="positions"):
        call([0, 50], [0, 1])
    with pytest.raises(AssertionError, match="the cache holds 32 rows"):
        call([0, 1], [0, 32])
    with pytest.raises(AssertionError, match="same slot"):
        call([0, 1], [5, 5])


# ---------------------------------------------------------------------------------------------
# Bounds and selection


@BOTH
@pytest.mark.parametrize("heads", [(8, 2, 128), (3, 3, 64)], ids=str)
@pytest.mark.parametrize("page", [16, 64, 256])
def test_bounds_of_the_pages_that_a_step_fills(gpu, page, heads, fp8):
    counts, lengths = [1, 1, 1, 3 * page, 5, 0, 2 * page + 1], [page, page + 1, 3 * page, 3 * page, 2 * page + 2, 2 * page, 4 * page]
    b = Batch(gpu, counts, lengths, heads, page=page, fp8=fp8, seed=page)
    bounds = torch.full_like(b.cache.empty_bounds(), 3.0)
    K.kv_page_bounds(b.cache, bounds, b.table, b.lens, b.cu_q, sum(counts))
    filled = torch.zeros(len(bounds), dtype=torch.bool)
    for i, (n, length) in enumerate(zip(counts, lengths)):
        for j in range((length - n) // page, length // page):
            if (j + 1) * page > length - n:
                p = int(b.table[i, j])
                filled[p] = True
                k = b.kv[0][p].float() if b.scales[0] is None else b.kv[0][p].float() * b.scales[0][p][..., None]
                assert torch.equal(bounds[p].cpu(), torch.stack((k.amin(1), k.amax(1)), 1).to(BF).cpu()), (i, j)
    assert 5 <= filled.sum() < len(bounds) and (bounds[~filled.to(gpu)] == 3).all()
    if not fp8:
        p = int(b.table[0, 0])
        b.kv[0][p, 0, 3, 5], b.kv[0][p, 0, 4, 6] = math.nan, math.inf
        K.kv_page_bounds(b.cache, bounds, b.table, b.lens, b.cu_q, sum(counts))
        assert torch.isnan(bounds[p, 0, :, 5]).all() and bounds[p, 0, 1, 6] == math.inf and torch.isfinite(bounds[p, 0, 0, 6])


def _selection(gpu, lengths, heads, keep, counts=None, page=16, seed=0, bounds=None, extra=0):
    counts = counts or [1] * len(lengths)
    b = Batch(gpu, counts, [1] * len(lengths), heads, page=page, seed=seed, extra_tokens=extra)
    g = torch.Generator().manual_seed(seed + 1)
    width, (h, hkv, d) = max(-(-n // page) for n in lengths) + 2, heads
    pages = len(lengths) * width
    table = torch.randperm(pages, generator=g).to(I32).view(len(lengths), width)
    if bounds is None:
        x = torch.randn(pages, hkv, 2, d, generator=g)
        bounds = torch.stack((x.amin(2), x.amax(2)), 2).to(BF)
    lens = torch.tensor(lengths, dtype=I32, device=gpu)
    cu_q = None if all(n == 1 for n in counts) and not extra else b.cu_q
    chosen, rows = K.kv_select_pages(b.q, bounds.to(gpu), table.to(gpu), lens, cu_q, page, keep)
    chosen, rows, t = chosen.cpu(), rows.cpu(), 0
    for i, (n, length) in enumerate(zip(counts, lengths)):
        for k in range(n):
            visible = max(length - n + k + 1, 0)
            want = O.select(b.q[t].cpu(), bounds[table[i].long()], visible, page, keep)
            for j in range(hkv):
                assert chosen[t, j].tolist() == table[i][want[j]].tolist() + [-1] * (keep - len(want[j])), (t, j)
                assert int(rows[t, j]) == visible - (-(-visible // page) - len(want[j])) * page
            t += 1
    assert (chosen[t:] == -1).all() and (rows[t:] == 0).all()


@pytest.mark.parametrize("keep", [1, 2, 5, 64, 300])
@pytest.mark.parametrize("heads", [(8, 2, 128), (3, 3, 64), (32, 2, 64), (5, 1, 128)], ids=str)
def test_selected_pages_are_the_oracles(gpu, heads, keep):
    _selection(gpu, [1, 16, 17, 16 * 66, 16 * 200 + 3, 0], heads, keep, seed=keep)


def test_selection_for_drafts_and_padding(gpu):
    _selection(gpu, [300, 33, 4, 600], (4, 2, 64), 4, counts=[3, 20, 6, 1], seed=5, extra=3)


def test_selection_from_more_pages_than_stay_in_lds(gpu):
    _selection(gpu, [16 * 9001 + 5, 16 * 8193], (2, 1, 64), 77, seed=6)


@pytest.mark.parametrize("heads, counts, lengths, extra", [
    ((4, 2, 128), [7] * 40 + [0, 1, 20, 0], [16 * (270 + i) + i for i in range(40)] + [5, 16 * 300, 16 * 310 + 3, 0], 5), ((6, 1, 64), [600], [16 * 700 + 9], 0), ((3, 3, 64), [2] * 200, [16 * 260 + i for i in range(200)], 1)],
    ids=["drafts", "prompt", "pairs"])  # fmt: skip
def test_selection_where_bounds_serve_several_tokens(gpu, heads, counts, lengths, extra):
    _selection(gpu, lengths, heads, 9, counts=counts, seed=11, extra=extra)


def test_selection_from_the_widest_tables(gpu):
    _selection(gpu, [16 * 16382, 16 * 2048, 7], (2, 1, 64), 30, seed=12)


def test_selection_reads_slices_and_bounds_of_one_layer_of_several(gpu):
    g = torch.Generator().manual_seed(13)
    b = Batch(gpu, [1, 3], [16 * 300, 16 * 280 + 5], (4, 2, 64), page=16, seed=13)
    bounds = torch.randn(b.kv[0].shape[0], 3, 2, 2, 64, generator=g).sort(dim=3).values.to(BF).to(gpu)
    wide = torch.randn(4, 8, 64, generator=g).to(BF).to(gpu)
    for pages, q in ((bounds[:, 1], wide[:, 2:6]), (bounds[:, 2], b.q)):
        got = K.kv_select_pages(q, pages, b.table, b.lens, b.cu_q, 16, 20)
        want = K.kv_select_pages(q.contiguous(), pages.contiguous(), b.table, b.lens, b.cu_q, 16, 20)
        assert torch.equal(got.page_table, want.page_table) and torch.equal(got.lengths, want.lengths)


def test_equal_scores_go_to_the_pages_that_come_first(gpu):
    g = torch.Generator().manual_seed(7)
    bounds = torch.randint(0, 2, (102, 2, 2, 64), generator=g).to(BF)  # few different scores
    bounds[:, 1] = 0.5
    _selection(gpu, [16 * 100], (4, 2, 64), 30, seed=8, bounds=bounds)


def test_scores_that_are_no_numbers(gpu):
    g = torch.Generator().manual_seed(9)
    x = torch.randn(102, 1, 2, 64, generator=g)
    bounds = torch.stack((x.amin(2), x.amax(2)), 2).to(BF)
    bounds[::7, 0, :, 3] = math.nan
    bounds[1::7, 0, 1, 3] = math.inf
    bounds[2::7, 0, 0, 4] = -math.inf
    _selection(gpu, [16 * 100 - 1], (3, 1, 64), 60, seed=10, bounds=bounds)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 3.0e38])
def test_queries_that_are_no_numbers(gpu, monkeypatch, bad):
    """Their scores are infinities and NaN, those of the other head and token are not."""
    made = Batch.__init__

    def with_bad_ones(self, *args, **kw):
        made(self, *args, **kw)
        self.q[0, 1, 5] = bad
        self.q[2, 2] = bad

    monkeypatch.setattr(Batch, "__init__", with_bad_ones)
    _selection(gpu, [16 * 100 + 3, 16 * 300, 16 * 290 + 1], (4, 2, 64), 30, seed=14)


def test_sparse_attention_of_all_pages_is_the_dense_call(gpu):
    b = Batch(gpu, [1, 1, 2], [200, 90, 333], page=16, seed=15)
    bounds = b.cache.empty_bounds().zero_()
    selected = K.kv_select_pages(b.q, bounds, b.table, b.lens, b.cu_q, 16, 30)
    b.check(*K.kv_attention(b.q, b.cache, *selected, None, b.scale))


# ---------------------------------------------------------------------------------------------
# Planning


def _plan_case(gpu, counts, lengths, page, tokens, spare, width, seed=0, into=False):
    g = torch.Generator().manual_seed(seed)
    held = [-(-n // page) for n in lengths]
    pages = sum(held) + spare
    order = torch.randperm(pages, generator=g).tolist()
    table, at = [], 0
    for n in held:
        table.append(order[at : at + n] + [-9] * (width - n))
        at += n
    free = order[at:] + [-1] * sum(held)
    want = O.plan(counts, lengths, table, free, spare, page, tokens)
    i32 = lambda x: torch.tensor(x, dtype=I32, device=gpu)  # noqa: E731
    wide = torch.full((len(counts), width + 3), -4, dtype=I32, device=gpu)
    wide[:, 1 : 1 + width] = torch.tensor(table, dtype=I32).view(len(counts), width)
    tab, pool = wide[:, 1 : 1 + width], paging.PagePool(i32(free), i32([spare]))
    c, n = i32(counts), i32(lengths)
    if into:
        mk = lambda k, d=I32: torch.full((k,), 77, dtype=d, device=gpu)  # noqa: E731
        plan = paging.StepPlan(mk(len(counts) + 1), n, mk(tokens, I64), mk(tokens, I64), mk(len(counts)), pool.count)
        paging.plan_step_into(c, n, tab, pool, page, plan)
    else:
        plan = paging.plan_step(c, n, tab, pool, page, tokens)
        assert n.tolist() == lengths and pool.count.tolist() == [spare]
    for name, got in {**plan._asdict(), "page_table": tab, "free": pool.free}.items():
        assert got.tolist() == want[name], name
    assert (wide[:, 0] == -4).all() and (wide[:, 1 + width :] == -4).all()
    return want


@pytest.mark.parametrize("into", [False, True])
@pytest.mark.parametrize("b", [1, 5, 64, 300, 1500, 65, 1024, 1025])
@pytest.mark.parametrize("scarce", [False, True])
def test_plans_are_the_oracles(gpu, b, scarce, into):
    g = torch.Generator().manual_seed(b)
    rand = lambda lo, hi, n=1: torch.randint(lo, hi, (n,), generator=g).tolist()  # noqa: E731
    for page, most in ((16, 40), (64, 3)):
        lengths, counts = rand(0, 150, b), rand(-1, most, b)
        need = sum(-(-(n + max(c, 0)) // page) + (-n // page) for n, c in zip(lengths, counts))
        tokens = sum(max(c, 0) for c in counts) + 5
        want = _plan_case(gpu, counts, lengths, page, tokens, need // 3 if scarce else need + 2, 200 // page + 2, seed=b, into=into)
        assert scarce or all(x == max(c, 0) for x, c in zip(want["granted"], counts))


def test_plans_of_long_prompts(gpu):
    """Tokens in a launch of their own; a table that is too narrow; fewer tokens than the counts say; nothing at all."""
    _plan_case(gpu, [9000, 0, 3000, 7], [5, 70, 16, 64], 16, 12007, 800, 700, seed=1)
    _plan_case(gpu, [9000, 0, 3000, 7], [5, 70, 16, 64], 16, 12007, 560, 700, seed=1, into=True)
    for into in (False, True):
        _plan_case(gpu, [90 + i % 40 - 200 * (i % 7 == 6) for i in range(150)], [i % 90 for i in range(150)], 16, 14000, 900, 20, seed=4, into=into)
    want = _plan_case(gpu, [40, 17, 3], [5, 0, 16], 16, 60, 50, 2, seed=2)
    assert want["granted"] == [0, 17, 3]
    _plan_case(gpu, [20, 30, 4], [1, 2, 3], 16, 33, 50, 8, seed=3)
    _plan_case(gpu, [0, 0], [3, 0], 16, 0, 1, 1)
    _plan_case(gpu, [-1, -1, 33], [32, 31, 0], 16, 33, 0, 3)
    plan = paging.plan_step(*(torch.empty(0, dtype=I32, device=gpu) for _ in range(2)), torch.empty(0, 4, dtype=I32, device=gpu), paging.PagePool.full(3, gpu), 16, 2)
    assert plan.cu_q.tolist() == [0] and plan.slots.tolist() == [-1, -1] and plan.free_count.tolist() == [3]


@pytest.mark.parametrize("b, tokens", [(3, 5), (70, 9001), (1100, 7)])
def test_the_results_of_a_plan_lie_apart_and_aligned(gpu, b, tokens):
    i32 = lambda *s: torch.zeros(*s, dtype=I32, device=gpu)  # noqa: E731
    plan = paging.plan_step(i32(b), i32(b), i32(b, 4), paging.PagePool.full(3, gpu), 16, tokens)
    assert [tuple(t.shape) for t in plan] == [(b + 1,), (b,), (tokens,), (tokens,), (b,), (1,)]
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in plan)
    assert all(t.data_ptr() % 16 == 0 and t.is_contiguous() for t in plan) and all(x[1] <= y[0] for x, y in zip(spans, spans[1:]))


def test_nonsense_in_a_plan_stays_in_memory(gpu):
    i32 = lambda x: torch.tensor(x, dtype=I32, device=gpu)  # noqa: E731
    big = 2**31 - 1
    for count in (-5, big):
        for lengths, counts in (([big, -big, 3], [1, 2, 3]), ([big, big, big], [-1, -7, big]), ([5, 5, 5], [big, big, big]), ([big, -5, 3] * 30, [big, -1, big] * 30), ([big, 1] * 600, [-1, big] * 600)):
            table, free = torch.full((len(counts), 4), big, dtype=I32, device=gpu), torch.full((6,), -big, dtype=I32, device=gpu)
            plan = paging.plan_step(i32(counts), i32(lengths), table, paging.PagePool(free, i32([count])), 16, 9)
            assert 0 <= int(plan.free_count) <= 6 and int(plan.cu_q[-1]) <= 9
            paging.plan_step(i32(counts), i32(lengths), table, paging.PagePool(free, i32([count])), 16, 20000)
    torch.cuda.synchronize()


# ---------------------------------------------------------------------------------------------
# Together


def _answer(gpu, fp8, keep, captured=False):
    """Requests come, are answered and end, planned on the device; every token's result against dense attention to the rows that the caches hold."""
    h, hkv, d, page, pages, b, width = 8, 2, 128, 16, 40, 3, 12
    g = torch.Generator().manual_seed(30)
    cache = K.KVCache.empty(pages, hkv, d, page, L.FP8 if fp8 else BF, gpu)
    for x in cache:
        if x is not None:
            x.view(torch.uint8).fill_(0x7F)  # NaN
    bounds = cache.empty_bounds().fill_(math.nan)
    pool = paging.PagePool.full(pages, gpu)
    table, lengths = torch.full((b, width), -1, dtype=I32, device=gpu), torch.zeros(b, dtype=I32, device=gpu)
    cos, sin = (x.to(gpu) for x in _tables(d, 300))
    w = [(1 + 0.2 * torch.randn(d, generator=g)).to(BF).to(gpu) for _ in range(2)]
    history = [torch.empty(0, 0)] * b
    scale = d**-0.5
    steps = [[70, 33, 0], [1, 1, 20], [1, 1, 1], [1, -1, 1], [1, 90, 1], [3, 1, 1]] + [[1, 1, 1]] * 18
    tokens = 110
    mk = lambda n, t=I32: torch.zeros(n, dtype=t, device=gpu)  # noqa: E731
    plan = paging.StepPlan(mk(b + 1), lengths, mk(tokens, I64), mk(tokens, I64), mk(b), pool.count)
    counts = mk(b)
    qkv = torch.zeros(tokens, h + 2 * hkv, d, dtype=BF, device=gpu)

    def step():
        paging.plan_step_into(counts, lengths, table, pool, page, plan)
        return K.kv_decode(*qkv.split((h, hkv, hkv), 1), *w, cos, sin, plan.position_ids, plan.slots, cache, table, lengths, plan.cu_q, scale, bounds=bounds, keep=keep)

    graph, out = None, None
    used = 0
    for n, new in enumerate(steps):
        counts.copy_(torch.tensor(new, dtype=I32))
        qkv.copy_(torch.randn(tokens, h + 2 * hkv, d, generator=g).to(BF))
        if not captured:
            out = step()
        elif graph is None:
            graph = torch.cuda.CUDAGraph()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.graph(graph, stream=side):
                out = step()
            graph.replay()
        else:
            graph.replay()
        torch.cuda.synchronize()
        used += 1
        want_lengths = [0 if c < 0 else history[i].shape[1] + c if history[i].numel() else c for i, c in enumerate(new)]
        assert lengths.tolist() == want_lengths and plan.granted.tolist() == [max(c, 0) for c in new]
        q = O.norm_rope(qkv[:, :h].cpu(), w[0].cpu(), cos.cpu(), sin.cpu(), plan.position_ids.cpu(), 1e-6)[0]
        first = 0
        for i, c in enumerate(new):
            length = want_lengths[i]
            rows = []
            j = torch.arange(length, device=gpu)
            p, r = table[i, j // page].long(), j % page
            for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
                y = x.to(torch.float32)[p, :, r].double()
                rows.append((y if s is None else y * s[p, :, r].double()[..., None]).transpose(0, 1).cpu())
            if history[i].numel() and c >= 0:
                assert torch.equal(rows[0][:, : history[i].shape[1]], history[i]), "rows of earlier steps have changed"
            history[i] = rows[0] if length else torch.empty(0, 0)
            for k in range(max(c, 0)):
                seen = O.sees(c, length)[k : k + 1].expand(1, length).clone()
                visible = length - c + k + 1
                if keep is not None:
                    of_pages = torch.stack([torch.stack((rows[0][:, m * page : (m + 1) * page].amin(1), rows[0][:, m * page : (m + 1) * page].amax(1)), 1) for m in range(-(-visible // page))])
                    # (queries are those of the oracle, not the rounded ones: pages whose scores lie closer together than that may go either way)
                    kept = O.select(q[first + k].to(BF), of_pages.to(BF), visible, page, keep)
                for head in range(hkv):
                    mine, mask = slice(head * (h // hkv), (head + 1) * (h // hkv)), seen.clone()
                    if keep is not None:
                        mask &= torch.tensor([m // page in kept[head] for m in range(length)])
                    want, _, mass, spread = O.attention(q[first + k : first + k + 1, mine], rows[0][head : head + 1], rows[1][head : head + 1], mask, scale)
                    # q is rounded to bf16 on the way: its score is off by u sum |q k| more
                    e = ((d + 8) * 2.0**-24 + U) * spread
                    _within(out[first + k : first + k + 1, mine], want, U * want.abs() + (U + 2 * (e[..., None] * math.log(2) + 2.0**-16)) * mass, f"step {n} request {i} token {k} head {head}")
            first += max(c, 0)
    return used


@BOTH
def test_requests_that_come_and_go(gpu, fp8):
    assert _answer(gpu, fp8, None) == 24


def test_requests_that_come_and_go_over_all_their_pages(gpu):
    assert _answer(gpu, False, 12) == 24


def test_a_captured_step_follows_its_requests(gpu):
    assert _answer(gpu, False, None, captured=True) == 24


def test_a_request_without_pages_disturbs_no_other(gpu):
    """Its tokens leave no row; what the others get is what they get without it."""
    g = torch.Generator().manual_seed(33)
    cos, sin = (x.to(gpu) for x in _tables(64, 60))
    qkv = torch.randn(9, 8, 64, generator=g).to(BF).to(gpu)
    results = []
    for counts, spare in (([4, 4, 1], 3), ([4, 4, 1], 2)):
        cache = K.KVCache.empty(8, 2, 64, 16, device=gpu)
        cache.k.zero_(), cache.v.zero_()
        table = torch.tensor([[6, 7, -1], [-1, -1, -1], [5, -1, -1]], dtype=I32, device=gpu)
        pool = paging.PagePool(torch.tensor([0, 1, 2, -1, -1, -1], dtype=I32, device=gpu), torch.tensor([spare - 2], dtype=I32, device=gpu))
        lengths = torch.tensor([20, 0, 3], dtype=I32, device=gpu)
        plan = paging.plan_step(torch.tensor(counts, dtype=I32, device=gpu), lengths, table, pool, 16, 9)
        o = K.kv_decode(*qkv.split((4, 2, 2), 1), None, None, cos, sin, plan.position_ids, plan.slots, cache, table, plan.lengths, plan.cu_q, 0.125)
        results.append((plan, o, cache))
    (all_, want, _), (denied, got, cache) = results
    assert all_.granted.tolist() == [4, 4, 1] and denied.granted.tolist() == [4, 0, 1] and denied.lengths.tolist() == [24, 0, 4]
    assert (denied.slots[4:8] == -1).all() and not cache.k[:5].any()
    assert torch.equal(got[:4], want[:4]) and torch.equal(got[8:], want[8:])


def test_the_latent_cache_takes_the_same_plan(gpu):
    """Slots, positions and lengths of a plan in the MLA layer's step: the rows go where the tables say."""
    g = torch.Generator().manual_seed(31)
    page, b = 16, 2
    cache = L.LatentCache.empty(9, page, device=gpu)
    pool, table = paging.PagePool.full(9, gpu), torch.full((b, 5), -1, dtype=I32, device=gpu)
    lengths = torch.zeros(b, dtype=I32, device=gpu)
    cos, sin = (x.to(gpu) for x in _tables(64, 100))
    w = torch.ones(512, dtype=BF, device=gpu)
    rows = [torch.empty(0, 512)] * b
    for counts in ([20, 3], [1, 1], [-1, 1], [30, 15]):
        c = torch.tensor(counts, dtype=I32, device=gpu)
        n = sum(max(x, 0) for x in counts)
        plan = paging.plan_step(c, lengths, table, pool, page, n + 1)
        lengths, pool = plan.lengths, paging.PagePool(pool.free, plan.free_count)
        kv_a = torch.randn(n + 1, 576, generator=g).to(BF).to(gpu)
        L.latent_cache_append(kv_a, w, cos, sin, plan.position_ids, plan.slots, cache)
        first = 0
        normed = torch.nn.functional.rms_norm(kv_a[:, :512].double().cpu(), (512,), eps=1e-6)
        for i, x in enumerate(counts):
            rows[i] = torch.empty(0, 512) if x < 0 else torch.cat((rows[i], normed[first : first + x]))
            first += max(x, 0)
        cu_rows = torch.cat((torch.zeros(1, dtype=I32, device=gpu), lengths.cumsum(0).to(I32)))
        got, _ = L.latent_cache_gather(cache, table, cu_rows, int(cu_rows[-1]))
        want = torch.cat(rows)
        _within(got, want, U * want.abs() + 2.0**-19 * want.abs(), f"{counts}")


def test_on_another_stream(gpu):
    b = Batch(gpu, [1, 1], [3000, 700], seed=16)
    want = b.attention()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [b.attention() for _ in range(5)]
        plan = paging.plan_step(torch.ones(2, dtype=I32, device=gpu), b.lens, b.table.clone(), paging.PagePool.full(3, gpu), 64, 2)
    s.synchronize()
    assert all(torch.equal(x, y) for one in got for x, y in zip(one, want)) and plan.cu_q.tolist() == [0, 1, 2]


def test_two_streams_at_once(gpu):
    """Calls in flight on two streams have workspaces of their own."""
    batches = [Batch(gpu, [1, 1, 2], [9000, 7000, 400], (8, 2, 128), page=16, seed=s) for s in (50, 51)]
    bounds = [torch.randn(b.kv[0].shape[0], 2, 2, 128, generator=torch.Generator().manual_seed(s)).sort(dim=2).values.to(BF).to(gpu) for s, b in enumerate(batches)]

    def calls(b, pages):
        selected = K.kv_select_pages(b.q, pages, b.table, b.lens, b.cu_q, 16, 40)
        return [*b.attention(), *selected, *K.kv_attention(b.q, b.cache, *selected, None, b.scale)]

    want = [calls(*x) for x in zip(batches, bounds)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(calls(batches[i], bounds[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for one in got[i]:
            assert all(torch.equal(x, y) for x, y in zip(one, want[i]))


@BOTH
def test_a_captured_sparse_step_is_the_eager_one(gpu, fp8):
    """A whole step in a graph (plan, append, bounds, selection, attention to the selected pages), replayed beside the same steps run eagerly on tensors of their own."""
    h, hkv, d, page, pages, b, width, tokens, keep = 8, 2, 64, 16, 200, 3, 60, 12, 4
    g = torch.Generator().manual_seed(52)
    cos, sin = (x.to(gpu) for x in _tables(d, 1000))
    counts, qkv = torch.zeros(b, dtype=I32, device=gpu), torch.zeros(tokens, h + 2 * hkv, d, dtype=BF, device=gpu)

    class State:
        def __init__(self):
            mk = lambda n, t=I32: torch.zeros(n, dtype=t, device=gpu)  # noqa: E731
            self.cache = K.KVCache.empty(pages, hkv, d, page, L.FP8 if fp8 else BF, gpu)
            for x in self.cache:
                if x is not None:
                    x.view(torch.uint8).zero_()
            self.bounds = self.cache.empty_bounds().zero_()
            self.pool, self.table, self.lengths = paging.PagePool.full(pages, gpu), torch.full((b, width), -1, dtype=I32, device=gpu), mk(b)
            self.plan = paging.StepPlan(mk(b + 1), self.lengths, mk(tokens, I64), mk(tokens, I64), mk(b), self.pool.count)

        def step(self):
            p = self.plan
            paging.plan_step_into(counts, self.lengths, self.table, self.pool, page, p)
            return K.kv_decode(*qkv.split((h, hkv, hkv), 1), None, None, cos, sin, p.position_ids, p.slots, self.cache, self.table, self.lengths, p.cu_q, d**-0.5, bounds=self.bounds, keep=keep)

        def all(self):
            return [x for x in (*self.cache, self.bounds, *self.pool, self.table, *self.plan) if x is not None]

    eager, captured = State(), State()
    eager.step(), captured.step()  # (no tokens)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        out = captured.step()
    for new in [[4, 4, 4]] * 20 + [[1, 1, 1], [2, -1, 3], [1, 9, 1], [-1, -1, 8]] + [[1, 1, 1]] * 6:
        counts.copy_(torch.tensor(new, dtype=I32))
        qkv.copy_(torch.randn(tokens, h + 2 * hkv, d, generator=g).to(BF))
        graph.replay()
        want = eager.step()
        torch.cuda.synchronize()
        n = sum(max(c, 0) for c in new)
        assert torch.equal(out[:n], want[:n]) and int(eager.plan.cu_q[-1]) == n
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(captured.all(), eager.all())), new


@BOTH
def test_a_compiled_step_writes_the_cache(gpu, fp8):
    """The same results and the same rows in the cache as the eager step's, whose tensors the compiled one changes in place."""
    g = torch.Generator().manual_seed(53)
    qkv = torch.randn(6, 8, 64, generator=g).to(BF).to(gpu)
    w = (1 + 0.1 * torch.randn(64, generator=g)).to(BF).to(gpu)
    cos, sin = (x.to(gpu) for x in _tables(64, 60))
    counts, lengths = torch.tensor([4, 2], dtype=I32, device=gpu), torch.tensor([30, 0], dtype=I32, device=gpu)

    def step(table, free, count, bounds, *cache):
        cache = K.KVCache(*cache)
        plan = paging.plan_step(counts, lengths, table, paging.PagePool(free, count), 16, 6)
        o = K.kv_decode(*qkv.split((4, 2, 2), 1), w, w, cos, sin, plan.position_ids, plan.slots, cache, table, plan.lengths, plan.cu_q, 0.125, bounds=bounds, keep=2)
        return o, K.kv_attention(qkv[:, :4].contiguous(), cache, table, plan.lengths, plan.cu_q, 0.125)[0] * 2, plan.slots + 1

    states = []
    for _ in range(2):
        cache = K.KVCache.empty(6, 2, 64, 16, L.FP8 if fp8 else BF, gpu)
        pool = paging.PagePool.full(6, gpu)
        state = [torch.tensor([[4, 5, -1], [-1, -1, -1]], dtype=I32, device=gpu), pool.free.flip(0).contiguous(), pool.count, cache.empty_bounds(), *(x for x in cache if x is not None)]
        for x in state[3:]:
            x.view(torch.uint8).zero_()
        state[2].fill_(4)
        states.append(state)
    with torch.no_grad():
        want = step(*states[0])
        got = torch.compile(step, backend="aot_eager", fullgraph=True)(*states[1])
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and want[2].tolist() == [16 * 5 + 15, 16 * 5 + 16, 16 * 3 + 1, 16 * 3 + 2, 16 * 2 + 1, 16 * 2 + 2]
    for x, y in zip(*states):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)) and y.view(torch.uint8).any()


# ---------------------------------------------------------------------------------------------
# Far apart and long


def _apart(x, gap):
    buffer = torch.empty((x.shape[0] - 1) * gap + x[0].numel(), dtype=x.dtype, device=x.device)
    y = buffer.as_strided(x.shape, (gap, *x.stride()[1:]))
    for a, b in zip(y, x):
        a.copy_(b)
    return y


@BOTH
def test_pages_that_lie_further_apart_than_32_bits_count(gpu, fp8):
    b = Batch(gpu, [2, 1], [100, 30], (4, 2, 64), page=64, fp8=fp8, seed=54)
    far = K.KVCache(*(None if x is None else _apart(x, (1 << 30) + 64 if x.dtype == torch.float32 else (1 << 31) + 64) for x in b.cache))
    for x, y in zip(K.kv_attention(b.q, far, b.table, b.lens, b.cu_q, b.scale), b.attention()):
        assert torch.equal(x, y)
    new, table = torch.randn(3, 8, 64, generator=torch.Generator().manual_seed(55)).to(BF).to(gpu), _tables(64, 10)
    last = b.kv[0].shape[0] - 1
    slots = torch.tensor([64 * last + 63, 64 * last, 5], device=gpu)
    bounds, far_bounds = (f(b.cache.empty_bounds().zero_()) for f in (lambda x: x, lambda x: _apart(x, (1 << 31) + 64)))
    pages, lens = torch.tensor([[last]], dtype=I32, device=gpu), torch.tensor([64], dtype=I32, device=gpu)
    for cache, edges in ((b.cache, bounds), (far, far_bounds)):
        K.kv_cache_append(*new.split((4, 2, 2), 1), None, None, *(x.to(gpu) for x in table), torch.arange(3, device=gpu), slots, cache)
        K.kv_page_bounds(cache, edges, pages, lens, None, 1)
    for x, y in zip((*b.cache, bounds), (*far, far_bounds)):
        assert x is None or torch.equal(x.view(torch.uint8), y.contiguous().view(torch.uint8))
    assert bounds[last].any() and not bounds[:last].any()
    wide = torch.arange(last, -1, -1, dtype=I32, device=gpu).repeat(1, 80)[:, :300].contiguous()
    finite = bounds.clone().copy_(torch.randn(bounds.shape, generator=torch.Generator().manual_seed(56)).sort(dim=2).values)
    far_bounds.copy_(finite)
    lens.fill_(64 * wide.shape[1])
    for x, y in zip(*(K.kv_select_pages(b.q[:1], x, wide, lens, None, 64, 30) for x in (finite, far_bounds))):
        assert torch.equal(x, y)
    del far, far_bounds, cache, edges, x, y
    torch.cuda.empty_cache()


def _repeated(gpu, page, entries, heads, seed):
    """One sequence whose table names the pages of another again and again: every row counts as often."""
    b = Batch(gpu, [1], [page * 2], heads, page=page, fp8=True, seed=seed)
    table, times = b.table[:, :2].repeat(1, entries // 2), entries // 2
    lens = torch.tensor([2 * page * times], dtype=I32, device=gpu)
    o, lse = K.kv_attention(b.q, b.cache, table, lens, None, b.scale)
    want, want_lse, mass, spread = O.attention(b.q.cpu(), *b.rows(b.table[0], 2 * page), O.sees(1, 2 * page, None), b.scale)
    e = (b.d + 8) * 2.0**-24 * spread
    # sums of n rows on top. A row's keys are dealt to 256 workgroups of four waves at least, and a lane adds the weights of 8 of 32 of them: n / 4096 steps, each off by
    # 2^-24 of a sum that never exceeds the whole; the products take 32 keys a step, with four roundings at most: n / 8192. Then 2048 such sums meet.
    n = 2 * page * times
    more = (n / 4096 + 2048) * 2.0**-24
    _within(o, want, U * want.abs() + (U + 2 * (e[..., None] * math.log(2) + 2.0**-16 + more)) * mass, "o")
    _within(lse, want_lse + math.log2(times), e.T + 2.0**-17 + 2 * more, "lse")


def test_a_page_that_a_table_names_again_and_again(gpu):
    _repeated(gpu, 16, 1 << 17, (8, 2, 64), 57)


def test_the_longest_sequence(gpu):
    """Almost 2^31 rows."""
    _repeated(gpu, 1 << 16, 32766, (4, 1, 64), 58)


def test_a_captured_call_follows_lengths_and_tables(gpu):
    b = Batch(gpu, [1, 2, 1], [40, 300, 1000], seed=17, page=16)
    want = b.attention()  # (the first call of a kind is not in the graph)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        got = b.attention()
    for lengths in ([40, 300, 1000], [1, 2, 999], [33, 290, 16], [40, 300, 1000]):
        b.lens.copy_(torch.tensor(lengths, dtype=I32))
        graph.replay()
        torch.cuda.synchronize()
        b.lengths = lengths
        b.check(*got, str(lengths))
        assert all(torch.equal(x, y) for x, y in zip(got, b.attention()))
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_what_an_operator_writes_counts_as_changed(gpu):
    b = Batch(gpu, [1], [64], (4, 2, 64), seed=18)
    bounds, cos = b.cache.empty_bounds(), torch.ones(80, 64, dtype=BF, device=gpu)
    one = torch.zeros(1, dtype=I64, device=gpu)
    versions = [x._version for x in (b.kv[0], b.kv[1], bounds, b.table)]
    K.kv_cache_append(b.q, b.q[:, :2], b.q[:, :2], None, None, cos, cos, one, one, b.cache)
    K.kv_page_bounds(b.cache, bounds, b.table, b.lens, b.cu_q, 1)
    paging.plan_step(torch.ones(1, dtype=I32, device=gpu), b.lens, b.table, paging.PagePool.full(3, gpu), 64, 1)
    assert all(x._version > v for x, v in zip((b.kv[0], b.kv[1], bounds, b.table), versions))


def test_empty_calls(gpu):
    b = Batch(gpu, [1], [64], (4, 2, 64), seed=19)
    none = lambda *s, d=BF: torch.empty(*s, dtype=d, device=gpu)  # noqa: E731
    o, lse = K.kv_attention(b.q[:0], b.cache, b.table, b.lens, torch.zeros(2, dtype=I32, device=gpu), b.scale)
    assert o.shape == (0, 4, 64) and lse.shape == (4, 0)
    K.kv_attention(b.q[:0], b.cache, b.table[:0], b.lens[:0], None, b.scale)
    assert K.kv_cache_append(b.q[:0], b.q[:0, :2], b.q[:0, :2], None, None, none(4, 64), none(4, 64), none(0, d=I64), none(0, d=I64), b.cache).shape == (0, 4, 64)
    selected = K.kv_select_pages(b.q, b.cache.empty_bounds(), b.table[:0], b.lens[:0], torch.zeros(1, dtype=I32, device=gpu), 64, 3)
    assert (selected.page_table == -1).all() and (selected.lengths == 0).all()


# ---------------------------------------------------------------------------------------------
# Refusals


def test_wrong_arguments_are_refused(gpu):
    b = Batch(gpu, [1, 2], [40, 50], (4, 2, 64), page=16, seed=40)
    before = [x.clone() for x in b.kv]
    z = lambda *s, d=BF: torch.zeros(*s, dtype=d, device=gpu)  # noqa: E731
    k, v = b.kv
    call = lambda **kw: K.kv_attention(*{**dict(q=b.q, c=b.cache, t=b.table, l=b.lens, cu=b.cu_q, s=0.1, m=None), **kw}.values())  # noqa: E731
    for match, kw in [
        ("q must be", dict(q=b.q.float())), ("q must be", dict(q=b.q[..., :32])), ("cu_q must be", dict(cu=b.cu_q[:2])), ("cu_q must be", dict(cu=b.cu_q.long())),
        ("lengths must be", dict(l=b.lens.long())), ("page_table must be", dict(t=b.table[:1])), ("page_table must be", dict(t=b.table.long())), ("tree_mask must be", dict(m=z(2, d=I64))),
        ("one token a sequence", dict(cu=None)), ("does not match cache.k", dict(c=K.KVCache(k, v[1:]))), ("does not match cache.k", dict(c=K.KVCache(k, v.to(L.FP8)))),
        ("has no scales", dict(c=K.KVCache(k, v, z(*k.shape[:3], d=torch.float32)))), ("needs a float32", dict(c=K.KVCache(k.to(L.FP8), v.to(L.FP8)))),
        ("is not contiguous", dict(c=K.KVCache(k.transpose(1, 2).contiguous().transpose(1, 2), v))), ("64 or 128", dict(c=K.KVCache(z(2, 2, 16, 96), z(2, 2, 16, 96)))),
        ("lengths must be", dict(q=b.q[:2], t=z(2, 2, 3, d=I32), l=z(2, 3, d=I32), cu=None)), ("page_table must be", dict(q=b.q[:2], t=z(2, 1, 3, d=I32), l=z(2, 2, d=I32), cu=None)),
        ("no cu_q", dict(t=z(2, 2, 3, d=I32), l=z(2, 2, d=I32))), ("one page table for all", dict(q=b.q[:2], t=z(2, 2, 3, d=I32), l=z(2, 2, d=I32), cu=None, m=z(2, d=I64))),
    ]:  # fmt: skip
        with pytest.raises(AssertionError, match=match):
            call(**kw)
    for match, kw in [("page size", dict(c=K.KVCache(k[:, :, :8].contiguous(), v[:, :, :8].contiguous()))), ("empty page table", dict(t=b.table[:, :0])), ("query heads", dict(q=z(3, 3, 64)))]:
        with pytest.raises(_C.PithError, match=match):
            call(**kw)
    with pytest.raises(RuntimeError, match="different devices|need tensors on a GPU"):
        call(l=b.lens.cpu())
    with pytest.raises(AssertionError, match="wrong dtype or shape"):
        K.kv_attention_into(b.q, b.cache, b.table, b.lens, b.cu_q, 0.1, None, torch.empty_like(b.q), z(4, 2, d=torch.float32))

    new = dict(q=z(3, 4, 64), k=z(3, 2, 64), v=z(3, 2, 64), qw=z(64), kw=z(64), cos=z(8, 64), sin=z(8, 64), p=z(3, d=I64), s=z(3, d=I64), c=b.cache)
    for match, kw in [("k must be", dict(k=z(3, 4, 64))), ("v has 2 tokens", dict(v=z(2, 2, 64))), ("given together", dict(qw=None)), ("tensors of one dtype", dict(qw=z(32))),
                      ("tensors of one dtype", dict(qw=z(64, d=torch.float32))), ("cos and sin must be", dict(cos=z(8, 32), sin=z(8, 32))), ("slots must be", dict(s=z(3, d=I32))), ("position_ids must be", dict(p=z(2, d=I64)))]:  # fmt: skip
        with pytest.raises(AssertionError, match=match):
            K.kv_cache_append(*{**new, **kw}.values())
    with pytest.raises(TypeError):
        K.kv_cache_append(*{**new, "qw": z(64, d=torch.float16), "kw": z(64, d=torch.float16)}.values())

    bounds = b.cache.empty_bounds()
    for match, kw in [("bounds must be", dict(b=bounds[1:])), ("bounds must be", dict(b=bounds.float())), ("page_table must be", dict(t=b.table[:1])), ("tokens = -1", dict(n=-1)), ("one token a sequence", dict(cu=None, n=3))]:
        with pytest.raises(AssertionError, match=match):
            K.kv_page_bounds(*{**dict(c=b.cache, b=bounds, t=b.table, l=b.lens, cu=b.cu_q, n=3), **kw}.values())
    select = lambda **kw: K.kv_select_pages(*{**dict(q=b.q, b=bounds, t=b.table, l=b.lens, cu=b.cu_q, p=16, k=2), **kw}.values())  # noqa: E731
    for match, kw in [("bounds must be", dict(b=bounds[..., :32])), ("q must be", dict(q=b.q.float())), ("keep = 0", dict(k=0)), ("page_table must be", dict(l=b.lens[:1]))]:  # (b is what lengths say)
        with pytest.raises(AssertionError, match=match):
            select(**kw)
    for match, kw in [("page size", dict(p=24)), ("query heads", dict(q=z(3, 3, 64))), ("at most 16384", dict(t=z(2, 16385, d=I32)))]:
        with pytest.raises(_C.PithError, match=match):
            select(**kw)
    for kw in (dict(keep=2), dict(keep=2, bounds=bounds, tree_mask=z(3, d=I64))):
        with pytest.raises(AssertionError, match="keep needs bounds"):
            K.kv_decode(*new.values(), b.table, b.lens, b.cu_q, 0.1, **kw)

    plan = dict(c=z(2, d=I32), l=z(2, d=I32), t=z(2, 3, d=I32), pool=paging.PagePool.full(4, gpu), p=16, n=3)
    for match, kw in [("counts must be", dict(c=z(2, d=I64))), ("lengths must be", dict(l=z(3, d=I32))), ("page_table must be", dict(t=z(3, 3, d=I32))), ("tokens = -1", dict(n=-1)),
                      ("pool.count must be", dict(pool=paging.PagePool(z(4, d=I32), z(2, d=I32)))), ("pool.free must be", dict(pool=paging.PagePool(z(8, d=I32)[::2], z(1, d=I32))))]:  # fmt: skip
        with pytest.raises(AssertionError, match=match):
            paging.plan_step(*{**plan, **kw}.values())
    with pytest.raises(_C.PithError, match="page size"):
        paging.plan_step(*{**plan, "p": 24}.values())
    torch.cuda.synchronize()
    assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip(before, b.kv))
