"""The latent cache's operators on the GPU against the fp64 oracle, through the public entry points.

Bounds are elementwise and come from the arithmetic, u = 2^-8 being bf16's half step relative to the value (torch.finfo(bfloat16).eps / 2):

  a result rounded once from fp32         u |want|, and 2^-20 |want| for the fp32 steps before it
  a sum of K products in fp32             K 2^-24 sum |a b| on top (K = 128 and 512; exact products)
  e4m3 rows                               2^-4 |want| of the value, but half of its finest step, 2^-10, times the row's scale at least
  attention                               the weights P (times the row's scale) are rounded to bf16: u sum P |c|. A score's sum of 576 products is off by
                                          at most d = 584 2^-24 (sum of their absolute values, in bits), its exp2, the subtraction of the maximum and the
                                          rescaling by 2^-16 in all: weight and denominator 2 (d ln 2 + 2^-16) sum P |c|. And u |want| for the result.
  lse                                     d + 2^-17 bits (|lse| < 64: its own step is 2^-18)
"""

import math
import sys

import pytest
import torch

from oracle import latent_oracle as O
from oracle import prologue_oracle as P
from pithtrain_amd import _C
from pithtrain_amd.operators.mla import MLA
from pithtrain_amd.operators.mla import latent as L

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
U = 2.0**-8
SCALE = 192**-0.5
I32, I64 = torch.int32, torch.int64


def _within(got, want, bound, what):
    got, want, bound = got.double().cpu(), want.double().cpu(), bound.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)), f"{what}: finite and non-finite values elsewhere than expected"
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine], want[~fine]), f"{what}: other infinities"
    over = ((got - want).abs() - bound)[fine]
    assert over.numel() == 0 or over.max() <= 0, f"{what}: off by {((got - want).abs() / bound.clamp_min(1e-300))[fine].max():.3f} times the bound"


MIN_WIDTH = 0  # of page tables: blocks of 64 query rows are for those that are wide


class Batch:
    """Sequences in a cache. counts: new tokens of each, lengths: cached rows of each. Everything that no sequence owns (rows behind the last one of a
    page, pages of nobody, table entries that are not needed) holds NaN or nonsense."""

    def __init__(self, dev, counts, lengths, h, page=64, fp8=False, tree=None, seed=0, extra_tokens=0, q_std=0.6):
        g = torch.Generator().manual_seed(seed)
        mk = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.counts, self.lengths, self.h, self.dev, self.page = counts, lengths, h, dev, page
        t = sum(counts) + extra_tokens
        need = [-(-n // page) for n in lengths]
        pages, width = sum(need) + 3, max(max(need), 1, MIN_WIDTH) + 1
        order = torch.randperm(pages, generator=g)
        table = torch.randint(-5, 2 * pages, (len(counts), width), generator=g).to(I32)  # entries behind a sequence's pages are never followed
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = order[at : at + n]
            at += n
        latent = torch.full((pages, page, 512), math.nan)
        k_pe = torch.full((pages, page, 64), math.nan)
        for i, n in enumerate(lengths):
            j = torch.arange(n)
            latent[table[i, j // page].long(), j % page] = mk(n, 512) * (0.5 + torch.rand(512, generator=g))
            k_pe[table[i, j // page].long(), j % page] = 2 * mk(n, 64)
        self.scale = None
        if fp8:
            self.scale = latent.abs().amax(-1) / 448
            latent = (latent / self.scale[..., None]).clamp(-448, 448).to(L.FP8)
            self.scale = self.scale.to(dev)
        else:
            latent = latent.to(BF)
        self.latent, self.k_pe, self.table = latent.to(dev), k_pe.to(BF).to(dev), table.to(dev)
        self.q_latent, self.q_pe = (q_std * mk(t, h, 512)).to(BF).to(dev), mk(t, h, 64).to(BF).to(dev)
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
        return L.LatentCache(self.latent, self.k_pe, self.scale)

    def rows(self, i):
        """Rows of sequence i at the values they hold."""
        j = torch.arange(self.lengths[i], device=self.dev)
        p, r = self.table[i, j // self.page].long(), j % self.page
        c = self.latent.to(torch.float32)[p, r].double() * (1.0 if self.scale is None else self.scale[p, r].double()[:, None])
        return c.cpu(), self.k_pe[p, r].double().cpu()

    def attention(self, words="own"):
        return L.latent_attention(self.q_latent, self.q_pe, self.cache, self.table, self.lens, self.cu_q, SCALE, self.words if words == "own" else words)

    def check(self, o, lse, what=""):
        o, lse, first = o.cpu(), lse.cpu(), 0
        for i, (n, length) in enumerate(zip(self.counts, self.lengths)):
            sl = slice(first, first + n)
            first += n
            if n == 0:
                continue
            c, p = self.rows(i)
            seen = O.sees(n, length, None if self.words is None else self.words[sl].tolist())
            want, want_lse, mass, spread = O.attention(self.q_latent[sl].cpu(), self.q_pe[sl].cpu(), c, p, seen, SCALE)
            d = 584 * 2.0**-24 * spread
            _within(o[sl], want, U * want.abs() + (U + 2 * (d[..., None] * math.log(2) + 2.0**-16)) * mass, f"{what} o of sequence {i}")
            _within(lse[:, sl], want_lse, d.T + 2.0**-17, f"{what} lse of sequence {i}")


LENGTH_SETS = {
    "one_row": ([1], [1]),
    "tiny": ([1, 1, 1, 1, 1], [1, 15, 16, 17, 31]),
    "tile_ends": ([1] * 6, [32, 33, 63, 64, 65, 96]),
    "ordinary": ([1, 1, 1], [517, 1, 1301]),
    "none": ([1, 0, 1, 0], [0, 70, 40, 0]),
    "few_tokens": ([2, 3, 1, 5], [2, 64, 700, 37]),
    "prompt": ([70, 33], [70, 129]),
    "contradiction": ([4, 3], [2, 0]),  # more new tokens than rows: the first of them see nothing
}


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("h", [16, 5])
@pytest.mark.parametrize("name", LENGTH_SETS)
def test_attention_matches_the_oracle(gpu, name, h, fp8):
    counts, lengths = LENGTH_SETS[name]
    b = Batch(gpu, counts, lengths, h, page=16 if name in ("tiny", "prompt") else 64, fp8=fp8, seed=len(name))
    b.check(*b.attention(), name)


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("h", [1, 128, 23])
def test_attention_of_other_head_counts(gpu, h, fp8):
    b = Batch(gpu, [1, 2], [333, 90], h, page=32, fp8=fp8, seed=h)
    b.check(*b.attention())


@pytest.mark.parametrize("page", [16, 32, 128, 1024])
def test_attention_page_sizes(gpu, page):
    b = Batch(gpu, [1, 3], [page + 5, 2 * page], 4, page=page, seed=page)
    b.check(*b.attention())


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
def test_attention_of_one_long_sequence_is_joined_from_many_parts(gpu, fp8):
    b = Batch(gpu, [1, 1], [20011, 3], 16, fp8=fp8, seed=3, q_std=1.5)
    b.check(*b.attention())


def test_attention_of_more_sequences_than_a_wavefront_scans_at_once(gpu):
    g = torch.Generator().manual_seed(4)
    counts = torch.randint(0, 3, (150,), generator=g).tolist()
    lengths = [max(n, int(x)) for n, x in zip(counts, torch.randint(0, 200, (150,), generator=g))]
    b = Batch(gpu, counts, lengths, 4, page=16, seed=5)
    b.check(*b.attention())


def test_large_scores_do_not_overflow(gpu):
    b = Batch(gpu, [1, 2], [300, 65], 16, seed=6, q_std=60.0)
    o, lse = b.attention()
    assert torch.isfinite(o.float()).all() and lse.abs().max() > 500
    # lse is in the hundreds here: its bound grows with it (one more rounding of 2^-24 |lse|)
    first = 0
    for i, (n, length) in enumerate(zip(b.counts, b.lengths)):
        c, p = b.rows(i)
        sl = slice(first, first + n)
        want, want_lse, mass, spread = O.attention(b.q_latent[sl].cpu(), b.q_pe[sl].cpu(), c, p, O.sees(n, length), SCALE)
        d = 584 * 2.0**-24 * spread + 2.0**-22 * want_lse.T.abs()
        _within(o[sl], want, U * want.abs() + (U + 2 * (d[..., None] * math.log(2) + 2.0**-16)) * mass, "o")
        _within(lse[:, sl], want_lse, d.T + 2.0**-17, "lse")
        first += n


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("kind", ["tree", "holes"])
@pytest.mark.parametrize("counts,lengths,h", [([1], [1], 16), ([8, 8], [517, 8], 16), ([64, 1, 33], [64, 300, 1000], 3), ([7, 0, 12], [40, 5, 12], 16), ([64], [63], 2)])
def test_tree_attention_matches_the_oracle(gpu, counts, lengths, h, kind, fp8):
    b = Batch(gpu, counts, lengths, h, page=16, fp8=fp8, tree=kind, seed=sum(counts) + h)
    o, lse = b.attention()
    b.check(o, lse, kind)
    if kind == "holes" and lengths == [1]:
        assert (o == 0).all() and (lse == -math.inf).all()


def test_a_chain_of_drafts_is_the_causal_call(gpu):
    b = Batch(gpu, [5, 9], [200, 60], 16, seed=8)
    words = torch.cat([L.tree_mask_of(torch.arange(-1, n - 1)) for n in b.counts]).to(gpu)
    for x, y in zip(b.attention(), b.attention(words)):
        assert torch.equal(x, y)


def test_words_of_trees_on_the_device(gpu, monkeypatch):
    """The same words as on the host, also for parents that are no drafts of their tree."""
    monkeypatch.delenv("PITHTRAIN_AMD_CHECK_POSITIONS", raising=False)
    g = torch.Generator().manual_seed(18)
    for n in (1, 3, 64):
        parents = torch.stack([torch.tensor([int(torch.randint(-1, max(i, 1), (1,), generator=g)) if i else -1 for i in range(n)]) for _ in range(5)])
        parents[2, ::3] = 2**40
        parents[3, ::2] = n
        words = L.tree_mask_of(parents)
        assert torch.equal(L.tree_mask_of(parents.to(gpu)).cpu(), words)
    monkeypatch.setenv("PITHTRAIN_AMD_CHECK_POSITIONS", "1")
    with pytest.raises(AssertionError, match="the tree has 64 drafts"):
        L.tree_mask_of(parents.to(gpu))


@pytest.mark.parametrize("tree", [None, "tree"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_row_that_a_token_does_not_see_cannot_reach_it(gpu, bad, tree):
    """The newest row of a sequence holds infinities or NaN: tokens that do not see it are computed as ever."""
    b = Batch(gpu, [6, 6], [70, 6], 16, page=16, seed=9, tree=tree)
    want_o, want_lse = b.attention()
    blind = torch.ones(12, dtype=torch.bool)
    for i in range(2):
        j = b.lengths[i] - 1
        page, row = b.table[i, j // 16].long(), j % 16
        b.latent[page, row, 100:] = bad
        b.k_pe[page, row] = bad
        blind[6 * i + 5] = False
        if tree:
            blind[6 * i : 6 * i + 6] = (b.words[6 * i : 6 * i + 6].cpu() >> 5) & 1 == 0
    assert 2 <= blind.sum() < 12
    o, lse = b.attention()
    assert torch.equal(o[blind], want_o[blind]) and torch.equal(lse[:, blind], want_lse[:, blind])
    assert torch.isnan(o[~blind].float()).any()


@pytest.mark.parametrize("h", [16, 40])
@pytest.mark.parametrize("bad", ["latent", "scale", "infinite scale"])
def test_a_row_of_e4m3_that_a_token_does_not_see_cannot_reach_it(gpu, bad, h):
    b = Batch(gpu, [3, 3], [70, 3], h, page=16, fp8=True, seed=13)
    want_o, want_lse = b.attention()
    for i in range(2):
        j = b.lengths[i] - 1
        page, row = b.table[i, j // 16].long(), j % 16
        if bad == "latent":
            b.latent.view(torch.uint8)[page, row, 40:] = 0x7F
        else:
            b.scale[page, row] = math.nan if bad == "scale" else math.inf
    blind = torch.tensor([True, True, False] * 2)
    o, lse = b.attention()
    assert torch.equal(o[blind], want_o[blind]) and torch.equal(lse[:, blind], want_lse[:, blind])
    assert torch.isnan(o[~blind].float()).any()


@pytest.mark.parametrize("h", [16, 40])
@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
def test_a_single_draft_that_does_not_see_itself_is_not_reached_by_its_row(gpu, fp8, h):
    b = Batch(gpu, [1, 1], [90, 1], h, page=16, fp8=fp8, tree="tree", seed=14)
    b.words.zero_()
    want_o, want_lse = b.attention()
    b.check(want_o, want_lse)
    for i in range(2):
        j = b.lengths[i] - 1
        page, row = b.table[i, j // 16].long(), j % 16
        b.latent[page, row] = math.nan
        b.k_pe[page, row] = math.nan
    o, lse = b.attention()
    assert torch.equal(o, want_o) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("name", LENGTH_SETS)
@pytest.mark.parametrize("h", [16, 37])
def test_blocks_of_64_rows_match_the_oracle(gpu, monkeypatch, name, h, fp8):
    monkeypatch.setattr(sys.modules[__name__], "MIN_WIDTH", 2048)
    test_attention_matches_the_oracle(gpu, name, h, fp8)


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("kind", ["tree", "holes"])
@pytest.mark.parametrize("counts,lengths,h", [([1], [1], 40), ([8, 8], [517, 8], 16), ([64, 1, 33], [64, 300, 1000], 3), ([7, 0, 12], [40, 5, 12], 16), ([64], [63], 2)])
def test_trees_in_blocks_of_64_rows_match_the_oracle(gpu, monkeypatch, counts, lengths, h, kind, fp8):
    monkeypatch.setattr(sys.modules[__name__], "MIN_WIDTH", 4096)
    test_tree_attention_matches_the_oracle(gpu, counts, lengths, h, kind, fp8)


# One row block over many workgroups; row blocks that are cut wherever the ranges end; more sequences than a wavefront scans at once.
@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("counts,lengths,h", [([4, 1], [20011, 3], 16), ([63], [3001], 128), ([2, 0, 1] * 40, list(range(7, 127)), 24)])
def test_work_lists_of_blocks_of_64_rows(gpu, monkeypatch, counts, lengths, h, fp8):
    monkeypatch.setattr(sys.modules[__name__], "MIN_WIDTH", 2048)
    b = Batch(gpu, counts, lengths, h, page=16, fp8=fp8, seed=15, q_std=1.0)
    b.check(*b.attention())


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("tree", [None, "tree"])
def test_blocks_of_64_rows_are_not_reached_by_rows_that_they_do_not_see(gpu, monkeypatch, bad, tree):
    monkeypatch.setattr(sys.modules[__name__], "MIN_WIDTH", 4096)
    test_a_row_that_a_token_does_not_see_cannot_reach_it(gpu, bad, tree)


@pytest.mark.parametrize("bad", ["latent", "scale", "infinite scale"])
def test_blocks_of_64_rows_are_not_reached_by_rows_of_e4m3_that_they_do_not_see(gpu, monkeypatch, bad):
    monkeypatch.setattr(sys.modules[__name__], "MIN_WIDTH", 4096)
    test_a_row_of_e4m3_that_a_token_does_not_see_cannot_reach_it(gpu, bad, 40)
    for fp8 in (False, True):
        test_a_single_draft_that_does_not_see_itself_is_not_reached_by_its_row(gpu, fp8, 40)


# The tests below say which kernel they are about and hold that the call takes it.
def _takes(b, rows):
    c = _C.LatentCacheArgs(latent=256, k_pe=256, pages=b.latent.shape[0], page_size=b.page, latent_ps=b.page * 512, k_pe_ps=b.page * 64, dtype=_C.PITH_BF16)
    args = _C.LatentAttnArgs(cache=c, T=b.q_latent.shape[0], B=len(b.counts), H=b.h, table_width=b.table.shape[1], table_rs=b.table.shape[1])
    assert _C.lib().pith_latent_attn_rows(_C.byref(args)) == rows


WIDTHS = {16: 0, 64: 2048}  # of page tables, by the rows of the kernel that they make calls of more than 16 rows a sequence take


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("name", LENGTH_SETS)
@pytest.mark.parametrize("rows, h", [(64, 37), (64, 128), (16, 16)])
def test_either_kernel_matches_the_oracle(gpu, monkeypatch, name, rows, h, fp8):
    monkeypatch.setattr(sys.modules[__name__], "MIN_WIDTH", WIDTHS[rows])
    counts, lengths = LENGTH_SETS[name]
    b = Batch(gpu, counts, lengths, h, page=16 if name in ("tiny", "prompt") else 64, fp8=fp8, seed=len(name) + h)
    _takes(b, rows)
    b.check(*b.attention(), name)


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("rows", [16, 64])
def test_token_offsets_that_go_back_in_either_kernel(gpu, monkeypatch, rows, fp8):
    """They are taken as their maximum so far: no token belongs to two sequences. More sequences than a wavefront scans at once."""
    monkeypatch.setattr(sys.modules[__name__], "MIN_WIDTH", WIDTHS[rows])
    n, h = 70, {16: 16, 64: 150}[rows]
    b = Batch(gpu, [3, 0] + [0] * (n - 3) + [5], [40] * n, h, seed=16, fp8=fp8)
    _takes(b, rows)
    want = b.attention()
    b.check(*want)
    b.cu_q[2:-1] = torch.tensor([0, 3, 1, -7], dtype=I32, device=gpu).repeat(n)[: n - 2]
    for x, y in zip(b.attention(), want):
        assert torch.equal(x, y)


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("rows", [16, 64])
def test_nonsense_in_the_index_tensors_stays_in_memory_in_either_kernel(gpu, monkeypatch, rows, fp8):
    """Pages, lengths and token offsets out of range: clamped, whatever comes of it."""
    monkeypatch.setattr(sys.modules[__name__], "MIN_WIDTH", WIDTHS[rows])
    b = Batch(gpu, [1, 2], [100, 130], {16: 8, 64: 40}[rows], seed=11, fp8=fp8)
    _takes(b, rows)
    if fp8:
        b.latent.view(torch.uint8).fill_(0x38)  # 1.0
        b.scale.fill_(1.0)
    else:
        b.latent.nan_to_num_(0.0)
    b.k_pe.nan_to_num_(0.0)
    table, lens, cu = b.table.clone(), b.lens.clone(), b.cu_q.clone()
    b.table[:] = torch.tensor([-(2**31), -1, 2**31 - 1], dtype=I32, device=gpu)[torch.arange(b.table.shape[1], device=gpu) % 3]
    assert torch.isfinite(b.attention()[0].float()).all()
    for far in ([2**31 - 1, 2**31 - 1], [-5, -(2**31)]):
        b.lens[:] = torch.tensor(far, dtype=I32, device=gpu)
        o, lse = b.attention()
        assert torch.isfinite(o.float()).all()
    assert (o == 0).all() and (lse == -math.inf).all()
    b.lens[:] = 50
    for offsets in ([0, 2**31 - 1, 5], [-7, 3, 1], [3, 2, 1], [-(2**31), 2**31 - 1, -(2**31)]):
        b.cu_q[:] = torch.tensor(offsets, dtype=I32, device=gpu)
        b.attention()
    torch.cuda.synchronize()
    b.table.copy_(table), b.lens.copy_(lens), b.cu_q.copy_(cu)
    b.check(*b.attention())


@pytest.mark.parametrize("tree", ["tree", "holes"])
@pytest.mark.parametrize("rows", [16, 64])
def test_tokens_behind_the_last_sequence_in_either_kernel(gpu, monkeypatch, rows, tree):
    """A padded batch: the rows of tokens that belong to no sequence are left as they were, the others as in a call without them."""
    monkeypatch.setattr(sys.modules[__name__], "MIN_WIDTH", WIDTHS[rows])
    h = {16: 4, 64: 40}[rows]
    b = Batch(gpu, [2, 1], [40, 300], h, seed=10, extra_tokens=5, tree=tree)
    _takes(b, rows)
    o, lse = torch.full((8, h, 512), 7.0, dtype=BF, device=gpu), torch.full((h, 8), 7.0, device=gpu)
    L.latent_attention_into(b.q_latent, b.q_pe, b.cache, b.table, b.lens, b.cu_q, SCALE, b.words, o, lse)
    assert (o[3:] == 7).all() and (lse[:, 3:] == 7).all()
    b.check(o[:3], lse[:, :3])


# Ranges that hold several row blocks, of one sequence and of several: a prompt against itself, a batch of many single tokens.
@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("rows, counts, lengths, h", [(64, [601, 3], [700, 40], 64), (16, [1] * 1100, [1 + 37 * i % 90 for i in range(1100)], 16)], ids=["prompt", "single tokens"])
def test_more_row_blocks_than_workgroups_in_either_kernel(gpu, monkeypatch, rows, counts, lengths, h, fp8):
    monkeypatch.setattr(sys.modules[__name__], "MIN_WIDTH", WIDTHS[rows])
    b = Batch(gpu, counts, lengths, h, page=16, seed=20, fp8=fp8)
    _takes(b, rows)
    b.check(*b.attention())


def test_empty_calls_return_empty_results(gpu):
    """No tokens, no sequences, no rows: nothing is written."""
    b = Batch(gpu, [0, 0], [40, 0], 4, seed=21)
    z = lambda *s, d=BF: torch.zeros(*s, dtype=d, device=gpu)  # noqa: E731
    cos, sin = _tables(8, gpu)
    none, start = z(0, d=I64), z(1, d=I32)

    def calls():
        L.latent_cache_append(z(0, 576), z(512), cos, sin, none, none, b.cache)
        return [
            b.attention()[0], b.attention()[1], L.latent_attention(z(3, 4, 512), z(3, 4, 64), b.cache, b.table[:0], b.lens[:0], start, SCALE)[0],
            *L.latent_cache_gather(b.cache, b.table[:0], start, 5), *L.latent_cache_gather(b.cache, b.table, z(3, d=I32), 0),
            *L.absorb_query(z(0, 4, 192), z(1024, 512), cos, sin, none), L.absorb_value(z(0, 4, 512), z(1024, 512)),
            MLA(4, 192, 128).decode(z(0, 4, 192), z(0, 576), z(512), z(1024, 512), cos, sin, none, none, b.cache, b.table, b.lens, b.cu_q),
        ]  # fmt: skip

    want = [(0, 4, 512), (4, 0), (3, 4, 512), (5, 512), (5, 64), (0, 512), (0, 64), (0, 4, 512), (0, 4, 64), (0, 4, 128), (0, 4, 128)]
    before = [t.clone() for t in b.cache[:2]]
    assert [tuple(t.shape) for t in calls()] == want
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(b.cache, before))


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("rows", [16, 64])
def test_a_query_that_is_not_finite_spoils_its_own_row_only(gpu, monkeypatch, rows, bad, fp8):
    """The same bits for all others of the batch, those of the same row block among them; joined from several parts, too."""
    monkeypatch.setattr(sys.modules[__name__], "MIN_WIDTH", WIDTHS[rows])
    h = {16: 5, 64: 24}[rows]
    b = Batch(gpu, [3, 1, 2], [700, 5000, 64], h, page=16, seed=19, fp8=fp8)
    _takes(b, rows)
    want_o, want_lse = b.attention()
    b.check(want_o, want_lse)
    spoilt = torch.zeros(6, h, dtype=torch.bool)
    for token, head in ((1, 2), (3, 0), (5, h - 1)):
        b.q_latent[token, head, 7] = bad
        spoilt[token, head] = True
    o, lse = b.attention()
    assert torch.equal(o[~spoilt], want_o[~spoilt]) and torch.equal(lse.T[~spoilt], want_lse.T[~spoilt])
    assert torch.isnan(o[spoilt].float()).all()


def test_large_scores_in_blocks_of_64_rows_do_not_overflow(gpu, monkeypatch):
    monkeypatch.setattr(sys.modules[__name__], "MIN_WIDTH", 2048)
    test_large_scores_do_not_overflow(gpu)


@pytest.mark.parametrize("width", [0, 2048])
@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
def test_scales_below_zero_and_of_zero(gpu, monkeypatch, fp8, width):
    monkeypatch.setattr(sys.modules[__name__], "MIN_WIDTH", width)
    b = Batch(gpu, [1, 5], [300, 97], 24, fp8=fp8, seed=17)
    b.check(*L.latent_attention(-b.q_latent, -b.q_pe, b.cache, b.table, b.lens, b.cu_q, -SCALE))
    # scale 0: the mean of the rows that are seen, each weight 1 exactly
    o, lse = L.latent_attention(b.q_latent, b.q_pe, b.cache, b.table, b.lens, b.cu_q, 0.0)
    for t, i, seen in [(0, 0, 300)] + [(1 + k, 1, 93 + k) for k in range(5)]:
        rows = b.rows(i)[0][:seen]
        mean, mass = rows.mean(0), rows.abs().mean(0)
        # (e4m3: a weight is its row's scale, rounded to bf16)
        _within(o[t], mean.expand(24, 512), (U * mean.abs() + ((U if fp8 else 0) + 2.0**-14) * mass).expand(24, 512), f"mean of token {t}")
        _within(lse[:, t], torch.full((24,), math.log2(seen)), torch.full((24,), 2.0**-17), f"lse of token {t}")


def test_tokens_behind_the_last_sequence_are_left_alone(gpu):
    b = Batch(gpu, [2, 1], [40, 300], 16, seed=10, extra_tokens=5)
    o = torch.full((8, 16, 512), 7.0, dtype=BF, device=gpu)
    lse = torch.full((16, 8), 7.0, device=gpu)
    L.latent_attention_into(b.q_latent, b.q_pe, b.cache, b.table, b.lens, b.cu_q, SCALE, None, o, lse)
    assert (o[3:] == 7).all() and (lse[:, 3:] == 7).all()
    b.check(o[:3], lse[:, :3])


def test_pages_and_lengths_out_of_range_stay_in_memory(gpu):
    """Page numbers are clamped to the cache, lengths to the table, token offsets to the tokens: nonsense gives some rows, never a fault."""
    b = Batch(gpu, [1, 2], [100, 130], 16, seed=11)
    b.latent.nan_to_num_(0.0)
    b.k_pe.nan_to_num_(0.0)
    b.table[:] = torch.tensor([-(2**31), -1, 2**31 - 1], dtype=I32, device=gpu)[torch.arange(b.table.shape[1], device=gpu) % 3]
    o, lse = b.attention()
    assert torch.isfinite(o.float()).all()
    for lens in ([2**31 - 1, 2**31 - 1], [-5, -(2**31)]):
        b.lens[:] = torch.tensor(lens, dtype=I32, device=gpu)
        o, lse = b.attention()
        assert torch.isfinite(o.float()).all()
    assert (o == 0).all() and (lse == -math.inf).all()
    b.lens[:] = 50
    for cu in ([0, 2**31 - 1, 5], [-7, 3, 1], [3, 2, 1]):
        b.cu_q[:] = torch.tensor(cu, dtype=I32, device=gpu)
        b.attention()
    torch.cuda.synchronize()


@pytest.mark.parametrize("width", [0, 2048])
def test_no_token_belongs_to_two_sequences(gpu, monkeypatch, width):
    """Token offsets that go back are taken as their maximum so far."""
    monkeypatch.setattr(sys.modules[__name__], "MIN_WIDTH", width)
    n = 70
    b = Batch(gpu, [3, 0] + [0] * (n - 3) + [5], [40] * n, 16, seed=16)
    want = b.attention()
    b.check(*want)
    down = b.cu_q.clone()
    down[2:-1] = torch.tensor([0, 3, 1, -7], dtype=I32, device=gpu).repeat(n)[: n - 2]
    assert not torch.equal(down, b.cu_q)
    b.cu_q.copy_(down)
    for x, y in zip(b.attention(), want):
        assert torch.equal(x, y)


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
def test_strided_queries_caches_and_tables(gpu, fp8):
    """Queries and page tables as slices, a cache that is one layer of an allocation for several, results into slices: the same bits."""
    b = Batch(gpu, [1, 3], [150, 70], 16, page=16, fp8=fp8, seed=12)
    want = b.attention()
    wide_q = torch.zeros(4, 17, 640, dtype=BF, device=gpu)
    wide_q[:, :16, :512], wide_q[:, :16, 512:576] = b.q_latent, b.q_pe
    raw = lambda t: t.view(torch.uint8) if t.dtype == L.FP8 else t  # noqa: E731
    layers = [None if t is None else torch.zeros(t.shape[0], 3, *t.shape[1:], dtype=t.dtype, device=gpu) for t in b.cache]
    for wide, t in zip(layers, b.cache):
        if t is not None:
            raw(wide)[:, 1] = raw(t)
    cache = L.LatentCache(*(None if t is None else t[:, 1] for t in layers))
    table = torch.full((2, b.table.shape[1] + 9), -3, dtype=I32, device=gpu)
    table[:, 4 : 4 + b.table.shape[1]] = b.table
    o = torch.zeros(4, 20, 512, dtype=BF, device=gpu)
    lse = torch.zeros(16, 9, device=gpu)
    args = (wide_q[:, :16, :512], wide_q[:, :16, 512:576], cache, table[:, 4 : 4 + b.table.shape[1]], b.lens, b.cu_q, SCALE, None)
    L.latent_attention_into(*args, o[:, 2:18], lse[:, 3:7])
    assert torch.equal(o[:, 2:18], want[0]) and torch.equal(lse[:, 3:7], want[1])
    assert (o[:, :2] == 0).all() and (o[:, 18:] == 0).all()
    for x, y in zip(L.latent_attention(*args), want):
        assert torch.equal(x, y)
    # heads in front of the tokens, and rows that are not 16-byte aligned (copied by the Python body)
    by_head = b.q_latent.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.zeros(4, 16, 65, dtype=BF, device=gpu)
    odd[..., 1:] = b.q_pe
    for x, y in zip(L.latent_attention(by_head, odd[..., 1:], cache, b.table, b.lens, b.cu_q, SCALE), want):
        assert torch.equal(x, y)


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
def test_a_cache_of_a_single_page_with_a_stride_of_its_own(gpu, fp8):
    g, w, _, cos, sin = _layer(1, 52, gpu)
    kv_a, idx = torch.randn(40, 576, generator=g).to(BF).to(gpu), torch.arange(40, device=gpu)
    table, cu = torch.zeros(1, 1, dtype=I32, device=gpu), torch.tensor([0, 40], dtype=I32, device=gpu)
    q_latent, q_pe = torch.randn(1, 4, 512, generator=g).to(BF).to(gpu), torch.randn(1, 4, 64, generator=g).to(BF).to(gpu)
    want = None
    for single in (lambda t: t, lambda t: t.as_strided(t.shape, (t.stride(1), *t.stride()[1:]))):
        cache = L.LatentCache(*(None if t is None else single(t) for t in L.LatentCache.empty(1, 64, L.FP8 if fp8 else BF, gpu)))
        L.latent_cache_append(kv_a, w, cos, sin, idx, idx, cache)
        got = (*L.latent_cache_gather(cache, table, cu, 40), *L.latent_attention(q_latent, q_pe, cache, table, cu[1:], cu[:2] // 40, SCALE))
        want = want or got
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert cache.latent.stride(0) == 512 and torch.isfinite(want[0].float()).all()


@pytest.mark.parametrize("offset", [1, 4])
def test_contiguous_rows_off_their_alignment(gpu, offset):
    """Every input that may begin anywhere, as a contiguous slice of a flat buffer that is 2 or 8 bytes off: the aligned call's bits."""

    def off(t):
        at = max(2 * offset // t.element_size(), 1)  # (fp32: 4 or 8 bytes)
        x = torch.empty(t.numel() + 8, dtype=t.dtype, device=gpu)[at : at + t.numel()].view(t.shape)
        x.copy_(t)
        assert x.is_contiguous() and x.data_ptr() % 16 != 0
        return x

    g, w, kv_b, cos, sin = _layer(5, 50, gpu)
    b = Batch(gpu, [1, 3], [150, 70], 5, seed=51)
    idx = torch.arange(4, device=gpu)
    attention = lambda f: L.latent_attention(f(b.q_latent), f(b.q_pe), b.cache, b.table, b.lens, b.cu_q, SCALE)  # noqa: E731
    q, kv_a = torch.randn(4, 5, 192, generator=g).to(BF).to(gpu), torch.randn(4, 576, generator=g).to(BF).to(gpu)
    query = lambda f: L.absorb_query(f(q), f(kv_b), f(cos), f(sin), idx)  # noqa: E731
    value = lambda f: [L.absorb_value(f(b.q_latent), f(kv_b))]  # noqa: E731

    def append(weight):
        def call(f):
            cache = L.LatentCache(*(torch.zeros(1, 16, n, dtype=BF, device=gpu) for n in (512, 64)))
            L.latent_cache_append(f(kv_a), f(weight), f(cos), f(sin), idx, idx, cache)
            return cache[:2]

        return call

    for call in (attention, query, value, append(w), append(w.float())):
        for x, y in zip(call(off), call(lambda t: t)):
            assert torch.equal(x, y)


def test_rows_beyond_32_bit_offsets(gpu):
    """A cache of 5 GB whose sequences lie in its last pages."""
    b = Batch(gpu, [1, 1], [100, 300], 16, seed=13)
    want = b.attention()
    pages = 75_000
    big = L.LatentCache(torch.empty(pages, 64, 512, dtype=BF, device=gpu), torch.empty(pages, 64, 64, dtype=BF, device=gpu))
    first = pages - len(b.latent)
    big.latent[first:], big.k_pe[first:] = b.latent, b.k_pe
    table = b.table + first
    for x, y in zip(L.latent_attention(b.q_latent, b.q_pe, big, table, b.lens, b.cu_q, SCALE), want):
        assert torch.equal(x, y)
    cu = torch.tensor([0, 100, 400], dtype=I32, device=gpu)
    for x, y in zip(L.latent_cache_gather(big, table, cu, 400), L.latent_cache_gather(b.cache, b.table, cu, 400)):
        assert torch.equal(x, y)
    g = torch.Generator().manual_seed(1)
    kv_a, w, cs = torch.randn(2, 576, generator=g).to(BF).to(gpu), torch.ones(512, device=gpu), torch.ones(4, 64, dtype=BF, device=gpu)
    slots = torch.tensor([pages * 64 - 1, pages * 64], device=gpu)  # the last row, and one behind it
    L.latent_cache_append(kv_a, w, cs, cs, torch.zeros(2, dtype=I64, device=gpu), slots, big)
    n, pe = O.append_rows(kv_a.cpu(), w.cpu(), cs.cpu(), cs.cpu(), torch.zeros(2, dtype=I64), 1e-6)
    _within(big.latent[-1, -1], n[0], (U + 2.0**-20) * n[0].abs(), "the last row")


# ---------------------------------------------------------------------------------------------
# append and gather


def _tables(positions, dev):
    cos, sin = P.cos_sin_table(torch.arange(positions), 64, base=10000.0, dtype=BF)
    return cos.to(dev), sin.to(dev)


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("tokens,page,weight", [(1, 16, BF), (3, 64, torch.float32), (130, 32, BF), (1021, 128, torch.float32)])
def test_append_matches_the_oracle(gpu, tokens, page, weight, fp8):
    g = torch.Generator().manual_seed(tokens)
    pages = -(-tokens // page) + 2
    kv_a = (1.7 * torch.randn(tokens, 640, generator=g)).to(BF)[:, 32:608]
    w = (1 + 0.3 * torch.randn(512, generator=g)).to(weight)
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    slots[1::7] = -1
    pos = torch.randint(0, 50, (tokens,), generator=g)
    cos, sin = _tables(50, gpu)
    cache = L.LatentCache.empty(pages, page, L.FP8 if fp8 else BF, gpu)
    before = [None if t is None else t.view(torch.uint8).random_(0, 100, generator=torch.Generator(gpu).manual_seed(2)).clone().view(t.dtype) for t in cache]
    L.latent_cache_append(kv_a.to(gpu)[:, :], w.to(gpu), cos, sin, pos.to(gpu), slots.to(gpu), cache, 1e-5)
    n, pe = O.append_rows(kv_a, w, cos.cpu(), sin.cpu(), pos, 1e-5)
    used = slots >= 0
    at = slots[used].to(gpu)
    turned = pe[used].abs() + kv_a[used][:, 512:].double().abs().amax(-1, keepdim=True)
    _within(cache.k_pe.view(-1, 64)[at], pe[used], U * pe[used].abs() + 2.0**-22 * turned, "k_pe")
    if fp8:
        scale = n[used].abs().amax(-1) / 448
        _within(cache.scale.view(-1)[at], scale, 2.0**-20 * scale, "scale")
        got = cache.latent.to(torch.float32).view(-1, 512)[at].double().cpu() * cache.scale.view(-1)[at].double().cpu()[:, None]
        _within(got, n[used], torch.maximum((2.0**-4 + 2.0**-18) * n[used].abs(), 2.0**-10 * scale[:, None]), "latent")
        assert (cache.latent.to(torch.float32).view(-1, 512)[at].abs().amax(-1) == 448).all()
    else:
        _within(cache.latent.view(-1, 512)[at], n[used], (U + 2.0**-20) * n[used].abs(), "latent")
    others = torch.ones(pages * page, dtype=torch.bool, device=gpu)
    others[at] = False
    for t, was in zip(cache, before):
        if t is not None:
            flat = lambda x: x.reshape(pages * page, -1).view(torch.uint8)[others]  # noqa: E731
            assert torch.equal(flat(t), flat(was)), "a row that no token names was written"


def test_append_of_a_row_of_zeros_and_of_far_positions(gpu):
    cos, sin = _tables(10, gpu)
    for dtype in (BF, L.FP8):
        cache = L.LatentCache.empty(1, 16, dtype, gpu)
        kv_a = torch.zeros(3, 576, dtype=BF, device=gpu)
        kv_a[:, 512:] = 1
        L.latent_cache_append(kv_a, torch.ones(512, device=gpu), cos, sin, torch.tensor([-4, 10**12, 9], device=gpu), torch.arange(3, device=gpu), cache)
        assert (cache.latent[0, :3].to(torch.float32) == 0).all() and (cache.scale is None or (cache.scale[0, :3] == 0).all())
        assert (cache.k_pe[0, 0] == 1).all() and torch.equal(cache.k_pe[0, 1], cache.k_pe[0, 2])  # clamped to the tables' ends


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("lengths,page", [([1], 16), ([5, 0, 64, 200], 64), ([1021], 16), ([3] * 130, 32)])
def test_gather_returns_the_rows_in_order(gpu, lengths, page, fp8):
    b = Batch(gpu, [0] * len(lengths), lengths, 1, page=page, fp8=fp8, seed=len(lengths), extra_tokens=1)
    total = sum(lengths)
    cu = torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=I32, device=gpu)
    rows = [b.rows(i) for i in range(len(lengths))]
    want, want_pe = torch.cat([r[0] for r in rows]), torch.cat([r[1] for r in rows])
    out, pe = torch.full((total + 3, 520), 7.0, dtype=BF, device=gpu)[:, :512], torch.full((total + 3, 64), 7.0, dtype=BF, device=gpu)
    L.latent_cache_gather_into(b.cache, b.table, cu, out, pe)
    _within(out[:total], want, (U if fp8 else 0.0) * want.abs(), "latent")
    assert torch.equal(pe[:total].double().cpu(), want_pe)
    assert (out[total:] == 7).all() and (pe[total:] == 7).all()
    for x, y in zip(L.latent_cache_gather(b.cache, b.table, cu, total), (out[:total], pe[:total])):
        assert torch.equal(x, y)
    few = total // 2  # room for fewer rows than the sequences have
    for x, y in zip(L.latent_cache_gather(b.cache, b.table, cu, few), (out[:few], pe[:few])):
        assert torch.equal(x, y)


# ---------------------------------------------------------------------------------------------
# absorbed products


def _absorbed_products(gpu, tokens, h):
    g = torch.Generator().manual_seed(tokens * 100 + h)
    q = torch.randn(tokens, h, 200, generator=g).to(BF)[..., 8:]
    w = (torch.randn(h * 256, 512, generator=g) * 512**-0.5).to(BF)
    pos = torch.randint(0, 50, (tokens,), generator=g)
    cos, sin = _tables(50, gpu)
    q_latent, q_pe = L.absorb_query(q.to(gpu)[..., :], w.to(gpu), cos, sin, pos.to(gpu))
    want, mass = O.absorb_query(q, w)
    _within(q_latent, want, U * want.abs() + 130 * 2.0**-24 * mass, "q_latent")
    want = O.rotate(q[..., 128:], cos.cpu(), sin.cpu(), pos)
    _within(q_pe, want, U * want.abs() + 2.0**-22 * q[..., 128:].double().abs().amax(-1, keepdim=True) * 2, "q_pe")
    x = torch.randn(h, tokens, 512, generator=g).to(BF).transpose(0, 1)
    got = L.absorb_value(x.to(gpu), w.to(gpu))
    want, mass = O.absorb_value(x, w)
    _within(got, want, U * want.abs() + 514 * 2.0**-24 * mass, "o")


@pytest.mark.parametrize("h", [1, 16, 37])
@pytest.mark.parametrize("tokens", [1, 15, 16, 17, 300])
def test_absorbed_products_match_the_oracle(gpu, tokens, h):
    _absorbed_products(gpu, tokens, h)


# Many tiles a compute unit, and workgroups whose tokens are more tiles than their ring has slots.
@pytest.mark.parametrize("tokens, h", [(90, 150), (200, 130), (270, 128), (580, 257)])
def test_absorbed_products_of_many_heads_match_the_oracle(gpu, tokens, h):
    _absorbed_products(gpu, tokens, h)


# ---------------------------------------------------------------------------------------------
# A run of them together


def _layer(h, seed, dev):
    g = torch.Generator().manual_seed(seed)
    w = (1 + 0.2 * torch.randn(512, generator=g)).to(BF)
    kv_b = (torch.randn(h * 256, 512, generator=g) * 512**-0.5).to(BF)
    return g, w.to(dev), kv_b.to(dev), *_tables(512, dev)


def _expanded_step(q, cache, table, length, kv_b, cos, sin, pos):
    """What training would compute for the newest rows of one sequence: gathered rows expanded to keys and values, then the framework's own
    attention over the whole sequence (its other rows' queries are zeros)."""
    from pithtrain_amd.operators.mla.hip import attention_func
    from pithtrain_amd.operators.mla_assemble import mla_assemble_qkv

    h, n = q.shape[1], q.shape[0]
    c, pe = L.latent_cache_gather(cache, table, torch.tensor([0, length], dtype=I32, device=q.device), length)
    kv = (c.float() @ kv_b.float().T).to(BF).view(1, length, h, 256)
    full = torch.zeros(1, length, h, 192, dtype=BF, device=q.device)
    full[0, length - n :] = q
    at = torch.zeros(length, dtype=I64, device=q.device)
    at[length - n :] = pos
    qs, ks, vs = mla_assemble_qkv(full, kv, pe.view(1, length, 1, 64), cos, sin, at[None])
    ks[..., 128:] = pe.view(1, length, 1, 64)  # the cache holds rotated rows already
    return attention_func(qs, ks, vs, SCALE, causal=True)[0, length - n :]


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
def test_prompt_then_steps_agree_with_the_expanded_layer(gpu, fp8):
    """A prompt into the cache, then three steps of one token and one of four, two sequences side by side: MLA.decode against the expanded form over
    the gathered rows. The two round at different places (q_latent, P, o_latent here; keys, values and P there), each by at most u relative and
    independently of one another, 2^-8 / sqrt(3) in the mean of the squares: six of them, and the scores' (of size about 2 bits) once more, stay
    below 3 2^-8 of the norm."""
    h = 16
    g, w, kv_b, cos, sin = _layer(h, 21, gpu)
    layer = MLA(h, 192, 128)
    cache = L.LatentCache.empty(40, 16, L.FP8 if fp8 else BF, gpu)
    cache.latent.view(torch.uint8).fill_(255), cache.k_pe.fill_(math.nan)
    table = torch.randperm(40, generator=g)[:38].view(2, 19).to(I32).to(gpu)
    lengths = [0, 0]
    for counts in ([200, 77], [1, 1], [1, 1], [1, 1], [4, 4], [0, 2]):
        t = sum(counts)
        q = torch.randn(t, h, 192, generator=g).to(BF).to(gpu)
        kv_a = torch.randn(t, 576, generator=g).to(BF).to(gpu)
        pos = torch.cat([torch.arange(a, a + n) for a, n in zip(lengths, counts)]).to(gpu)
        lengths = [a + n for a, n in zip(lengths, counts)]
        seq = torch.cat([torch.full((n,), i) for i, n in enumerate(counts)]).to(gpu)
        slots = table[seq, pos // 16].long() * 16 + pos % 16
        cu = torch.tensor([0, counts[0], t], dtype=I32, device=gpu)
        lens = torch.tensor(lengths, dtype=I32, device=gpu)
        o = layer.decode(q, kv_a, w, kv_b, cos, sin, pos, slots, cache, table, lens, cu)
        first = 0
        for i, n in enumerate(counts):
            if n:
                sl = slice(first, first + n)
                want = _expanded_step(q[sl], cache, table[i : i + 1], lengths[i], kv_b, cos, sin, pos[sl]).double()
                assert (o[sl].double() - want).norm() < 3 * 2.0**-8 * want.norm()
                first += n
        # and the same bits from the parts
        ql, qp = L.absorb_query(q, kv_b, cos, sin, pos)
        assert torch.equal(o, L.absorb_value(L.latent_attention(ql, qp, cache, table, lens, cu, layer.softmax_scale)[0], kv_b))


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("prefix,new", [(1, 1), (77, 130), (300, 33), (1000, 257)])
def test_a_prompt_behind_a_cached_prefix_in_expanded_form(gpu, prefix, new, fp8):
    """Gathered rows as keys in two parts (nothing is rotated again) and values, without a mask; the prompt against itself, causal; the two joined by
    their LSE. Against the layer in 64 bits, from the rows that the cache holds.

    Per element: keys, values, weights, the part and the rotated parts are rounded to bf16. With k = |q| . |W| |c| + |q_pe| . |p| the largest score of
    absolute values of a row, in nats, a score is off by at most d = 3 u k (the query's rotation and the key's, which is rounded once here and once in the
    cache) + 2^-13 k (sums of 512 and 192 fp32 products): 2 d of the mass, as weight and denominator; the value's and the weight's rounding u each, the part's u of |o|, of both parts."""
    from pithtrain_amd.operators.mla.hip import _mla_fwd
    from pithtrain_amd.operators.mla_assemble import mla_assemble_qkv
    from pithtrain_amd.operators.ring_attention.mla import _online_softmax_combine_log2

    h, page = 4, 16
    g, w, kv_b, _, _ = _layer(h, 60 + new, gpu)
    cos, sin = _tables(prefix + new, gpu)
    total = prefix + new
    cache = L.LatentCache.empty(-(-total // page) + 1, page, L.FP8 if fp8 else BF, gpu)
    table = torch.randperm(cache.latent.shape[0], generator=g)[: -(-total // page)][None].to(I32).to(gpu)
    pos = torch.arange(total, device=gpu)
    kv_a = torch.randn(total, 576, generator=g).to(BF).to(gpu)
    L.latent_cache_append(kv_a, w, cos, sin, pos, table[0, pos // page].long() * page + pos % page, cache)
    q = (0.5 * torch.randn(1, new, h, 192, generator=g)).to(BF).to(gpu)

    # as a program does it
    offsets = torch.tensor([0, prefix], dtype=I32, device=gpu)
    c, pe = L.latent_cache_gather(cache, table, offsets, prefix)
    kv = (c @ kv_b.T).view(1, prefix, h, 256)
    mine, mine_pe = L.latent_cache_gather(cache, table, torch.tensor([0, total], dtype=I32, device=gpu), total)
    own_kv = (mine[prefix:] @ kv_b.T).view(1, new, h, 256)
    q_rot, k_own, v_own = mla_assemble_qkv(q, own_kv, kv_a[None, prefix:, None, 512:], cos, sin, pos[None, prefix:])
    before = _mla_fwd(q_rot, kv[..., :128].contiguous(), kv[..., 128:].contiguous(), SCALE, causal=False, k_pe=pe[None])
    own = _mla_fwd(q_rot, k_own, v_own, SCALE, causal=True)
    o, lse = _online_softmax_combine_log2(*before, *own)

    rows, rot = (t.double().cpu() for t in (mine, mine_pe))
    qc, wt = q[0].double().cpu(), kv_b.double().cpu().view(h, 256, 512)
    qr = O.rotate(q[0, :, :, 128:].cpu(), cos.cpu(), sin.cpu(), pos[prefix:].cpu())
    seen = O.sees(new, total)
    for i in range(h):
        keys, values = rows @ wt[i, :128].T, rows @ wt[i, 128:].T
        keys_mass, values_mass = rows.abs() @ wt[i, :128].abs().T, rows.abs() @ wt[i, 128:].abs().T
        s = ((qc[:, i, :128] @ keys.T + qr[:, i] @ rot.T) * SCALE).masked_fill(~seen, -math.inf)
        weights = s.softmax(-1)
        want, want_lse = weights @ values, torch.logsumexp(s, -1) / math.log(2)
        k = ((qc[:, i, :128].abs() @ (keys.abs() + 2.0**-7 * keys_mass).T + qr[:, i].abs() @ rot.abs().T) * SCALE).masked_fill(~seen, 0).amax(-1)
        d = (3 * U + 2.0**-13) * k
        mass = weights @ (values.abs() + 2.0**-13 * values_mass)
        _within(o[0, :, i], want, (3 * U + 2.0**-10 + 2 * d)[:, None] * mass, f"o of head {i}")
        _within(lse[0, i], want_lse, d / math.log(2) + 2.0**-14, f"lse of head {i}")


def test_results_do_not_depend_on_the_run(gpu):
    b = Batch(gpu, [1] * 9, [3000 + 37 * i for i in range(9)], 16, seed=30)
    first = b.attention()
    for _ in range(3):
        for x, y in zip(b.attention(), first):
            assert torch.equal(x, y)


def test_two_streams_and_two_calls_at_once(gpu):
    a, b = (Batch(gpu, [1, 2], [2500, 40 + s], 16, seed=s, fp8=bool(s)) for s in (0, 1))
    want = a.attention(), b.attention()
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    got = [[], []]
    for _ in range(5):
        for k, (s, x) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(s):
                got[k].append(x.attention())
    torch.cuda.synchronize()
    for k in range(2):
        for pair in got[k]:
            assert all(torch.equal(x, y) for x, y in zip(pair, want[k]))


def test_blocks_of_64_rows_over_runs_streams_and_replays(gpu, monkeypatch):
    """The same bits from call to call, from two calls at once on two streams, and from a graph whose lengths change in place between its replays."""
    monkeypatch.setattr(sys.modules[__name__], "MIN_WIDTH", 2048)
    a, b = (Batch(gpu, [3] * 9, [2000 + 37 * i for i in range(9)], 16, seed=40 + s, fp8=bool(s), page=16) for s in (0, 1))
    want = a.attention(), b.attention()
    a.check(*want[0])
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for k, (s, x) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(s):
                got[k].append(x.attention())
    torch.cuda.synchronize()
    for k in range(2):
        for pair in got[k]:
            assert all(torch.equal(x, y) for x, y in zip(pair, want[k]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = a.attention()
    for step in (0, 1000, 1990, 3):
        a.lens.copy_(torch.tensor(a.lengths, dtype=I32) - step)
        for t in out:
            t.fill_(math.nan)
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, a.attention())), step


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
def test_a_captured_step_follows_its_sequences(gpu, fp8):
    """One graph of a decoding step, replayed while lengths, slots, pages and tokens change in place (padded sequences among them), with eager work and
    another graph in between: every replay equals the eager call."""
    h, b, page = 16, 3, 16
    g, w, kv_b, cos, sin = _layer(h, 31, gpu)
    layer = MLA(h, 192, 128)
    cache = L.LatentCache.empty(64, page, L.FP8 if fp8 else BF, gpu)
    cache.latent.view(torch.uint8).zero_(), cache.k_pe.normal_(generator=torch.Generator(gpu).manual_seed(1))
    if fp8:
        cache.scale.fill_(1.0)
    table = torch.randperm(64, generator=g)[:60].view(b, 20).to(I32).to(gpu)
    q, kv_a = torch.empty(b, h, 192, dtype=BF, device=gpu), torch.empty(b, 576, dtype=BF, device=gpu)
    pos, slots = torch.zeros(b, dtype=I64, device=gpu), torch.full((b,), -1, dtype=I64, device=gpu)
    lens, cu = torch.zeros(b, dtype=I32, device=gpu), torch.arange(b + 1, dtype=I32, device=gpu)
    step = lambda: layer.decode(q, kv_a, w, kv_b, cos, sin, pos, slots, cache, table, lens, cu)  # noqa: E731

    def fill(lengths):
        q.copy_(torch.randn(b, h, 192, generator=g))
        kv_a.copy_(torch.randn(b, 576, generator=g))
        n = torch.tensor(lengths)
        lens.copy_(n)
        at = (n - 1).clamp(min=0)
        pos.copy_(at)
        where = table.cpu()[torch.arange(b), at // page].long() * page + at % page
        slots.copy_(torch.where(n > 0, where, -1))

    fill([5, 6, 7])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    long = Batch(gpu, [1], [5000], h, seed=33)
    with torch.cuda.graph(other):
        long_out = long.attention()
    want_long = long.attention()
    for lengths in ([1, 1, 1], [16, 17, 300], [0, 320, 33], [2, 0, 0], [319, 318, 320]):
        fill(lengths)
        out.fill_(math.nan)
        graph.replay()
        other.replay()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step()), lengths
        assert all(torch.equal(x, y) for x, y in zip(long_out, want_long))
        assert all((out[i] == 0).all() for i, n in enumerate(lengths) if n == 0)


def test_what_is_written_counts_as_changed(gpu):
    """A backward that saved a tensor which one of the operators has written since is refused, in place of computing with the new contents."""
    b = Batch(gpu, [1, 2], [150, 40], 16, seed=34)
    o, lse = torch.zeros(3, 16, 512, dtype=BF, device=gpu), torch.zeros(16, 3, device=gpu)
    rows, pe = torch.zeros(190, 512, dtype=BF, device=gpu), torch.zeros(190, 64, dtype=BF, device=gpu)
    cos, sin = _tables(8, gpu)
    kv_a, ones, idx = torch.zeros(3, 576, dtype=BF, device=gpu), torch.ones(512, device=gpu), torch.arange(3, device=gpu)
    cu = torch.tensor([0, 150, 190], dtype=I32, device=gpu)
    calls = [
        (b.cache[:2], lambda: L.latent_cache_append(kv_a, ones, cos, sin, idx, idx, b.cache)),
        ((rows, pe), lambda: L.latent_cache_gather_into(b.cache, b.table, cu, rows, pe)),
        ((o, lse), lambda: L.latent_attention_into(b.q_latent, b.q_pe, b.cache, b.table, b.lens, b.cu_q, SCALE, None, o, lse)),
    ]
    for written, call in calls:
        for t in written:
            x = torch.ones_like(t, requires_grad=True)
            y = x * t
            with torch.no_grad():
                call()
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.sum().backward()


def test_compiled_operators_match_eager(gpu):
    b = Batch(gpu, [1, 2], [150, 40], 16, seed=34)
    f = torch.compile(lambda q, p, c, k: L.latent_attention(q, p, L.LatentCache(c, k), b.table, b.lens, b.cu_q, SCALE), backend="aot_eager", fullgraph=True)
    with torch.no_grad():
        for x, y in zip(f(b.q_latent, b.q_pe, b.latent, b.k_pe), b.attention()):
            assert torch.equal(x, y)


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
def test_a_compiled_decoding_step_writes_the_cache(gpu, fp8):
    """The same result and the same rows in the cache as the eager step's, whose tensors the compiled one changes in place."""
    g, w, kv_b, cos, sin = _layer(4, 35, gpu)
    q, kv_a = torch.randn(3, 4, 192, generator=g).to(BF).to(gpu), torch.randn(3, 576, generator=g).to(BF).to(gpu)
    idx, table = torch.arange(3, device=gpu), torch.zeros(1, 1, dtype=I32, device=gpu)
    lens, cu = torch.tensor([3], dtype=I32, device=gpu), torch.tensor([0, 3], dtype=I32, device=gpu)
    layer = MLA(4, 192, 128)

    def step(*cache):
        return layer.decode(q, kv_a, w, kv_b, cos, sin, idx, idx, L.LatentCache(*cache), table, lens, cu)

    caches = [[t for t in L.LatentCache.empty(1, 16, L.FP8 if fp8 else BF, gpu) if t is not None] for _ in range(2)]
    for t in caches[0] + caches[1]:
        t.view(torch.uint8).zero_()
    with torch.no_grad():
        want = step(*caches[0])
        got = torch.compile(step, backend="aot_eager", fullgraph=True)(*caches[1])
    assert torch.equal(got, want)
    for x, y in zip(*caches):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)) and y.view(torch.uint8).any()


# ---------------------------------------------------------------------------------------------
# Refusals


def test_wrong_arguments_are_refused(gpu):
    b = Batch(gpu, [1, 2], [40, 50], 4, seed=40)
    call = lambda **kw: L.latent_attention(*{**dict(q=b.q_latent, p=b.q_pe, c=b.cache, t=b.table, l=b.lens, cu=b.cu_q, s=SCALE, m=None), **kw}.values())  # noqa: E731
    with pytest.raises(AssertionError, match="q_latent must be"):
        call(q=b.q_latent[..., :256])
    with pytest.raises(AssertionError, match="q_latent must be"):
        call(q=b.q_latent.float())
    with pytest.raises(AssertionError, match="q_pe must be"):
        call(p=b.q_pe[:2])
    with pytest.raises(AssertionError, match="cu_q must be"):
        call(cu=b.cu_q[:2])
    with pytest.raises(AssertionError, match="cu_q must be"):
        call(cu=b.cu_q.long())
    with pytest.raises(AssertionError, match="lengths must be"):
        call(l=b.lens.long())
    with pytest.raises(AssertionError, match="page_table must be"):
        call(t=b.table[:1])
    with pytest.raises(AssertionError, match="tree_mask must be"):
        call(m=torch.zeros(2, dtype=I64, device=gpu))
    with pytest.raises(AssertionError, match="k_pe does not match"):
        call(c=L.LatentCache(b.latent, b.k_pe[1:]))
    with pytest.raises(AssertionError, match="has no scale"):
        call(c=L.LatentCache(b.latent, b.k_pe, torch.ones(b.k_pe.shape[:2], device=gpu)))
    with pytest.raises(AssertionError, match="needs a float32 scale"):
        call(c=L.LatentCache(b.latent.to(L.FP8), b.k_pe))
    with pytest.raises(AssertionError, match="page are not contiguous"):
        call(c=L.LatentCache(b.latent.transpose(0, 1).contiguous().transpose(0, 1), b.k_pe))
    with pytest.raises(_C.PithError, match="page size"):
        call(c=L.LatentCache(b.latent[:, :48], b.k_pe[:, :48]))
    with pytest.raises(_C.PithError, match="empty page table"):
        call(t=b.table[:, :0])
    with pytest.raises(RuntimeError, match="different devices|need tensors on a GPU"):
        call(l=b.lens.cpu())
    w = torch.zeros(4 * 256, 512, dtype=BF, device=gpu)
    with pytest.raises(AssertionError, match="kv_b_weight must be"):
        L.absorb_value(b.q_latent, w[:-1])
    with pytest.raises(AssertionError, match="o_latent must be"):
        L.absorb_value(b.q_pe, w)
    cos, sin = _tables(8, gpu)
    kv_a, ones, idx = torch.zeros(3, 576, dtype=BF, device=gpu), torch.ones(512, device=gpu), torch.zeros(3, dtype=I64, device=gpu)
    with pytest.raises(AssertionError, match="kv_a must be"):
        L.latent_cache_append(kv_a[:, :512], ones, cos, sin, idx, idx, b.cache)
    with pytest.raises(AssertionError, match="slots must be"):
        L.latent_cache_append(kv_a, ones, cos, sin, idx, idx.int(), b.cache)
    with pytest.raises(AssertionError, match="cos and sin must be"):
        L.latent_cache_append(kv_a, ones, cos[:, :32], sin[:, :32], idx, idx, b.cache)
    with pytest.raises(TypeError):
        L.latent_cache_append(kv_a, ones.half(), cos, sin, idx, idx, b.cache)
    with pytest.raises(RuntimeError, match="has no backward"):
        call(q=b.q_latent.clone().requires_grad_())


def test_index_checks_on_request(gpu, monkeypatch):
    monkeypatch.setenv("PITHTRAIN_AMD_CHECK_POSITIONS", "1")
    cos, sin = _tables(8, gpu)
    cache = L.LatentCache.empty(2, 16, BF, gpu)
    kv_a, ones = torch.zeros(3, 576, dtype=BF, device=gpu), torch.ones(512, device=gpu)
    idx = lambda *x: torch.tensor(x, device=gpu)  # noqa: E731
    call = lambda pos, slots: L.latent_cache_append(kv_a, ones, cos, sin, pos, slots, cache)  # noqa: E731
    call(idx(0, 7, 3), idx(-1, 31, -1))
    with pytest.raises(AssertionError, match="position_ids span"):
        call(idx(0, 8, 3), idx(0, 1, 2))
    with pytest.raises(AssertionError, match="slots go up to"):
        call(idx(0, 0, 0), idx(0, 1, 32))
    with pytest.raises(AssertionError, match="same slot"):
        call(idx(0, 0, 0), idx(0, 5, 5))
    with pytest.raises(AssertionError, match="position_ids span"):
        L.absorb_query(torch.zeros(3, 2, 192, dtype=BF, device=gpu), torch.zeros(512, 512, dtype=BF, device=gpu), cos, sin, idx(0, -1, 3))
    b = Batch(gpu, [65], [70], 1, seed=41)
    with pytest.raises(AssertionError, match="more than 64"):
        b.attention(torch.zeros(65, dtype=I64, device=gpu))
