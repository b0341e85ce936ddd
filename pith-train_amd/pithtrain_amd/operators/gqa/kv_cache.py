"""
The GQA layer while it answers: a paged cache of keys and values, attention of new tokens to it, and attention to selected pages, backed by
libpith_hip.so.

Training runs qk_norm_rope and causal attention over whole sequences (pithtrain/models/qwen3_30b_a3b.py:413-438). A token that is answered leaves its
normalised, rotated key and its value in a cache and attends to the rows of its sequence:

    kv_cache_append    norm + rotation of q and k, k and v of new tokens into cache pages (bf16, or e4m3 with one scale a row and head)
    kv_attention       causal attention of the newest tokens of every sequence to its cached rows, or of a tree of drafted tokens
    kv_decode          the two in a row: what stands between the layer's projections

For long contexts, attention to a few pages that a cheap score selects for each token and key-value head:

    kv_page_bounds     least and largest key features of the pages that new tokens filled
    kv_select_pages    the pages whose bounds allow the largest q . k, as page tables of the heads for kv_attention

 T : new tokens of all sequences, one behind the other, b : sequences, h : query heads, hkv : key-value heads, d : head dim (64 or 128).
Token counts, lengths, page tables, slots and tree masks (plan_step and latent.tree_mask_of make them) are device tensors that only the kernels read: a captured graph follows their contents.
The operators serve; they have no backward. Arguments that require a gradient are refused while gradients are recorded.
"""

from typing import NamedTuple, Optional, Tuple

import torch

from pithtrain_amd import _C
from pithtrain_amd._ext import define_op
from pithtrain_amd.operators.mla.latent import (
    FP8, MAX_DRAFTS, _aligned_rows, _check_positions, _checking, _index, _launch, _no_gradients, _strides, _table_args, _unit,
)  # fmt: skip

HEAD_DIMS = (64, 128)  # what the kernels are built for


class KVCache(NamedTuple):
    """Pages of cached rows. k, v [pages, hkv, page_size, d] bf16 or float8_e4m3fn, k_scale, v_scale [pages, hkv, page_size] fp32 (e4m3 only: a feature is
    value * scale of its row and head). page_size is a power of two from 16 to 65536; a page is contiguous, pages may be further apart (the layers of
    a model can share one allocation) and begin at multiples of 16 bytes. Slot s is row s % page_size of page s // page_size."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None

    @classmethod
    def empty(cls, pages: int, kv_heads: int, head_dim: int = 128, page_size: int = 64, dtype: torch.dtype = torch.bfloat16, device="cuda") -> "KVCache":
        """A cache with room for pages * page_size rows; rows hold nothing until kv_cache_append writes them."""
        assert dtype in (torch.bfloat16, FP8), f"the cache holds bfloat16 or float8_e4m3fn, not {dtype}"
        mk = lambda *s, dtype: torch.empty(pages, kv_heads, page_size, *s, dtype=dtype, device=device)  # noqa: E731
        scale = [mk(dtype=torch.float32) for _ in range(2)] if dtype == FP8 else [None, None]
        return cls(mk(head_dim, dtype=dtype), mk(head_dim, dtype=dtype), *scale)

    def empty_bounds(self) -> torch.Tensor:
        """Room for kv_page_bounds of this cache, [pages, hkv, 2, d] bf16; holds nothing yet."""
        pages, heads, _, d = self.k.shape
        return torch.empty(pages, heads, 2, d, dtype=torch.bfloat16, device=self.k.device)


class SelectedPages(NamedTuple):
    """Pages of every token and key-value head, for kv_attention(q, cache, *selected, None, scale). page_table [T, hkv, keep] int32, -1 behind the last;
    lengths [T, hkv] int32: the rows that they make."""

    page_table: torch.Tensor
    lengths: torch.Tensor


def _contiguous_pages(t: torch.Tensor, what: str) -> None:
    sizes, strides, expected = t.shape[1:], t.stride()[1:], 1
    for n, st in zip(reversed(sizes), reversed(strides)):
        assert n == 1 or st == expected, f"a page of {what} is not contiguous"
        expected *= n


def _cache_args(like: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor], v_scale: Optional[torch.Tensor]) -> "_C.KVCacheArgs":
    _C.require_device(like, k, v, *(t for t in (k_scale, v_scale) if t is not None))
    assert k.dtype in (torch.bfloat16, FP8) and k.dim() == 4 and k.shape[3] in HEAD_DIMS, (
        f"cache.k must be a bfloat16 or float8_e4m3fn [pages, heads, page_size, 64 or 128] tensor, got {k.dtype} {list(k.shape)}"
    )
    assert v.dtype == k.dtype and v.shape == k.shape, "cache.v does not match cache.k"
    _contiguous_pages(k, "cache.k")
    _contiguous_pages(v, "cache.v")
    pages, heads, page_size, d = k.shape
    args = _C.KVCacheArgs(
        k=k.data_ptr(), v=v.data_ptr(), pages=pages, page_size=page_size, heads=heads, dim=d, k_ps=k.stride(0), v_ps=v.stride(0), dtype=_C.PITH_BF16,
    )  # fmt: skip
    if k.dtype == FP8:
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            assert t is not None and t.dtype == torch.float32 and t.shape == k.shape[:3], f"an e4m3 cache needs a float32 {name} [pages, heads, page_size]"
            _contiguous_pages(t, f"cache.{name}")
        args.k_scale, args.v_scale, args.k_scale_ps, args.v_scale_ps = k_scale.data_ptr(), v_scale.data_ptr(), k_scale.stride(0), v_scale.stride(0)
        args.dtype = _C.PITH_FP8_E4M3
    else:
        assert k_scale is None and v_scale is None, "a bfloat16 cache has no scales"
    return args


def _rows(t: torch.Tensor, name: str, heads: Optional[int], d: int) -> None:
    assert t.dtype == torch.bfloat16 and t.dim() == 3 and t.shape[2] == d and heads in (None, t.shape[1]), (
        f"{name} must be a bfloat16 [tokens, {'heads' if heads is None else heads}, {d}] tensor, got {t.dtype} {list(t.shape)}"
    )


def _sequences(args, like, page_table, lengths, cu_q, t, head_tables=None) -> None:
    """Fills the fields of page_table, lengths and cu_q; head_tables: key-value heads where each may have its own."""
    _C.require_device(like, page_table, lengths, *(() if cu_q is None else (cu_q,)))
    if head_tables is not None and lengths.dim() == 2:
        b = lengths.shape[0]
        args.lengths = _index(lengths, torch.int32, (b, head_tables), "lengths")
        assert page_table.dtype == torch.int32 and page_table.dim() == 3 and tuple(page_table.shape[:2]) == (b, head_tables), (
            f"page_table must be an int32 [b={b}, heads={head_tables}, pages] tensor, got {page_table.dtype} {list(page_table.shape)}"
        )
        _unit(page_table, "page_table")
        width = page_table.shape[2]
        args.page_table, args.table_width = page_table.data_ptr(), width
        args.table_hs = page_table.stride(1) if head_tables > 1 else width
        args.table_rs = page_table.stride(0) if b > 1 else width * head_tables
        args.head_tables = 1
        assert cu_q is None, "page tables of the heads go with one token a sequence: no cu_q"
    else:
        assert lengths.dim() == 1, "lengths must be one-dimensional, or [b, heads] with a page table of every head"
        b = lengths.shape[0]
        args.lengths = _index(lengths, torch.int32, (b,), "lengths")
        args.page_table, args.table_rs, args.table_width = _table_args(page_table, b)
    args.B, args.T = b, t
    if cu_q is None:
        assert t == b, f"{t} tokens of {b} sequences: without cu_q there is one token a sequence"
    else:
        args.cu_q = _index(cu_q, torch.int32, (b + 1,), "cu_q")


# ---------------------------------------------------------------------------------------------
# Bodies of the ops for calls that the native path does not take (it words no errors), and their fake (shape) implementations.


def _append_body(q, k, v, q_weight, k_weight, cos, sin, position_ids, slots, k_cache, v_cache, k_scale, v_scale, eps):
    _C.require_device(q, k, v, cos, sin, position_ids, slots, *(w for w in (q_weight, k_weight) if w is not None))
    cache = _cache_args(q, k_cache, v_cache, k_scale, v_scale)
    d, heads = cache.dim, cache.heads
    _rows(q, "q", None, d)
    t, h, _ = q.shape
    for name, x in (("k", k), ("v", v)):
        _rows(x, name, heads, d)
        assert x.shape[0] == t, f"{name} has {x.shape[0]} tokens, q has {t}"
    assert cos.dtype == sin.dtype == torch.bfloat16 and cos.dim() == 2 and cos.shape == sin.shape and cos.shape[1] == d, f"cos and sin must be bfloat16 [positions, {d}]"
    assert (q_weight is None) == (k_weight is None), "q_weight and k_weight are given together or not at all"
    code = _C.PITH_BF16
    if q_weight is not None:
        assert q_weight.dtype == k_weight.dtype and tuple(q_weight.shape) == tuple(k_weight.shape) == (d,), f"q_weight and k_weight must be [{d}] tensors of one dtype"
        code = _C.dtype_code(q_weight)
        q_weight, k_weight = _aligned_rows(q_weight), _aligned_rows(k_weight)
    q, k, v = _aligned_rows(q), _aligned_rows(k), _aligned_rows(v)
    cos, sin = (x if x.is_contiguous() and x.data_ptr() % 16 == 0 else x.clone(memory_format=torch.contiguous_format) for x in (cos, sin))
    out = torch.empty((t, h, d), dtype=q.dtype, device=q.device)
    args = _C.KVAppendArgs(
        q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_weight=None if q_weight is None else q_weight.data_ptr(),
        k_weight=None if k_weight is None else k_weight.data_ptr(), cos=cos.data_ptr(), sin=sin.data_ptr(),
        position_ids=_index(position_ids, torch.int64, (t,), "position_ids"), slots=_index(slots, torch.int64, (t,), "slots"),
        q_out=out.data_ptr(), T=t, P=cos.shape[0], H=h, eps=float(eps), weight_dtype=code, cache=cache,
    )  # fmt: skip
    for name, x in (("q", q), ("k", k), ("v", v), ("q_out", out)):
        ts, hs = _strides(x)
        setattr(args, name + "_ts", ts)
        setattr(args, name + "_hs", hs)
    if _checking(slots) and t:
        _check_positions(position_ids, cos.shape[0])
        used = slots[slots >= 0]
        rows = cache.pages * cache.page_size
        assert used.numel() == 0 or int(used.max()) < rows, f"slots go up to {int(used.max())}, the cache holds {rows} rows"
        assert used.unique().numel() == used.numel(), "two tokens name the same slot"
    _launch("pith_kv_append", args, q)
    return out


def _append_fake(q, k, v, q_weight, k_weight, cos, sin, position_ids, slots, k_cache, v_cache, k_scale, v_scale, eps):
    assert q.dim() == 3, "q must be [tokens, heads, features]"
    return q.new_empty(q.shape)


def kv_attention_into(
    q: torch.Tensor, cache: KVCache, page_table: torch.Tensor, lengths: torch.Tensor, cu_q: Optional[torch.Tensor], softmax_scale: float,
    tree_mask: Optional[torch.Tensor], o: torch.Tensor, lse: torch.Tensor,
) -> None:  # fmt: skip
    """kv_attention into tensors of the caller's: o [T, h, d] bf16, whose rows begin at multiples of 16 bytes, and lse [h, T] fp32; neither overlaps what the
    call reads. Tokens from cu_q[b] on keep what they hold."""
    _no_gradients("kv_attention_into", q, *cache, o, lse)
    _C.require_device(q, o, lse)
    cache_args = _cache_args(q, *cache)
    _rows(q, "q", None, cache_args.dim)
    t, h, d = q.shape
    assert o.dtype == torch.bfloat16 and tuple(o.shape) == (t, h, d), "o has the wrong dtype or shape"
    assert lse.dtype == torch.float32 and tuple(lse.shape) == (h, t), "lse has the wrong dtype or shape"
    _unit(o, "o")
    _unit(lse, "lse")
    q = _aligned_rows(q)
    args = _C.KVAttnArgs(q=q.data_ptr(), cache=cache_args, o=o.data_ptr(), lse=lse.data_ptr(), H=h, lse_hs=lse.stride(0) if h > 1 else t, scale=float(softmax_scale))
    _sequences(args, q, page_table, lengths, cu_q, t, cache_args.heads)
    args.q_ts, args.q_hs = _strides(q)
    args.o_ts, args.o_hs = _strides(o)
    if tree_mask is not None:
        assert not args.head_tables, "a tree of drafts goes with one page table for all heads"
        _C.require_device(q, tree_mask)
        args.tree_mask = _index(tree_mask, torch.int64, (t,), "tree_mask")
        if cu_q is not None and _checking(cu_q) and args.B:
            assert int((cu_q[1:] - cu_q[:-1]).max()) <= MAX_DRAFTS, f"a tree has more than {MAX_DRAFTS} tokens"
    with torch.cuda.device(q.device):
        need = _C.lib().pith_kv_attn_workspace_bytes(_C.byref(args))
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        args.workspace, args.workspace_bytes = workspace.data_ptr(), need
        _C.check(_C.lib().pith_kv_attn(_C.byref(args), _C.current_stream(q)))
    torch.autograd.graph.increment_version((o, lse))  # (a backward that saved one of them notices)


def _attention_body(q, k, v, k_scale, v_scale, page_table, lengths, cu_q, softmax_scale, tree_mask):
    o, lse = _attention_fake(q, k, v, k_scale, v_scale, page_table, lengths, cu_q, softmax_scale, tree_mask)
    kv_attention_into(q, KVCache(k, v, k_scale, v_scale), page_table, lengths, cu_q, softmax_scale, tree_mask, o, lse)
    return o, lse


def _attention_fake(q, k, v, k_scale, v_scale, page_table, lengths, cu_q, softmax_scale, tree_mask):
    assert q.dim() == 3, "q must be [tokens, heads, features]"
    t, h, d = q.shape
    return q.new_empty((t, h, d)), q.new_empty((h, t), dtype=torch.float32)


def _check_bounds(bounds: torch.Tensor, heads: Optional[int], d: Optional[int], pages: Optional[int]) -> int:
    shape = tuple(bounds.shape)
    assert bounds.dtype == torch.bfloat16 and bounds.dim() == 4 and shape[2] == 2 and shape[3] in HEAD_DIMS and heads in (None, shape[1]) and d in (None, shape[3]) and pages in (None, shape[0]), (
        f"bounds must be a bfloat16 [pages, heads, 2, d] tensor beside the cache, got {bounds.dtype} {list(shape)}"
    )
    _contiguous_pages(bounds, "bounds")
    return bounds.stride(0)


def _bounds_body(k, v, k_scale, v_scale, bounds, page_table, lengths, cu_q, tokens):
    assert tokens >= 0, f"tokens = {tokens}"
    cache = _cache_args(k, k, v, k_scale, v_scale)
    _C.require_device(k, bounds)
    args = _C.KVBoundsArgs(cache=cache, bounds=bounds.data_ptr(), bounds_ps=_check_bounds(bounds, cache.heads, cache.dim, cache.pages))
    _sequences(args, k, page_table, lengths, cu_q, tokens)
    _launch("pith_kv_bounds", args, k)


def _bounds_fake(k, v, k_scale, v_scale, bounds, page_table, lengths, cu_q, tokens):
    return None


def _select_body(q, bounds, page_table, lengths, cu_q, page_size, keep):
    _C.require_device(q, bounds)
    stride = _check_bounds(bounds, None, None, None)
    pages, heads, _, d = bounds.shape
    _rows(q, "q", None, d)
    table, rows = _select_fake(q, bounds, page_table, lengths, cu_q, page_size, keep)
    q = _aligned_rows(q)
    args = _C.KVSelectArgs(
        q=q.data_ptr(), bounds=bounds.data_ptr(), table_out=table.data_ptr(), lengths_out=rows.data_ptr(), H=q.shape[1], heads=heads, dim=d, pages=pages,
        page_size=page_size, keep=keep, bounds_ps=stride,
    )  # fmt: skip
    _sequences(args, q, page_table, lengths, cu_q, q.shape[0])
    args.q_ts, args.q_hs = _strides(q)
    with torch.cuda.device(q.device):
        need = _C.lib().pith_kv_select_workspace_bytes(_C.byref(args))
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        args.workspace, args.workspace_bytes = workspace.data_ptr(), need
        if args.T and not args.B:  # (tokens of nobody)
            table.fill_(-1)
            rows.zero_()
        _C.check(_C.lib().pith_kv_select(_C.byref(args), _C.current_stream(q)))
    return table, rows


def _select_fake(q, bounds, page_table, lengths, cu_q, page_size, keep):
    assert q.dim() == 3 and bounds.dim() == 4, "q must be [tokens, heads, features] and bounds [pages, heads, 2, features]"
    assert keep >= 1, f"keep = {keep} pages"
    t, heads = q.shape[0], bounds.shape[1]
    return q.new_empty((t, heads, keep), dtype=torch.int32), q.new_empty((t, heads), dtype=torch.int32)


_append_op = define_op("kv_append", _append_body, _append_fake)
_attention_op = define_op("kv_attention", _attention_body, _attention_fake)
_bounds_op = define_op("kv_bounds", _bounds_body, _bounds_fake)
_select_op = define_op("kv_select", _select_body, _select_fake)


# ---------------------------------------------------------------------------------------------


def kv_cache_append(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor], cos: torch.Tensor, sin: torch.Tensor,
    position_ids: torch.Tensor, slots: torch.Tensor, cache: KVCache, eps: float = 1e-6,
) -> torch.Tensor:  # fmt: skip
    """Keys and values of new tokens into the cache; returns the queries that go with them, [T, h, d]. q [T, h, d], k, v [T, hkv, d] bf16 as the projections
    leave them (slices of one projection are read in place); q_weight, k_weight [d] (bf16 or fp32) those of q_norm and k_norm, or None both: no norm; cos /
    sin [positions, d] bf16 the rotary module's tables (the rotation is qk_norm_rope's), position_ids and slots [T] int64. Each is rounded once from fp32.
    An e4m3 row's scale is its largest magnitude / 448. Tokens with a slot below 0 or beyond the cache leave no row (padding). Two tokens of a call must not
    share a slot; positions beyond the tables are clamped to them (PITHTRAIN_AMD_CHECK_POSITIONS=1 raises in all these cases but padding, at the price
    of a device synchronisation)."""
    return _append_op(q, k, v, q_weight, k_weight, cos, sin, position_ids, slots, cache.k, cache.v, cache.k_scale, cache.v_scale, eps)


def kv_attention(
    q: torch.Tensor, cache: KVCache, page_table: torch.Tensor, lengths: torch.Tensor, cu_q: Optional[torch.Tensor], softmax_scale: float,
    tree_mask: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:  # fmt: skip
    """(o [T, h, d] bf16, lse [h, T] fp32 in base 2): attention of the newest tokens of b sequences to their cached rows. Query head i reads key-value head
    i // (h / hkv).

    Tokens cu_q[i] .. cu_q[i + 1] - 1 are the n newest of sequence i, whose lengths[i] cached rows (theirs included: append them first) lie in the
    pages page_table[i]; without cu_q every sequence has one. Token k of them sees the rows up to lengths[i] - n + k; with tree_mask ([T] int64) all rows in
    front of the n newest, and of those row j where bit j of the token's word is set (latent.tree_mask_of makes such words; n is at most 64). A token that sees
    no row gets 0 and an lse of -inf. Tokens from cu_q[b] on are not written. The same call gives the same bits; in a batch of other sequences a token's last
    bits may differ. page_table [b, pages], lengths [b] and cu_q [b + 1] are int32, on the device.

    With page_table [b, hkv, pages] and lengths [b, hkv] every key-value head has rows of its own (kv_select_pages; one token a sequence, no cu_q)."""
    return _attention_op(q, cache.k, cache.v, cache.k_scale, cache.v_scale, page_table, lengths, cu_q, softmax_scale, tree_mask)


def kv_page_bounds(cache: KVCache, bounds: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, cu_q: Optional[torch.Tensor], tokens: int) -> None:
    """Least and largest key features of the pages that the newest tokens filled, into bounds [pages, hkv, 2, d] bf16 (KVCache.empty_bounds): of every page
    whose last row is one of theirs (append them first). Other pages' bounds stay. tokens: T of the step; the rest as in kv_attention. Called
    in every step, it has the bounds of all full pages there."""
    _bounds_op(cache.k, cache.v, cache.k_scale, cache.v_scale, bounds, page_table, lengths, cu_q, tokens)


def kv_select_pages(
    q: torch.Tensor, bounds: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, cu_q: Optional[torch.Tensor], page_size: int, keep: int,
) -> SelectedPages:  # fmt: skip
    """The pages that every token and key-value head attends to: its own (the last one that it sees), and the keep - 1 others that score highest, in the order
    of the sequence; all of them where there are no more than keep. A page's score is the largest over the query heads of the group of
    sum_d max(q_d least_d, q_d largest_d), which no q . k of the page exceeds (but for the rounding of an e4m3 cache's bounds); equal scores go to the page that
    comes first, NaN is above all. q [T, h, d] are rotated queries, bounds kv_page_bounds', page_table (up to 16384 pages wide), lengths, cu_q as in kv_attention
    (causal). Tokens in front of cu_q[0] and from cu_q[b] on get no page and no row."""
    return SelectedPages(*_select_op(q, bounds, page_table, lengths, cu_q, page_size, keep))


def kv_decode(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor], cos: torch.Tensor, sin: torch.Tensor,
    position_ids: torch.Tensor, slots: torch.Tensor, cache: KVCache, page_table: torch.Tensor, lengths: torch.Tensor, cu_q: Optional[torch.Tensor],
    softmax_scale: float, eps: float = 1e-6, tree_mask: Optional[torch.Tensor] = None, bounds: Optional[torch.Tensor] = None, keep: Optional[int] = None,
) -> torch.Tensor:  # fmt: skip
    """The layer between its projections for new tokens, o [T, h, d]: their rows go into the cache, then they attend to the cached rows of their sequences
    (lengths count the new rows). With bounds (KVCache.empty_bounds, which every step of the sequences must have been given) they are kept up to date, and
    with keep too a token attends to that many pages only. Arguments as in the functions above, each looked at when its turn comes: where the attention's are
    refused, the rows have been written. Rows of o from cu_q[b] on hold nothing."""
    assert keep is None or (bounds is not None and tree_mask is None), "keep needs bounds, and goes with causal attention"
    q = kv_cache_append(q, k, v, q_weight, k_weight, cos, sin, position_ids, slots, cache, eps)
    if bounds is not None:
        kv_page_bounds(cache, bounds, page_table, lengths, cu_q, q.shape[0])
    if keep is None:
        return kv_attention(q, cache, page_table, lengths, cu_q, softmax_scale, tree_mask)[0]
    selected = kv_select_pages(q, bounds, page_table, lengths, cu_q, cache.k.shape[2], keep)
    return kv_attention(q, cache, selected.page_table, selected.lengths, None, softmax_scale)[0]


__all__ = [
    "KVCache", "SelectedPages", "kv_cache_append", "kv_attention", "kv_attention_into", "kv_page_bounds", "kv_select_pages", "kv_decode", "HEAD_DIMS",
]  # fmt: skip
