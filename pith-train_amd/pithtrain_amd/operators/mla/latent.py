"""
The MLA layer while it answers: a cache of latent vectors and the absorbed form of its attention, backed by libpith_hip.so.

What the layer of pithtrain/models/deepseek_v2_lite.py:420-470 leaves behind for a token is one normalised latent vector (kv_lora_rank = 512
features, :430-435) and one rotated key part (64 features, :446-447), both shared by all heads. Training expands them to keys and values of every
head (kv_b_proj, then mla_assemble_qkv and attention); a token that is answered is cheaper in the latent space: with W_uk, W_uv the two halves of
kv_b_proj.weight of a head,

    q . [W_uk c | p] = (W_uk^T q_nope) . c + q_pe . p        and        sum_j P_j (W_uv c_j) = W_uv sum_j P_j c_j

    latent_cache_append   norm + rotation of new tokens, into cache pages (bf16, or e4m3 with one scale a row)
    absorb_query          q -> (W_uk^T q_nope, rotated q_pe)
    latent_attention      causal attention of the newest tokens of every sequence to its cached rows, or of a tree of drafted tokens
    absorb_value          its result -> W_uv of it, the input of o_proj
    latent_cache_gather   cached rows back as bf16, for the expanded form of a prompt behind a cached prefix (see there)
    latent_decode         the first four in a row: what stands between the layer's projections (MLA.decode calls it)

 T : new tokens of all sequences, one behind the other, b : sequences, h : heads.
Token counts, lengths, page tables, slots and tree masks are device tensors that only the kernels read: a captured graph follows their contents.
The operators serve; they have no backward. Arguments that require a gradient are refused while gradients are recorded.
"""

import os
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad

from pithtrain_amd import _C
from pithtrain_amd._ext import define_op

LATENT, ROPE, NOPE, VALUE = 512, 64, 128, 128  # what the kernels are built for (DeepSeek-V2-Lite)
MAX_DRAFTS = 64                                # tokens of a tree: bits of a mask word
FP8 = torch.float8_e4m3fn


class LatentCache(NamedTuple):
    """Pages of cached rows. latent [pages, page_size, 512] bf16 or float8_e4m3fn, k_pe [pages, page_size, 64] bf16, scale [pages, page_size] fp32
    (e4m3 only: a feature is value * scale of its row). page_size is a power of two from 16 to 65536; rows of a page are contiguous, pages may be
    further apart (the layers of a model can share one allocation) and begin at multiples of 16 bytes. Slot s is row s % page_size of page
    s // page_size."""

    latent: torch.Tensor
    k_pe: torch.Tensor
    scale: Optional[torch.Tensor] = None

    @classmethod
    def empty(cls, pages: int, page_size: int = 64, dtype: torch.dtype = torch.bfloat16, device="cuda") -> "LatentCache":
        """A cache with room for pages * page_size rows; rows hold nothing until latent_cache_append writes them."""
        assert dtype in (torch.bfloat16, FP8), f"the cache holds bfloat16 or float8_e4m3fn, not {dtype}"
        mk = lambda *s, dtype: torch.empty(pages, page_size, *s, dtype=dtype, device=device)  # noqa: E731
        return cls(mk(LATENT, dtype=dtype), mk(ROPE, dtype=torch.bfloat16), mk(dtype=torch.float32) if dtype == FP8 else None)


def _unit(t: torch.Tensor, what: str) -> None:
    assert t.shape[-1] == 1 or t.stride(-1) == 1, f"{what} is not contiguous along its last dim"


def _index(t: torch.Tensor, dtype: torch.dtype, shape: Tuple[int, ...], what: str) -> int:
    assert t.dtype == dtype and tuple(t.shape) == shape and t.is_contiguous(), f"{what} must be a contiguous {dtype} tensor of shape {list(shape)}, got {t.dtype} {list(t.shape)}"
    return t.data_ptr()


def _cache_args(like: torch.Tensor, latent: torch.Tensor, k_pe: torch.Tensor, scale: Optional[torch.Tensor]) -> "_C.LatentCacheArgs":
    _C.require_device(like, latent, k_pe, *(() if scale is None else (scale,)))
    assert latent.dtype in (torch.bfloat16, FP8) and latent.dim() == 3 and latent.shape[2] == LATENT, (
        f"cache.latent must be a bfloat16 or float8_e4m3fn [pages, page_size, {LATENT}] tensor, got {latent.dtype} {list(latent.shape)}"
    )
    pages, page_size, _ = latent.shape
    assert k_pe.dtype == torch.bfloat16 and tuple(k_pe.shape) == (pages, page_size, ROPE), "cache.k_pe does not match cache.latent"
    assert latent.stride()[1:] == (LATENT, 1) and k_pe.stride()[1:] == (ROPE, 1), "rows of a cache page are not contiguous"
    args = _C.LatentCacheArgs(
        latent=latent.data_ptr(), k_pe=k_pe.data_ptr(), pages=pages, page_size=page_size,
        latent_ps=latent.stride(0), k_pe_ps=k_pe.stride(0), dtype=_C.PITH_BF16,
    )  # fmt: skip
    if latent.dtype == FP8:
        assert scale is not None and scale.dtype == torch.float32 and tuple(scale.shape) == (pages, page_size), "an e4m3 cache needs a float32 scale [pages, page_size]"
        assert scale.stride(1) == 1, "scales of a cache page are not contiguous"
        args.scale, args.scale_ps, args.dtype = scale.data_ptr(), scale.stride(0), _C.PITH_FP8_E4M3
    else:
        assert scale is None, "a bfloat16 cache has no scale"
    return args


def _tables(cos: torch.Tensor, sin: torch.Tensor) -> int:
    assert cos.dtype == sin.dtype == torch.bfloat16, "cos and sin must be bfloat16"
    assert cos.dim() == 2 and cos.shape == sin.shape and cos.shape[1] == ROPE, f"cos and sin must be [positions, {ROPE}]"
    assert cos.is_contiguous() and sin.is_contiguous(), "cos or sin is not contiguous"
    return cos.shape[0]


def _checking(index: torch.Tensor) -> bool:
    """Whether index tensors are looked at on the host, at the price of a device synchronisation (never while a graph is captured)."""
    return os.environ.get("PITHTRAIN_AMD_CHECK_POSITIONS") == "1" and not (index.is_cuda and torch.cuda.is_current_stream_capturing())


def _check_positions(position_ids: torch.Tensor, positions: int) -> None:
    if _checking(position_ids) and position_ids.numel():
        lo, hi = int(position_ids.min()), int(position_ids.max())
        assert 0 <= lo and hi < positions, f"position_ids span [{lo}, {hi}], the rotary tables hold {positions} positions"


def _no_gradients(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """The ops' refusal, for calls that write into tensors of the caller's and so go past them."""
    recorded = torch.is_grad_enabled()
    for t in tensors:
        if t is not None and recorded and t.requires_grad:
            raise RuntimeError(f"{what} has no backward: call it under torch.no_grad(), or detach what requires a gradient")
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{what} has no forward-mode derivative")


def _launch(name: str, args, like: torch.Tensor) -> None:
    with torch.cuda.device(like.device):
        _C.check(getattr(_C.lib(), name)(_C.byref(args), _C.current_stream(like)))


# ---------------------------------------------------------------------------------------------
# Bodies of the ops for calls that the native path does not take (it words no errors), and their fake (shape) implementations.


def _aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy whose rows the kernels can read 16 bytes at a time."""
    ok = t.data_ptr() % 16 == 0 and all(st % 8 == 0 for n, st in zip(t.shape[:-1], t.stride()[:-1]) if n > 1) and (t.shape[-1] == 1 or t.stride(-1) == 1)
    return t if ok else t.clone(memory_format=torch.contiguous_format)  # (contiguous() would be t itself where only its beginning is off)


def _strides(t: torch.Tensor) -> Tuple[int, int]:
    """Token and head stride; those of a dimension of one element are never used and need not be multiples of 8."""
    t_ts, t_hs = t.stride(0), t.stride(1)
    return (t_ts if t.shape[0] > 1 else t.shape[1] * t.shape[2]), (t_hs if t.shape[1] > 1 else t.shape[2])


def _append_body(kv_a, weight, cos, sin, position_ids, slots, latent, k_pe, scale, eps):
    _C.require_device(kv_a, weight, cos, sin, position_ids, slots)
    assert kv_a.dtype == torch.bfloat16 and kv_a.dim() == 2 and kv_a.shape[1] == LATENT + ROPE, f"kv_a must be a bfloat16 [tokens, {LATENT + ROPE}] tensor, got {kv_a.dtype} {list(kv_a.shape)}"
    _unit(kv_a, "kv_a")
    t = kv_a.shape[0]
    assert tuple(weight.shape) == (LATENT,) and weight.is_contiguous(), f"weight must be a contiguous [{LATENT}] tensor"
    positions = _tables(cos, sin)
    cache = _cache_args(kv_a, latent, k_pe, scale)
    kv_a, weight = _aligned_rows(kv_a), _aligned_rows(weight)
    args = _C.LatentAppendArgs(
        kv_a=kv_a.data_ptr(), weight=weight.data_ptr(), cos=cos.data_ptr(), sin=sin.data_ptr(),
        position_ids=_index(position_ids, torch.int64, (t,), "position_ids"), slots=_index(slots, torch.int64, (t,), "slots"),
        T=t, P=positions, kv_a_rs=kv_a.stride(0) if t > 1 else LATENT + ROPE, eps=float(eps), weight_dtype=_C.dtype_code(weight), cache=cache,
    )  # fmt: skip
    if _checking(slots) and t:
        _check_positions(position_ids, positions)
        used = slots[slots >= 0]
        rows = latent.shape[0] * latent.shape[1]
        assert used.numel() == 0 or int(used.max()) < rows, f"slots go up to {int(used.max())}, the cache holds {rows} rows"
        assert used.unique().numel() == used.numel(), "two tokens name the same slot"
    _launch("pith_latent_append", args, kv_a)


def _append_fake(kv_a, weight, cos, sin, position_ids, slots, latent, k_pe, scale, eps):
    return None


def _table_args(page_table: torch.Tensor, b: int) -> Tuple[int, int, int]:
    assert page_table.dtype == torch.int32 and page_table.dim() == 2 and page_table.shape[0] == b, f"page_table must be an int32 [b={b}, pages] tensor, got {page_table.dtype} {list(page_table.shape)}"
    _unit(page_table, "page_table")
    width = page_table.shape[1]
    return page_table.data_ptr(), (page_table.stride(0) if b > 1 else width), width


def latent_cache_gather_into(cache: LatentCache, page_table: torch.Tensor, cu_rows: torch.Tensor, latent_out: torch.Tensor, k_pe_out: torch.Tensor) -> None:
    """latent_cache_gather into tensors of the caller's, [rows, 512] and [rows, 64] bf16 with rows of their own stride that begin at multiples of 16
    bytes; those from cu_rows[b] on keep what they hold."""
    _no_gradients("latent_cache_gather_into", *cache, latent_out, k_pe_out)
    _C.require_device(latent_out, k_pe_out, page_table, cu_rows)
    rows = latent_out.shape[0]
    for name, t, d in (("latent_out", latent_out, LATENT), ("k_pe_out", k_pe_out, ROPE)):
        assert t.dtype == torch.bfloat16 and tuple(t.shape) == (rows, d), f"{name} must be a bfloat16 [rows, {d}] tensor"
        _unit(t, name)
    assert cu_rows.dim() == 1 and cu_rows.numel() >= 1, "cu_rows must hold one more offset than there are sequences"
    b = cu_rows.numel() - 1
    args = _C.LatentGatherArgs(cache=_cache_args(latent_out, *cache), cu_rows=_index(cu_rows, torch.int32, (b + 1,), "cu_rows"),
                               latent_out=latent_out.data_ptr(), k_pe_out=k_pe_out.data_ptr(), B=b, rows=rows,
                               latent_rs=latent_out.stride(0) if rows > 1 else LATENT, k_pe_rs=k_pe_out.stride(0) if rows > 1 else ROPE)  # fmt: skip
    args.page_table, args.table_rs, args.table_width = _table_args(page_table, b)
    _launch("pith_latent_gather", args, latent_out)
    torch.autograd.graph.increment_version((latent_out, k_pe_out))


def _gather_body(latent, k_pe, scale, page_table, cu_rows, rows):
    assert rows >= 0, f"rows = {rows}"
    latent_out = torch.empty((rows, LATENT), dtype=torch.bfloat16, device=latent.device)
    k_pe_out = torch.empty((rows, ROPE), dtype=torch.bfloat16, device=latent.device)
    latent_cache_gather_into(LatentCache(latent, k_pe, scale), page_table, cu_rows, latent_out, k_pe_out)
    return latent_out, k_pe_out


def _gather_fake(latent, k_pe, scale, page_table, cu_rows, rows):
    return latent.new_empty((rows, LATENT), dtype=torch.bfloat16), latent.new_empty((rows, ROPE), dtype=torch.bfloat16)


def _absorb_args(x: torch.Tensor, weight: torch.Tensor, out: torch.Tensor, features: int, what: str):
    _C.require_device(x, weight)
    assert x.dtype == torch.bfloat16 and x.dim() == 3 and x.shape[2] == features, f"{what} must be a bfloat16 [tokens, heads, {features}] tensor, got {x.dtype} {list(x.shape)}"
    t, h, _ = x.shape
    assert weight.dtype == torch.bfloat16 and weight.numel() == h * (NOPE + VALUE) * LATENT and weight.shape[-1] == LATENT and weight.is_contiguous(), (
        f"kv_b_weight must be a contiguous bfloat16 [{h} * {NOPE + VALUE}, {LATENT}] tensor, got {weight.dtype} {list(weight.shape)}"
    )
    x, weight = _aligned_rows(x), _aligned_rows(weight)
    args = _C.LatentAbsorbArgs(x=x.data_ptr(), weight=weight.data_ptr(), out=out.data_ptr(), T=t, H=h, P=1)
    args.x_ts, args.x_hs = _strides(x)
    args.out_ts, args.out_hs = _strides(out)
    return args, (x, weight)


def _absorb_query_body(q, weight, cos, sin, position_ids):
    q_latent, q_pe = _absorb_query_fake(q, weight, cos, sin, position_ids)
    args, keep = _absorb_args(q, weight, q_latent, NOPE + ROPE, "q")
    _C.require_device(q, cos, sin, position_ids)
    args.P = _tables(cos, sin)
    args.cos, args.sin, args.position_ids = cos.data_ptr(), sin.data_ptr(), _index(position_ids, torch.int64, (q.shape[0],), "position_ids")
    args.q_pe = q_pe.data_ptr()
    args.q_pe_ts, args.q_pe_hs = _strides(q_pe)
    _check_positions(position_ids, args.P)
    _launch("pith_latent_absorb_query", args, q)
    del keep
    return q_latent, q_pe


def _absorb_query_fake(q, weight, cos, sin, position_ids):
    assert q.dim() == 3, "q must be [tokens, heads, features]"
    t, h, _ = q.shape
    return q.new_empty((t, h, LATENT)), q.new_empty((t, h, ROPE))


def _absorb_value_body(o_latent, weight):
    out = _absorb_value_fake(o_latent, weight)
    args, keep = _absorb_args(o_latent, weight, out, LATENT, "o_latent")
    _launch("pith_latent_absorb_value", args, o_latent)
    del keep
    return out


def _absorb_value_fake(o_latent, weight):
    assert o_latent.dim() == 3, "o_latent must be [tokens, heads, features]"
    t, h, _ = o_latent.shape
    return o_latent.new_empty((t, h, VALUE))


def latent_attention_into(
    q_latent: torch.Tensor, q_pe: torch.Tensor, cache: LatentCache, page_table: torch.Tensor, lengths: torch.Tensor, cu_q: torch.Tensor,
    softmax_scale: float, tree_mask: Optional[torch.Tensor], o: torch.Tensor, lse: torch.Tensor,
) -> None:  # fmt: skip
    """latent_attention into tensors of the caller's: o [T, h, 512] bf16, whose rows begin at multiples of 16 bytes, and lse [h, T] fp32; neither overlaps
    what the call reads. Tokens from cu_q[b] on keep what they hold."""
    _no_gradients("latent_attention_into", q_latent, q_pe, *cache, o, lse)
    _C.require_device(q_latent, q_pe, page_table, lengths, cu_q, o, lse)
    assert q_latent.dtype == torch.bfloat16 and q_latent.dim() == 3 and q_latent.shape[2] == LATENT, f"q_latent must be a bfloat16 [tokens, heads, {LATENT}] tensor, got {q_latent.dtype} {list(q_latent.shape)}"
    t, h, _ = q_latent.shape
    assert q_pe.dtype == torch.bfloat16 and tuple(q_pe.shape) == (t, h, ROPE), f"q_pe must be a bfloat16 [{t}, {h}, {ROPE}] tensor, got {q_pe.dtype} {list(q_pe.shape)}"
    assert o.dtype == torch.bfloat16 and tuple(o.shape) == (t, h, LATENT), "o has the wrong dtype or shape"
    assert lse.dtype == torch.float32 and tuple(lse.shape) == (h, t), "lse has the wrong dtype or shape"
    _unit(o, "o")
    _unit(lse, "lse")
    assert lengths.dim() == 1, "lengths must be one-dimensional"
    b = lengths.shape[0]
    q_latent, q_pe = _aligned_rows(q_latent), _aligned_rows(q_pe)
    args = _C.LatentAttnArgs(
        q_latent=q_latent.data_ptr(), q_pe=q_pe.data_ptr(), cache=_cache_args(q_latent, *cache),
        lengths=_index(lengths, torch.int32, (b,), "lengths"), cu_q=_index(cu_q, torch.int32, (b + 1,), "cu_q"),
        o=o.data_ptr(), lse=lse.data_ptr(), T=t, B=b, H=h, lse_hs=lse.stride(0) if h > 1 else t, scale=float(softmax_scale),
    )  # fmt: skip
    args.page_table, args.table_rs, args.table_width = _table_args(page_table, b)
    args.q_ts, args.q_hs = _strides(q_latent)
    args.q_pe_ts, args.q_pe_hs = _strides(q_pe)
    args.o_ts, args.o_hs = _strides(o)
    if tree_mask is not None:
        _C.require_device(q_latent, tree_mask)
        args.tree_mask = _index(tree_mask, torch.int64, (t,), "tree_mask")
        if _checking(cu_q) and b:
            assert int((cu_q[1:] - cu_q[:-1]).max()) <= MAX_DRAFTS, f"a tree has more than {MAX_DRAFTS} tokens"
    with torch.cuda.device(q_latent.device):
        need = _C.lib().pith_latent_attn_workspace_bytes(_C.byref(args))
        workspace = torch.empty(need, dtype=torch.uint8, device=q_latent.device)
        args.workspace, args.workspace_bytes = workspace.data_ptr(), need
        _C.check(_C.lib().pith_latent_attn(_C.byref(args), _C.current_stream(q_latent)))
    torch.autograd.graph.increment_version((o, lse))  # (a backward that saved one of them notices)


def _attention_body(q_latent, q_pe, latent, k_pe, scale, page_table, lengths, cu_q, softmax_scale, tree_mask):
    o, lse = _attention_fake(q_latent, q_pe, latent, k_pe, scale, page_table, lengths, cu_q, softmax_scale, tree_mask)
    latent_attention_into(q_latent, q_pe, LatentCache(latent, k_pe, scale), page_table, lengths, cu_q, softmax_scale, tree_mask, o, lse)
    return o, lse


def _attention_fake(q_latent, q_pe, latent, k_pe, scale, page_table, lengths, cu_q, softmax_scale, tree_mask):
    assert q_latent.dim() == 3, "q_latent must be [tokens, heads, features]"
    t, h, d = q_latent.shape
    return q_latent.new_empty((t, h, d)), q_latent.new_empty((h, t), dtype=torch.float32)


_append_op = define_op("latent_append", _append_body, _append_fake)
_gather_op = define_op("latent_gather", _gather_body, _gather_fake)
_absorb_query_op = define_op("latent_absorb_query", _absorb_query_body, _absorb_query_fake)
_absorb_value_op = define_op("latent_absorb_value", _absorb_value_body, _absorb_value_fake)
_attention_op = define_op("latent_attention", _attention_body, _attention_fake)


# ---------------------------------------------------------------------------------------------


def latent_cache_append(
    kv_a: torch.Tensor, weight: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, position_ids: torch.Tensor, slots: torch.Tensor,
    cache: LatentCache, eps: float = 1e-6,
) -> None:  # fmt: skip
    """Rows of new tokens into the cache: rms_norm(kv_a[:, :512], eps) * weight and the rotated kv_a[:, 512:], each rounded once from fp32. kv_a
    [T, 576] bf16 is the output of kv_a_proj_with_mqa, weight [512] (bf16 or fp32) that of kv_a_layernorm, cos / sin [positions, 64] bf16 the rotary
    module's tables (the rotation is mla_assemble_qkv's), position_ids and slots [T] int64. An e4m3 row's scale is its largest magnitude / 448.
    Tokens with a slot below 0 or beyond the cache are skipped (padding). Two tokens of a call must not share a slot; positions beyond the tables are
    clamped to them (PITHTRAIN_AMD_CHECK_POSITIONS=1 raises in all these cases but padding, at the price of a device synchronisation)."""
    _append_op(kv_a, weight, cos, sin, position_ids, slots, cache.latent, cache.k_pe, cache.scale, eps)


def latent_cache_gather(cache: LatentCache, page_table: torch.Tensor, cu_rows: torch.Tensor, rows: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """(latent [rows, 512], k_pe [rows, 64]) bf16: the first cu_rows[i + 1] - cu_rows[i] cached rows of every sequence i, one sequence behind the
    other. page_table [b, n] int32: the pages of each; cu_rows [b + 1] int32 ascending from 0, on the device; rows: how many to make room for, at
    least cu_rows[b]. Rows from cu_rows[b] on are not written.

    With kv_b_proj the rows become keys in two parts and values, for the expanded form of a prompt behind a cached prefix: _mla_fwd(q, k_nope, v, scale,
    causal=False, k_pe=k_pe) of the rotated queries over the prefix (k_pe is rotated already; mla_assemble_qkv would do it again), _mla_fwd(..., causal=True) of
    the prompt over itself, and _online_softmax_combine_log2 of the two."""
    return _gather_op(cache.latent, cache.k_pe, cache.scale, page_table, cu_rows, rows)


def absorb_query(q: torch.Tensor, kv_b_weight: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, position_ids: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q_latent [T, h, 512], q_pe [T, h, 64]) of q [T, h, 192] bf16: its first 128 features times W_uk, its last 64 rotated. kv_b_weight is
    kv_b_proj.weight, [h * 256, 512] bf16, of whose 256 rows a head the first 128 are W_uk. Tables and position_ids as in latent_cache_append."""
    return _absorb_query_op(q, kv_b_weight, cos, sin, position_ids)


def absorb_value(o_latent: torch.Tensor, kv_b_weight: torch.Tensor) -> torch.Tensor:
    """o [T, h, 128] = W_uv o_latent of every head, W_uv the last 128 of its 256 rows of kv_b_weight (see absorb_query)."""
    return _absorb_value_op(o_latent, kv_b_weight)


def latent_attention(
    q_latent: torch.Tensor, q_pe: torch.Tensor, cache: LatentCache, page_table: torch.Tensor, lengths: torch.Tensor, cu_q: torch.Tensor,
    softmax_scale: float, tree_mask: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:  # fmt: skip
    """(o_latent [T, h, 512] bf16, lse [h, T] fp32 in base 2): attention of the newest tokens of b sequences to their cached rows.

    Tokens cu_q[i] .. cu_q[i + 1] - 1 are the n newest of sequence i, whose lengths[i] cached rows (theirs included: append them first) lie in the
    pages page_table[i]. Token k of them sees the rows up to lengths[i] - n + k; with tree_mask ([T] int64) all rows in front of the n newest, and of
    those row j where bit j of the token's word is set (tree_mask_of makes such words; n is at most 64). A token that sees no row gets 0 and an lse
    of -inf. Tokens from cu_q[b] on are not written. The same call gives the same bits; in a batch of other sequences a token's last bits may differ.
    page_table [b, pages], lengths [b] and cu_q [b + 1] are int32, on the device."""
    return _attention_op(q_latent, q_pe, cache.latent, cache.k_pe, cache.scale, page_table, lengths, cu_q, softmax_scale, tree_mask)


def tree_mask_of(parents: torch.Tensor) -> torch.Tensor:
    """Words for latent_attention from parents [..., n] (n at most 64): draft j of a tree hangs on draft parents[j] of the same tree, or on the
    sequence itself where that is negative (or n or more: no draft of this tree), and sees its ancestors and itself. Every parent comes
    before its children. int64 [..., n]. PITHTRAIN_AMD_CHECK_POSITIONS=1 raises for parents beyond the tree, at the price of a device synchronisation."""
    n = parents.shape[-1]
    assert n <= MAX_DRAFTS, f"a tree has at most {MAX_DRAFTS} tokens, got {n}"
    if _checking(parents) and parents.numel():
        assert int(parents.max()) < n, f"a parent is draft {int(parents.max())}, the tree has {n} drafts"
    own = torch.ones((), dtype=torch.int64, device=parents.device) << torch.arange(n, device=parents.device)
    words = own.expand(parents.shape).clone()
    at = parents = torch.where(parents < n, parents.long(), -1)
    for _ in range(n):  # one step up the tree for all drafts at once
        words |= torch.where(at >= 0, own[at.clamp(0, max(n - 1, 0))] if n else own, 0)
        at = torch.where(at >= 0, parents.gather(-1, at.clamp(min=0)), at)
    return words


def latent_decode(
    q: torch.Tensor, kv_a: torch.Tensor, norm_weight: torch.Tensor, kv_b_weight: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
    position_ids: torch.Tensor, slots: torch.Tensor, cache: LatentCache, page_table: torch.Tensor, lengths: torch.Tensor, cu_q: torch.Tensor,
    softmax_scale: float, eps: float = 1e-6, tree_mask: Optional[torch.Tensor] = None,
) -> torch.Tensor:  # fmt: skip
    """The layer between its projections for new tokens, o [T, h, 128]: their rows go into the cache, then q [T, h, 192] attends to the cached rows
    of its sequences (lengths count the new rows). Five launches, or six for very many rows; arguments as in the functions above. Rows of o from
    cu_q[b] on hold nothing. What is refused for q, kv_a, a weight, the tables, the cache or a gradient has written nothing; page_table, lengths, cu_q and
    tree_mask are looked at when the new rows are in the cache (the same call with the right ones writes them again)."""
    q_latent, q_pe = absorb_query(q, kv_b_weight, cos, sin, position_ids)  # first: what it refuses must leave the cache as it was
    latent_cache_append(kv_a, norm_weight, cos, sin, position_ids, slots, cache, eps)
    o_latent, _ = latent_attention(q_latent, q_pe, cache, page_table, lengths, cu_q, softmax_scale, tree_mask)
    return absorb_value(o_latent, kv_b_weight)


__all__ = [
    "LatentCache", "latent_cache_append", "latent_cache_gather", "latent_cache_gather_into", "absorb_query", "absorb_value", "latent_attention",
    "latent_attention_into", "latent_decode", "tree_mask_of", "MAX_DRAFTS",
]  # fmt: skip
