"""The latent cache's operators on a machine without a GPU: the oracle's pins, the C interface of include/pith_latent.h, what the Python entry points
refuse, and their shape propagation."""

import ctypes
import math
import os
import re
import subprocess
import sys

import pytest
import torch

from oracle import latent_oracle as O
from oracle import prologue_oracle as P
from pithtrain_amd import _C
from pithtrain_amd.operators.mla import MLA
from pithtrain_amd.operators.mla import latent as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "pith_latent.h")
BF = torch.bfloat16


# ---------------------------------------------------------------------------------------------
# The oracle


def _layer(s, h, seed):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *sh: torch.randn(*sh, generator=g, dtype=torch.float64)  # noqa: E731
    cos, sin = P.cos_sin_table(torch.arange(s + 5), 64)
    return mk(s, h, 192), mk(s, 576), mk(512), mk(h * 256, 512) / 20, cos, sin, torch.arange(s) + 3


def test_absorbed_form_equals_the_expanded_layer():
    """Queries in the latent space against the rows themselves, then W_uv: the layer as the reference writes it, to rounding of fp64."""
    s, h, scale = 23, 3, 192**-0.5
    q, kv_a, w, kv_b, cos, sin, pos = _layer(s, h, 1)
    n, pe = O.append_rows(kv_a, w, cos, sin, pos, 1e-6)
    want = O.expanded(q, n, pe, kv_b, cos, sin, pos, scale)
    q_latent, _ = O.absorb_query(q, kv_b)
    o, lse, mass, _ = O.attention(q_latent, O.rotate(q[..., 128:], cos, sin, pos), n, pe, O.sees(s, s), scale)
    got, _ = O.absorb_value(o, kv_b)
    assert (got - want).abs().max() < 1e-11 * want.abs().max()
    assert (mass >= o.abs() - 1e-12).all()
    # the rows in two pieces, joined by their lse
    a, la, _, _ = O.attention(q_latent[-1:], O.rotate(q[-1:, :, 128:], cos, sin, pos[-1:]), n[:9], pe[:9], O.sees(1, 9), scale)
    b, lb, _, _ = O.attention(q_latent[-1:], O.rotate(q[-1:, :, 128:], cos, sin, pos[-1:]), n[9:], pe[9:], O.sees(1, s - 9), scale)
    wa, wb = (torch.exp2(x - lse[:, -1:]).T[..., None] for x in (la, lb))
    assert (wa * a + wb * b - o[-1:]).abs().max() < 1e-12


def test_rows_of_the_norm_and_the_rotation():
    g = torch.Generator().manual_seed(2)
    kv_a, ones = torch.randn(7, 576, generator=g, dtype=torch.float64), torch.ones(512, dtype=torch.float64)
    cos, sin = P.cos_sin_table(torch.arange(9), 64)
    n, pe = O.append_rows(kv_a, ones, cos, sin, torch.tensor([0, 1, 2, 3, 4, 8, 0]), 0.0)
    assert torch.allclose(n.square().mean(-1), torch.ones(7, dtype=torch.float64))
    assert torch.allclose(n, torch.nn.functional.rms_norm(kv_a[:, :512], (512,), eps=0.0))
    assert torch.equal(pe[0], P.deinterleave(kv_a[0, 512:]))  # position 0: no turn
    assert torch.allclose(pe.norm(dim=-1), kv_a[:, 512:].norm(dim=-1))


def test_visibility_by_words_of_a_chain_is_causal():
    chain = L.tree_mask_of(torch.arange(-1, 11))
    assert torch.equal(O.sees(12, 30, chain), O.sees(12, 30))


def test_tree_words_from_parents():
    parents = torch.tensor([[-1, 0, 0, 2, -1, 3], [-1, 0, 1, 2, 3, 4]])
    words = L.tree_mask_of(parents)
    for row, p in zip(words.tolist(), parents.tolist()):
        for j, w in enumerate(row):
            want, at = 0, j
            while at >= 0:
                want |= 1 << at
                at = p[at]
            assert w == want
    full = L.tree_mask_of(torch.arange(-1, 63))
    assert int(full[63]) == -1 and int(full[62]) == (1 << 63) - 1
    assert L.tree_mask_of(torch.empty(0, dtype=torch.int64)).shape == (0,)
    with pytest.raises(AssertionError, match="at most 64"):
        L.tree_mask_of(torch.arange(-1, 64))


@pytest.mark.parametrize("far", [3, 64, 2**31, 2**62])
def test_a_parent_that_is_no_draft_of_the_tree_is_none(far, monkeypatch):
    """On a GPU an index behind the last draft would end the process, not raise."""
    parents = torch.tensor([[-1, 0, 1], [far, 0, far], [-far, -1, far]])
    monkeypatch.delenv("PITHTRAIN_AMD_CHECK_POSITIONS", raising=False)
    assert L.tree_mask_of(parents).tolist() == [[1, 3, 7], [1, 3, 4], [1, 2, 4]]
    monkeypatch.setenv("PITHTRAIN_AMD_CHECK_POSITIONS", "1")
    with pytest.raises(AssertionError, match="the tree has 3 drafts"):
        L.tree_mask_of(parents)
    assert L.tree_mask_of(parents[:1]).tolist() == [[1, 3, 7]]


# ---------------------------------------------------------------------------------------------
# The C interface


def test_library_exports_every_declared_symbol():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(pith_latent_[a-z0-9_]+)\s*\(", text)))
    assert sorted(_C.LATENT_SYMBOLS) == declared
    for name in declared:
        assert hasattr(_C.lib(), name), f"{name} is declared in pith_latent.h but not exported"


STRUCTS = {
    "pith_latent_cache": _C.LatentCacheArgs, "pith_latent_append_args": _C.LatentAppendArgs, "pith_latent_gather_args": _C.LatentGatherArgs,
    "pith_latent_absorb_args": _C.LatentAbsorbArgs, "pith_latent_attn_args": _C.LatentAttnArgs,
}  # fmt: skip
# struct sizes of a version of this part of the interface: a change here needs a new version
STRUCT_SIZES = {100: {"pith_latent_cache": 72, "pith_latent_append_args": 152, "pith_latent_gather_args": 152, "pith_latent_absorb_args": 128, "pith_latent_attn_args": 256}}


def test_struct_layouts_match_the_header(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "pith_latent.h"', 'int main(void){printf("version %d\\n", PITH_LATENT_VERSION);']
    for cname, st in STRUCTS.items():
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in st._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.strip().splitlines())
    assert int(got["version"]) == _C.PITH_LATENT_VERSION == _C.lib().pith_latent_version()
    for cname, st in STRUCTS.items():
        assert int(got[cname]) == ctypes.sizeof(st) == STRUCT_SIZES[_C.PITH_LATENT_VERSION][cname], cname
        for f, _ in st._fields_:
            assert int(got[f"{cname}.{f}"]) == getattr(st, f).offset, f"{cname}.{f}"


@pytest.mark.parametrize("symbol, version", [("pith_latent_version", 100), ("pith_latent_version", 99), ("pith_version", 1)])
def test_the_native_path_is_loaded_with_its_own_version_only(tmp_path, symbol, version):
    """A library of another version lays arguments out differently. One symbol of it is put in front of the built library's."""
    src, shim = tmp_path / "shim.c", tmp_path / "shim.so"
    src.write_text(f"int {symbol}(void) {{ return {version}; }}\n")
    subprocess.run(["gcc", "-shared", "-fPIC", str(src), "-o", str(shim)], check=True)
    code = f"import ctypes; ctypes.CDLL({str(shim)!r}, ctypes.RTLD_GLOBAL); from pithtrain_amd import _ext"
    env = {**os.environ, "PYTHONPATH": os.path.join(ROOT, "pith-train_amd")}
    run = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True)
    if version == _C.PITH_LATENT_VERSION:
        assert run.returncode == 0, run.stderr
    else:
        assert run.returncode == 1 and "build both again" in run.stderr, run.stderr


def _cache(**kw):
    base = dict(latent=256, k_pe=256, scale=None, pages=8, page_size=64, latent_ps=64 * 512, k_pe_ps=64 * 64, scale_ps=0, dtype=_C.PITH_BF16)
    return _C.LatentCacheArgs(**{**base, **kw})


def _append(**kw):
    base = dict(kv_a=256, weight=256, cos=256, sin=256, position_ids=256, slots=256, T=4, P=16, kv_a_rs=576, eps=1e-6, weight_dtype=_C.PITH_BF16, cache=_cache())
    return _C.LatentAppendArgs(**{**base, **kw})


def _gather(**kw):
    base = dict(cache=_cache(), page_table=256, cu_rows=256, latent_out=256, k_pe_out=256, B=2, rows=10, table_rs=4, table_width=4, latent_rs=512, k_pe_rs=64)
    return _C.LatentGatherArgs(**{**base, **kw})


def _absorb(**kw):
    base = dict(x=256, weight=256, out=256, q_pe=256, cos=256, sin=256, position_ids=256, T=4, H=2, P=16, x_ts=1024, x_hs=512, out_ts=1024, out_hs=512, q_pe_ts=128, q_pe_hs=64)
    return _C.LatentAbsorbArgs(**{**base, **kw})


def _attn(**kw):
    base = dict(q_latent=256, q_pe=256, cache=_cache(), page_table=256, lengths=256, cu_q=256, tree_mask=None, o=256, lse=256, workspace=256, workspace_bytes=1 << 40,
                T=4, B=2, H=2, table_rs=4, table_width=4, q_ts=1024, q_hs=512, q_pe_ts=128, q_pe_hs=64, o_ts=1024, o_hs=512, lse_hs=4, scale=0.07)  # fmt: skip
    return _C.LatentAttnArgs(**{**base, **kw})


NULL, SHAPE, DTYPE, UNSUPPORTED, ALIGN = (_C.PITH_ERR_NULL_POINTER, _C.PITH_ERR_BAD_SHAPE, _C.PITH_ERR_BAD_DTYPE, _C.PITH_ERR_UNSUPPORTED, _C.PITH_ERR_MISALIGNED)
FP8 = dict(dtype=_C.PITH_FP8_E4M3, scale=256, scale_ps=64)
BAD_CACHES = [
    (dict(dtype=1), DTYPE), (dict(latent=None), NULL), (dict(k_pe=None), NULL), (dict(dtype=_C.PITH_FP8_E4M3), NULL), (dict(page_size=8), SHAPE),
    (dict(page_size=48), SHAPE), (dict(page_size=1 << 17), SHAPE), (dict(pages=0), SHAPE), (dict(pages=1 << 26), SHAPE), (dict(latent_ps=64 * 512 - 8), SHAPE),
    (dict(k_pe_ps=64 * 64 - 8), SHAPE), (dict(latent=264), ALIGN), (dict(latent_ps=64 * 512 + 4), ALIGN), (dict(k_pe_ps=64 * 64 + 4), ALIGN),
    ({**FP8, "scale_ps": 63}, SHAPE), ({**FP8, "scale": 258}, ALIGN), ({**FP8, "latent_ps": 64 * 512 + 8}, ALIGN),
]  # fmt: skip
CALLS = {
    "pith_latent_append": (_append, [
        (dict(kv_a=None), NULL), (dict(slots=None), NULL), (dict(T=-1), SHAPE), (dict(P=0), SHAPE), (dict(kv_a_rs=568), SHAPE), (dict(kv_a_rs=580), ALIGN),
        (dict(kv_a=264), ALIGN), (dict(weight=264), ALIGN), (dict(slots=260), ALIGN), (dict(weight_dtype=2), DTYPE)]),
    "pith_latent_gather": (_gather, [
        (dict(page_table=None), NULL), (dict(k_pe_out=None), NULL), (dict(B=-1), SHAPE), (dict(rows=-1), SHAPE), (dict(rows=1 << 31), SHAPE), (dict(table_width=0), SHAPE),
        (dict(table_rs=3), SHAPE), (dict(latent_rs=504), SHAPE), (dict(latent_rs=516), ALIGN), (dict(latent_out=264), ALIGN)]),
    "pith_latent_absorb_query": (_absorb, [
        (dict(x=None), NULL), (dict(q_pe=None), NULL), (dict(position_ids=None), NULL), (dict(T=-1), SHAPE), (dict(H=0), SHAPE), (dict(P=0), SHAPE), (dict(x_hs=184), SHAPE),
        (dict(out_ts=504), SHAPE), (dict(q_pe_hs=56), SHAPE), (dict(x_ts=1028), ALIGN), (dict(weight=264), ALIGN), (dict(q_pe=264), ALIGN), (dict(q_pe_ts=132), ALIGN)]),
    "pith_latent_absorb_value": (_absorb, [
        (dict(x=None), NULL), (dict(out=None), NULL), (dict(T=1 << 21), SHAPE), (dict(H=2000), SHAPE), (dict(x_hs=504), SHAPE), (dict(out_hs=120), SHAPE), (dict(out=264), ALIGN)]),
    "pith_latent_attn": (_attn, [
        (dict(q_latent=None), NULL), (dict(lengths=None), NULL), (dict(workspace=None), NULL), (dict(lse=None), NULL), (dict(page_table=None), NULL), (dict(T=-1), SHAPE),
        (dict(H=0), SHAPE), (dict(H=2000), SHAPE), (dict(table_width=0), SHAPE), (dict(table_rs=3), SHAPE), (dict(q_hs=504), SHAPE), (dict(o_ts=504), SHAPE),
        (dict(lse_hs=3), SHAPE), (dict(workspace_bytes=64), SHAPE), (dict(table_width=1 << 26, table_rs=1 << 26), UNSUPPORTED),
        (dict(T=1 << 20, H=1024, lse_hs=1 << 20, table_width=1 << 10, table_rs=1 << 10), UNSUPPORTED), (dict(q_latent=264), ALIGN), (dict(q_pe_hs=68), ALIGN),
        (dict(o_ts=1028), ALIGN), (dict(workspace=384), ALIGN), (dict(tree_mask=260), ALIGN)]),
}  # fmt: skip


@pytest.mark.parametrize("name", CALLS)
def test_bad_arguments_are_rejected_before_anything_is_launched(name):
    """There is no device here, so a launch would show as PITH_ERR_LAUNCH."""
    make, bad = CALLS[name]
    fn = getattr(_C.lib(), name)
    assert fn(None, None) == NULL
    with_cache = [] if make is _absorb else [(dict(cache=_cache(**kw)), code) for kw, code in BAD_CACHES]
    for kw, code in bad + with_cache:
        assert fn(ctypes.byref(make(**kw)), None) == code, (kw, _C.lib().pith_last_error())
        assert _C.lib().pith_last_error().startswith(name.encode())


@pytest.mark.parametrize("name", CALLS)
def test_empty_calls_launch_nothing(name):
    make, _ = CALLS[name]
    fn = getattr(_C.lib(), name)
    empty = [dict(rows=0), dict(B=0)] if make is _gather else [dict(T=0), dict(B=0)] if make is _attn else [dict(T=0)]
    for kw in empty:
        assert fn(ctypes.byref(make(**kw)), None) == _C.PITH_OK


@pytest.mark.parametrize("fp8", [False, True])
def test_the_stride_of_a_single_page_is_not_used(fp8):
    """A tensor whose first dimension has one element may carry any stride there."""
    odd = dict(pages=1, latent_ps=515, k_pe_ps=3, **(dict(FP8, scale_ps=1) if fp8 else {}))
    for name, (make, _) in CALLS.items():
        if make is not _absorb:
            args = make(cache=_cache(**odd), **({"rows": 0} if make is _gather else {"T": 0}))
            assert getattr(_C.lib(), name)(ctypes.byref(args), None) == _C.PITH_OK, _C.lib().pith_last_error()


def test_workspace_grows_with_nothing_but_the_device_and_the_row_blocks():
    need = lambda **kw: _C.lib().pith_latent_attn_workspace_bytes(ctypes.byref(_attn(**kw)))  # noqa: E731
    assert need(T=0) == need(B=0) == 0 and need() > 0
    assert need(table_width=4096, table_rs=4096) == need()  # whatever the lengths
    assert need(T=1000, lse_hs=1000) - need() < 1 << 20
    assert need(H=0) == 0  # what pith_latent_attn rejects


def test_rows_of_a_workgroup_go_by_the_rows_of_a_sequence_and_the_work_list():
    rows = lambda **kw: _C.lib().pith_latent_attn_rows(ctypes.byref(_attn(**kw)))  # noqa: E731
    wide = dict(table_width=4096, table_rs=4096)
    assert rows(T=0) == rows(B=0) == rows(H=0) == 0  # nothing to launch, or what pith_latent_attn rejects
    assert rows(T=2, H=16, lse_hs=2, **wide) == 16  # sixteen rows a sequence
    assert rows(T=3, H=16, lse_hs=3, **wide) == 64
    assert rows(T=2, H=17, lse_hs=2, **wide) == 64
    assert rows(T=64, H=128, lse_hs=64) == 64 and rows(T=3, H=16, lse_hs=3) == 16  # and a work list of some length


# ---------------------------------------------------------------------------------------------
# The Python entry points


def _zeros(*s, d=BF, dev="cpu"):
    return torch.zeros(*s, dtype=d, device=dev)


def _calls(dev):
    z = lambda *s, d=BF: _zeros(*s, d=d, dev=dev)  # noqa: E731
    i32, i64 = torch.int32, torch.int64
    cache = L.LatentCache(z(4, 16, 512), z(4, 16, 64))
    return {
        "append": lambda: L.latent_cache_append(z(3, 576), z(512), z(8, 64), z(8, 64), z(3, d=i64), z(3, d=i64), cache),
        "gather": lambda: L.latent_cache_gather(cache, z(2, 2, d=i32), z(3, d=i32), 5),
        "query": lambda: L.absorb_query(z(3, 2, 192), z(512, 512), z(8, 64), z(8, 64), z(3, d=i64)),
        "value": lambda: L.absorb_value(z(3, 2, 512), z(512, 512)),
        "attention": lambda: L.latent_attention(z(3, 2, 512), z(3, 2, 64), cache, z(2, 2, d=i32), z(2, d=i32), z(3, d=i32), 0.1),
    }


@pytest.mark.parametrize("name", _calls("cpu"))
def test_cpu_tensors_are_refused(name):
    with pytest.raises(RuntimeError, match="need tensors on a GPU"):
        _calls("cpu")[name]()


def test_shapes_propagate_without_a_device():
    calls = _calls("meta")
    assert calls["append"]() is None
    assert [tuple(t.shape) for t in calls["gather"]()] == [(5, 512), (5, 64)]
    assert [tuple(t.shape) for t in calls["query"]()] == [(3, 2, 512), (3, 2, 64)]
    assert calls["value"]().shape == (3, 2, 128)
    o, lse = calls["attention"]()
    assert (o.shape, o.dtype, lse.shape, lse.dtype) == ((3, 2, 512), BF, (2, 3), torch.float32)


def test_arguments_that_require_a_gradient_are_refused():
    w, x = _zeros(512, 512), _zeros(3, 2, 512).requires_grad_()
    with pytest.raises(RuntimeError, match="has no backward"):
        L.absorb_value(x, w)
    with pytest.raises(RuntimeError, match="has no backward"):
        L.absorb_value(x.detach(), w.requires_grad_())
    with torch.no_grad(), pytest.raises(RuntimeError, match="need tensors on a GPU"):
        L.absorb_value(x, w)


def _into_calls():
    """Calls into tensors of the caller's, with every tensor that could record a gradient."""
    z, i32 = _zeros, torch.int32
    gather = [z(4, 16, 512), z(4, 16, 64), z(5, 512), z(5, 64)]
    gather8 = [z(4, 16, 512, d=L.FP8), z(4, 16, 64), z(4, 16, d=torch.float32), z(5, 512), z(5, 64)]
    attention = [z(3, 2, 512), z(3, 2, 64), z(4, 16, 512), z(4, 16, 64), z(3, 2, 512), z(2, 3, d=torch.float32)]
    return {
        "gather": (gather, lambda c, p, o, op: L.latent_cache_gather_into(L.LatentCache(c, p), z(2, 2, d=i32), z(3, d=i32), o, op)),
        "gather_e4m3": (gather8, lambda c, p, s, o, op: L.latent_cache_gather_into(L.LatentCache(c, p, s), z(2, 2, d=i32), z(3, d=i32), o, op)),
        "attention": (attention, lambda q, qp, c, p, o, lse: L.latent_attention_into(q, qp, L.LatentCache(c, p), z(2, 2, d=i32), z(2, d=i32), z(3, d=i32), 0.1, None, o, lse)),
    }


@pytest.mark.parametrize("name", _into_calls())
def test_calls_into_given_tensors_refuse_gradients(name):
    tensors, call = _into_calls()[name]
    for i, t in enumerate(tensors):
        if t.dtype == L.FP8:
            continue
        one = [x.clone().requires_grad_() if k == i else x for k, x in enumerate(tensors)]
        with pytest.raises(RuntimeError, match="has no backward"):
            call(*one)
        for mode in (torch.no_grad, torch.inference_mode):
            with mode(), pytest.raises(RuntimeError, match="need tensors on a GPU"):
                call(*one)
        with torch.autograd.forward_ad.dual_level(), torch.no_grad(), pytest.raises(RuntimeError, match="has no forward-mode derivative"):
            one[i] = torch.autograd.forward_ad.make_dual(t, t)
            call(*one)


@pytest.mark.parametrize("name", _calls("cpu"))
def test_tangents_are_refused(name):
    """Forward-mode derivatives would be left out of the result in silence."""
    forward_ad = torch.autograd.forward_ad
    with forward_ad.dual_level():
        dual = lambda *s, d=BF: forward_ad.make_dual(_zeros(*s, d=d, dev="meta"), _zeros(*s, d=d, dev="meta"))  # noqa: E731
        z = lambda *s, d=BF: _zeros(*s, d=d, dev="meta")  # noqa: E731
        i32, i64 = torch.int32, torch.int64
        cache = L.LatentCache(z(4, 16, 512), dual(4, 16, 64))
        call = {
            "append": lambda: L.latent_cache_append(dual(3, 576), z(512), z(8, 64), z(8, 64), z(3, d=i64), z(3, d=i64), L.LatentCache(z(4, 16, 512), z(4, 16, 64))),
            "gather": lambda: L.latent_cache_gather(cache, z(2, 2, d=i32), z(3, d=i32), 5),
            "query": lambda: L.absorb_query(z(3, 2, 192), dual(512, 512), z(8, 64), z(8, 64), z(3, d=i64)),
            "value": lambda: L.absorb_value(dual(3, 2, 512), z(512, 512)),
            "attention": lambda: L.latent_attention(z(3, 2, 512), z(3, 2, 64), cache, z(2, 2, d=i32), z(2, d=i32), z(3, d=i32), 0.1),
        }[name]
        for mode in (torch.no_grad, torch.enable_grad):
            with mode(), pytest.raises(RuntimeError, match="has no forward-mode derivative"):
                call()
        with torch.inference_mode():  # (no tangents there)
            call()


@pytest.mark.parametrize("mode", [torch.no_grad, torch.enable_grad, torch.inference_mode])
@pytest.mark.parametrize("dtype", [BF, L.FP8])
def test_appending_counts_as_a_change_of_the_cache(dtype, mode):
    """A backward that saved a tensor of the cache (or a view that shares it) must not take its new rows for the old ones."""
    layers = L.LatentCache.empty(8, 16, dtype, "meta")
    cache = L.LatentCache(*(None if t is None else t[::2] for t in layers))
    gradient = torch.ones(4, 16, 64, dtype=BF, device="meta", requires_grad=True)
    y = gradient * cache.k_pe
    before = [t._version for t in layers if t is not None]
    with mode():
        L.latent_cache_append(*(t.to("meta") for t in (_zeros(3, 576), _zeros(512), _zeros(8, 64), _zeros(8, 64), _zeros(3, d=torch.int64), _zeros(3, d=torch.int64))), cache)
    assert all(t._version > v for t, v in zip([t for t in layers if t is not None], before))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("name", ["q", "kv_a", "norm_weight", "kv_b_weight", "cos", "latent", "k_pe"])
def test_a_decoding_step_that_is_refused_for_a_gradient_writes_nothing(name):
    z, i32, i64 = (lambda *s, d=BF: _zeros(*s, d=d, dev="meta")), torch.int32, torch.int64
    t = dict(q=z(2, 2, 192), kv_a=z(2, 576), norm_weight=z(512), kv_b_weight=z(512, 512), cos=z(8, 64), sin=z(8, 64), position_ids=z(2, d=i64), slots=z(2, d=i64),
             latent=z(4, 16, 512), k_pe=z(4, 16, 64), page_table=z(2, 2, d=i32), lengths=z(2, d=i32), cu_q=z(3, d=i32))  # fmt: skip

    def call():
        cache = L.LatentCache(t["latent"], t["k_pe"])
        args = [t[n] for n in ("q", "kv_a", "norm_weight", "kv_b_weight", "cos", "sin", "position_ids", "slots")]
        return MLA(2, 192, 128).decode(*args, cache, *(t[n] for n in ("page_table", "lengths", "cu_q")))

    assert call().shape == (2, 2, 128) and t["latent"]._version > 0  # (the count says who wrote)
    t[name].requires_grad_()
    before = t["latent"]._version, t["k_pe"]._version
    with pytest.raises(RuntimeError, match="has no backward"):
        call()
    assert (t["latent"]._version, t["k_pe"]._version) == before
    with torch.no_grad():
        call()


def test_a_cache_made_in_inference_mode_can_be_written_outside_it():
    with torch.inference_mode():
        cache = L.LatentCache.empty(4, 16, device="meta")
    with torch.no_grad():
        L.latent_cache_append(*(t.to("meta") for t in (_zeros(3, 576), _zeros(512), _zeros(8, 64), _zeros(8, 64), _zeros(3, d=torch.int64), _zeros(3, d=torch.int64))), cache)


def test_a_cache_of_another_type_is_refused():
    with pytest.raises(AssertionError, match="bfloat16 or float8_e4m3fn"):
        L.LatentCache.empty(2, dtype=torch.float16, device="cpu")
    c = L.LatentCache.empty(2, 32, L.FP8, "cpu")
    assert c.latent.shape == (2, 32, 512) and c.scale.shape == (2, 32) and L.LatentCache.empty(2, device="cpu").scale is None


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("shape", [(512,), (3, 576), (3, 2, 192)])
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_rows_that_begin_off_the_alignment_are_copied(offset, shape, dtype):
    """Also where they lie one behind the other already, as slices of a flat buffer do."""
    x = torch.arange(offset + math.prod(shape)).to(dtype)[offset:].view(shape)
    got = L._aligned_rows(x)
    assert got.data_ptr() % 16 == 0 and got.is_contiguous() and torch.equal(got, x)
    assert (got.data_ptr() == x.data_ptr()) == (x.data_ptr() % 16 == 0)


def test_decode_is_for_the_layers_head_dims():
    z = _zeros
    rest = (z(1, 576), z(512), z(512, 512), z(8, 64), z(8, 64), z(1), z(1), None, z(1), z(1), z(2))
    with pytest.raises(AssertionError, match="dq=192"):
        MLA(2, 128, 128).decode(z(1, 2, 128), *rest)
    with pytest.raises(AssertionError, match="q must be"):
        MLA(4, 192, 128).decode(z(1, 2, 192), *rest)


def test_direct_loads_are_the_only_users_of_m0(tmp_path):
    """csrc/attn_tiles.h sets M0 inside inline assembly, which the compiler cannot be told about: it must not use the register itself."""
    from pithtrain_amd import build as B

    for src in ("latent_attn.hip", "latent_attn_wide.hip", "latent_absorb.hip"):
        out = tmp_path / (src + ".s")
        cmd = [B._hipcc(), *B.HIPCC_FLAGS, *B.SOURCE_FLAGS.get(src, []), "-I", B.INCLUDE_DIR, "-I", B.SRC_DIR, "--cuda-device-only", "-S", os.path.join(B.SRC_DIR, src), "-o", str(out)]
        subprocess.run(cmd, check=True, capture_output=True)
        text = re.sub(r";;#ASMSTART.*?;;#ASMEND", "", out.read_text(), flags=re.S)
        assert not [line for line in text.splitlines() if re.search(r"\bm0\b", line.split(";")[0])]
