"""The key-value cache's operators and the planning of a step on a machine without a GPU: the oracle's pins, the C interface of include/pith_kv.h, what the
Python entry points refuse, and their shape propagation."""

import ctypes
import math
import os
import re
import subprocess
import sys

import pytest
import torch

from oracle import kv_oracle as O
from oracle import prologue_oracle as P
from pithtrain_amd import _C
from pithtrain_amd.operators import paging
from pithtrain_amd.operators.gqa import kv_cache as K

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "pith_kv.h")
BF = torch.bfloat16


# ---------------------------------------------------------------------------------------------
# The oracle


def test_attention_of_the_last_rows_is_the_causal_layer():
    """All rows as new ones: scaled_dot_product_attention with grouped heads; and the rows in two pieces, joined by their lse."""
    g = torch.Generator().manual_seed(1)
    mk = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    n, h, hkv, d = 19, 6, 2, 64
    q, k, v = mk(n, h, d), mk(hkv, n, d), mk(hkv, n, d)
    o, lse, mass, spread = O.attention(q, k, v, O.sees(n, n), 0.2)
    want = torch.nn.functional.scaled_dot_product_attention(q.transpose(0, 1), k.repeat_interleave(3, 0), v.repeat_interleave(3, 0), is_causal=True, scale=0.2)
    assert (o - want.transpose(0, 1)).abs().max() < 1e-12
    s = torch.einsum("ihd,hjd->hij", q, k.repeat_interleave(3, 0)) * 0.2
    want = torch.logsumexp(s.masked_fill(torch.ones(n, n).triu(1).bool(), -math.inf), -1) / math.log(2)
    assert (lse - want).abs().max() < 1e-12 and (mass >= o.abs() - 1e-12).all() and (spread > 0).all()
    a, la, _, _ = O.attention(q[-1:], k[:, :9], v[:, :9], O.sees(1, 9), 0.2)
    b, lb, _, _ = O.attention(q[-1:], k[:, 9:], v[:, 9:], O.sees(1, n - 9), 0.2)
    wa, wb = (torch.exp2(x - lse[:, -1:]).T[..., None] for x in (la, lb))
    assert (wa * a + wb * b - o[-1:]).abs().max() < 1e-12


def test_norm_and_rotation_are_the_prologues():
    g = torch.Generator().manual_seed(2)
    x, w = torch.randn(7, 3, 64, generator=g, dtype=torch.float64), torch.rand(64, generator=g, dtype=torch.float64)
    cos, sin = P.cos_sin_table(torch.arange(20).unsqueeze(0), 64)
    cos, sin = cos[0].to(BF), sin[0].to(BF)
    pos = torch.tensor([0, 3, 19, 3, 2, 1, 0])
    got, mass = O.norm_rope(x, w, cos, sin, pos, 1e-6)
    assert torch.allclose(got, P.norm_rope_fwd(x.unsqueeze(0), w, cos[pos].unsqueeze(0), sin[pos].unsqueeze(0), 1e-6)[0])
    assert (mass >= got.abs() - 1e-12).all()


def test_no_row_of_a_page_scores_above_its_bound():
    g = torch.Generator().manual_seed(3)
    keys, q = torch.randn(9, 2, 16, 64, generator=g), torch.randn(6, 64, generator=g)
    s = O.scores(q, torch.stack([O.bounds(x) for x in keys]))
    dots = torch.einsum("ghd,pgrd->pghr", q.double().view(2, 3, 64), keys.double()).amax((2, 3)).T
    assert (s.double() >= dots - 1e-5).all()
    kept = O.select(q, torch.stack([O.bounds(x) for x in keys]), 9 * 16 - 3, 16, 4)
    for row, best in zip(s[:, :8], kept):
        assert best == sorted(row.topk(3).indices.tolist()) + [8]
    assert O.select(q, torch.stack([O.bounds(x) for x in keys]), 50, 16, 4) == [[0, 1, 2, 3]] * 2


def test_a_plan_by_hand():
    got = O.plan([1, -1, 3, 0, 40], [16, 20, 15, 5, 0], [[7, -1, -1], [3, 4, -1], [5, -1, -1], [6, -1, -1], [-1, -1, -1]], [9, 8, 0, 0, 0, 0], 1, 16, 46)
    # pages 3 and 4 come back: the pool is 9 3 4; request 0 takes 4, request 2 takes 3, the last one would need three
    assert got["free"] == [9, 3, 4, 0, 0, 0] and got["free_count"] == [1]
    assert got["page_table"] == [[7, 4, -1], [3, 4, -1], [5, 3, -1], [6, -1, -1], [-1, -1, -1]]
    assert got["granted"] == [1, 0, 3, 0, 0] and got["lengths"] == [17, 0, 18, 5, 0] and got["cu_q"] == [0, 1, 1, 4, 4, 44]
    assert got["position_ids"] == [16, 15, 16, 17] + list(range(40)) + [0, 0] and got["slots"] == [64, 95, 48, 49] + [-1] * 42


# ---------------------------------------------------------------------------------------------
# The C interface


def test_library_exports_every_declared_symbol():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(pith_[a-z0-9_]+)\s*\(", text)))
    assert sorted(_C.KV_SYMBOLS) == declared
    for name in declared:
        assert hasattr(_C.lib(), name), f"{name} is declared in pith_kv.h but not exported"


STRUCTS = {
    "pith_kv_cache": _C.KVCacheArgs, "pith_plan_step_args": _C.PlanStepArgs, "pith_kv_append_args": _C.KVAppendArgs, "pith_kv_attn_args": _C.KVAttnArgs,
    "pith_kv_bounds_args": _C.KVBoundsArgs, "pith_kv_select_args": _C.KVSelectArgs,
}  # fmt: skip
# struct sizes of a version of this part of the interface: a change here needs a new version
STRUCT_SIZES = {
    100: {"pith_kv_cache": 104, "pith_plan_step_args": 152, "pith_kv_append_args": 280, "pith_kv_attn_args": 272, "pith_kv_bounds_args": 176,
          "pith_kv_select_args": 176},
}  # fmt: skip


def test_struct_layouts_match_the_header(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "pith_kv.h"', 'int main(void){printf("version %d\\n", PITH_KV_VERSION);']
    for cname, st in STRUCTS.items():
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in st._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.strip().splitlines())
    assert int(got["version"]) == _C.PITH_KV_VERSION == _C.lib().pith_kv_version()
    for cname, st in STRUCTS.items():
        assert int(got[cname]) == ctypes.sizeof(st) == STRUCT_SIZES[_C.PITH_KV_VERSION][cname], (cname, got[cname])
        for f, _ in st._fields_:
            assert int(got[f"{cname}.{f}"]) == getattr(st, f).offset, f"{cname}.{f}"


@pytest.mark.parametrize("version", [100, 99])
def test_the_native_path_is_loaded_with_its_own_version_only(tmp_path, version):
    src, shim = tmp_path / "shim.c", tmp_path / "shim.so"
    src.write_text(f"int pith_kv_version(void) {{ return {version}; }}\n")
    subprocess.run(["gcc", "-shared", "-fPIC", str(src), "-o", str(shim)], check=True)
    code = f"import ctypes; ctypes.CDLL({str(shim)!r}, ctypes.RTLD_GLOBAL); from pithtrain_amd import _ext"
    env = {**os.environ, "PYTHONPATH": os.path.join(ROOT, "pith-train_amd")}
    run = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True)
    if version == _C.PITH_KV_VERSION:
        assert run.returncode == 0, run.stderr
    else:
        assert run.returncode == 1 and "build both again" in run.stderr, run.stderr


def _cache(**kw):
    base = dict(k=256, v=256, pages=8, page_size=64, heads=2, dim=128, k_ps=2 * 64 * 128, v_ps=2 * 64 * 128, dtype=_C.PITH_BF16)
    return _C.KVCacheArgs(**{**base, **kw})


def _plan(**kw):
    base = dict(counts=256, lengths=256, page_table=256, free_pages=256, free_count=256, cu_q=256, position_ids=256, slots=256, granted=256, lengths_out=256,
                free_count_out=256, workspace=256, workspace_bytes=1 << 40, B=2, T=4, table_rs=4, table_width=4, pool_size=8, page_size=64)  # fmt: skip
    return _C.PlanStepArgs(**{**base, **kw})


def _append(**kw):
    base = dict(q=256, k=256, v=256, q_weight=256, k_weight=256, cos=256, sin=256, position_ids=256, slots=256, q_out=256, T=4, P=16, H=4, q_ts=512, q_hs=128, k_ts=256,
                k_hs=128, v_ts=256, v_hs=128, q_out_ts=512, q_out_hs=128, eps=1e-6, weight_dtype=_C.PITH_BF16, cache=_cache())  # fmt: skip
    return _C.KVAppendArgs(**{**base, **kw})


def _attn(**kw):
    base = dict(q=256, cache=_cache(), page_table=256, lengths=256, cu_q=256, tree_mask=None, o=256, lse=256, workspace=256, workspace_bytes=1 << 40, T=4, B=2, H=4,
                table_rs=4, table_hs=0, table_width=4, q_ts=512, q_hs=128, o_ts=512, o_hs=128, lse_hs=4, scale=0.07, head_tables=0)  # fmt: skip
    return _C.KVAttnArgs(**{**base, **kw})


def _bounds(**kw):
    base = dict(cache=_cache(), bounds=256, page_table=256, lengths=256, cu_q=256, T=4, B=2, table_rs=4, table_width=4, bounds_ps=512)
    return _C.KVBoundsArgs(**{**base, **kw})


def _select(**kw):
    base = dict(q=256, bounds=256, page_table=256, lengths=256, cu_q=256, table_out=256, lengths_out=256, workspace=256, workspace_bytes=1 << 40, T=4, B=2, H=4, heads=2,
                dim=128, pages=8, page_size=64, keep=2, q_ts=512, q_hs=128, table_rs=4, table_width=4, bounds_ps=512)  # fmt: skip
    return _C.KVSelectArgs(**{**base, **kw})


NULL, SHAPE, DTYPE, UNSUPPORTED, ALIGN = (_C.PITH_ERR_NULL_POINTER, _C.PITH_ERR_BAD_SHAPE, _C.PITH_ERR_BAD_DTYPE, _C.PITH_ERR_UNSUPPORTED, _C.PITH_ERR_MISALIGNED)
FP8 = dict(dtype=_C.PITH_FP8_E4M3, k_scale=256, v_scale=256, k_scale_ps=128, v_scale_ps=128)
BAD_CACHES = [
    (dict(dtype=1), DTYPE), (dict(k=None), NULL), (dict(v=None), NULL), (dict(dtype=_C.PITH_FP8_E4M3), NULL), ({**FP8, "v_scale": None}, NULL), (dict(page_size=8), SHAPE),
    (dict(page_size=48), SHAPE), (dict(page_size=1 << 17), SHAPE), (dict(pages=0), SHAPE), (dict(pages=1 << 26), SHAPE), (dict(heads=0), SHAPE), (dict(heads=1025), SHAPE),
    (dict(dim=96), UNSUPPORTED), (dict(dim=192), UNSUPPORTED), (dict(k_ps=2 * 64 * 128 - 8), SHAPE), (dict(v_ps=64 * 128), SHAPE), (dict(k=264), ALIGN), (dict(v=248), ALIGN),
    (dict(v_ps=2 * 64 * 128 + 4), ALIGN), ({**FP8, "k_scale_ps": 127}, SHAPE), ({**FP8, "v_scale": 258}, ALIGN), ({**FP8, "k_ps": 2 * 64 * 128 + 8}, ALIGN),
]  # fmt: skip
TABLES = [
    (dict(T=-1), SHAPE), (dict(B=-1), SHAPE), (dict(T=1 << 21), SHAPE), (dict(cu_q=None), SHAPE), (dict(table_width=0), SHAPE), (dict(table_width=-1), SHAPE), (dict(table_rs=3), SHAPE),
    (dict(table_width=1 << 26, table_rs=1 << 26), UNSUPPORTED), (dict(page_table=None), NULL), (dict(lengths=None), NULL), (dict(cu_q=258), ALIGN), (dict(lengths=258), ALIGN),
]  # fmt: skip
CALLS = {
    "pith_plan_step": (_plan, [
        (dict(counts=None), NULL), (dict(lengths=None), NULL), (dict(page_table=None), NULL), (dict(free_pages=None), NULL), (dict(free_count=None), NULL), (dict(cu_q=None), NULL),
        (dict(slots=None), NULL), (dict(granted=None), NULL), (dict(free_count_out=None), NULL), (dict(B=-1), SHAPE), (dict(B=1 << 21), SHAPE), (dict(T=-1), SHAPE), (dict(T=1 << 31), SHAPE),
        (dict(pool_size=-1), SHAPE), (dict(pool_size=1 << 31), SHAPE), (dict(page_size=24), SHAPE), (dict(page_size=8), SHAPE), (dict(table_rs=3), SHAPE),
        (dict(table_width=1 << 26, table_rs=1 << 26), UNSUPPORTED), (dict(T=1 << 20, workspace_bytes=16), SHAPE), (dict(T=1 << 20, workspace=None), NULL), (dict(slots=260), ALIGN),
        (dict(counts=258), ALIGN), (dict(workspace=264), ALIGN)]),
    "pith_kv_append": (_append, [
        (dict(q=None), NULL), (dict(v=None), NULL), (dict(q_out=None), NULL), (dict(slots=None), NULL), (dict(q_weight=None), NULL), (dict(T=-1), SHAPE), (dict(P=0), SHAPE), (dict(H=0), SHAPE),
        (dict(H=1025), SHAPE), (dict(T=0x7fffffff), UNSUPPORTED), (dict(q_hs=1 << 29), UNSUPPORTED), (dict(q_ts=120), SHAPE), (dict(k_hs=64), SHAPE), (dict(v_ts=64), SHAPE), (dict(q_out_hs=120), SHAPE), (dict(q_ts=516), ALIGN),
        (dict(v_hs=132), ALIGN), (dict(k=264), ALIGN), (dict(cos=264), ALIGN), (dict(k_weight=264), ALIGN), (dict(slots=260), ALIGN), (dict(weight_dtype=2), DTYPE)]),
    "pith_kv_attn": (_attn, TABLES + [
        (dict(q=None), NULL), (dict(workspace=None), NULL), (dict(lse=None), NULL), (dict(H=0), SHAPE), (dict(H=3), SHAPE), (dict(H=1026), SHAPE), (dict(q_hs=120), SHAPE), (dict(o_ts=120), SHAPE),
        (dict(lse_hs=3), SHAPE), (dict(workspace_bytes=64), SHAPE), (dict(q=264), ALIGN), (dict(q_hs=132), ALIGN), (dict(o_ts=516), ALIGN), (dict(workspace=384), ALIGN),
        (dict(tree_mask=260), ALIGN), (dict(head_tables=1, table_hs=4, table_rs=8, T=2, cu_q=None, tree_mask=256), UNSUPPORTED), (dict(head_tables=1, table_hs=4, table_rs=8), UNSUPPORTED),
        (dict(head_tables=1, table_hs=3, table_rs=8, T=2, cu_q=None), SHAPE)]),
    "pith_kv_bounds": (_bounds, TABLES + [(dict(bounds=None), NULL), (dict(bounds_ps=504), SHAPE), (dict(bounds_ps=516), ALIGN), (dict(bounds=264), ALIGN)]),
    "pith_kv_select": (_select, TABLES + [
        (dict(q=None), NULL), (dict(bounds=None), NULL), (dict(table_out=None), NULL), (dict(workspace=None), NULL), (dict(H=3), SHAPE), (dict(heads=0), SHAPE), (dict(dim=32), UNSUPPORTED),
        (dict(keep=0), SHAPE), (dict(keep=1 << 21), SHAPE), (dict(pages=0), SHAPE), (dict(page_size=20), SHAPE), (dict(bounds_ps=504), SHAPE), (dict(q_ts=120), SHAPE), (dict(q=264), ALIGN),
        (dict(q_hs=132), ALIGN), (dict(bounds_ps=516), ALIGN), (dict(workspace=128), ALIGN), (dict(workspace_bytes=64), SHAPE),
        (dict(T=1 << 20, heads=128, H=128, bounds_ps=128 * 256, table_width=64, table_rs=64), UNSUPPORTED), (dict(table_width=16385, table_rs=16385), UNSUPPORTED)]),
}  # fmt: skip


@pytest.mark.parametrize("name", CALLS)
def test_bad_arguments_are_rejected_before_anything_is_launched(name):
    """There is no device here, so a launch would show as PITH_ERR_LAUNCH."""
    make, bad = CALLS[name]
    fn = getattr(_C.lib(), name)
    assert fn(None, None) == NULL
    with_cache = [] if make in (_plan, _select) else [(dict(cache=_cache(**kw)), code) for kw, code in BAD_CACHES]
    for kw, code in bad + with_cache:
        assert fn(ctypes.byref(make(**kw)), None) == code, (kw, _C.lib().pith_last_error())
        assert _C.lib().pith_last_error().startswith(name.encode())


@pytest.mark.parametrize("name", [n for n in CALLS if n != "pith_plan_step"])
def test_empty_calls_launch_nothing(name):
    make, _ = CALLS[name]
    for kw in [dict(T=0)] + ([] if make is _append else [dict(B=0)]):
        assert getattr(_C.lib(), name)(ctypes.byref(make(**kw)), None) == _C.PITH_OK


@pytest.mark.parametrize("fp8", [False, True])
def test_the_stride_of_a_single_page_is_not_used(fp8):
    odd = dict(pages=1, k_ps=515, v_ps=3, **(dict(FP8, k_scale_ps=1, v_scale_ps=0) if fp8 else {}))
    for name, (make, _) in CALLS.items():
        if make not in (_plan, _select):
            assert getattr(_C.lib(), name)(ctypes.byref(make(cache=_cache(**odd), T=0)), None) == _C.PITH_OK, _C.lib().pith_last_error()


def test_workspaces():
    lib = _C.lib()
    plan = lambda **kw: lib.pith_plan_step_workspace_bytes(ctypes.byref(_plan(**kw)))  # noqa: E731
    assert plan() == 0 and plan(T=1 << 20) > 0 and plan(B=5000) >= 16 * 5000 and plan(page_size=8) == 0
    attn = lambda **kw: lib.pith_kv_attn_workspace_bytes(ctypes.byref(_attn(**kw)))  # noqa: E731
    assert attn(T=0) == attn(B=0) == attn(H=3) == 0 and attn() > 0
    assert attn(table_width=4096, table_rs=4096) == attn(table_width=64, table_rs=64)  # whatever the lengths
    select = lambda **kw: lib.pith_kv_select_workspace_bytes(ctypes.byref(_select(**kw)))  # noqa: E731
    assert select() == 4 * 2 * 128 * 8 and select(T=0) == select(keep=0) == 0 and select(table_width=129) == 2 * select()


def test_the_workspace_of_a_selection_is_bounded():
    """64 MB, or what one token needs, however many tokens there are."""
    select = lambda **kw: _C.lib().pith_kv_select_workspace_bytes(ctypes.byref(_select(**kw)))  # noqa: E731
    prompt = dict(heads=4, H=32, table_width=2048, table_rs=2048, bounds_ps=1024)
    assert select(T=1, **prompt) == 4 * 2048 * 8 and select(T=1024, **prompt) == 64 << 20
    assert [select(T=t, **prompt) for t in (1025, 8192, 100000)] == [64 << 20] * 3
    assert select(T=9, heads=1024, H=1024, table_width=16384, table_rs=16384, bounds_ps=1 << 18) == 1024 * 16384 * 8


def test_rows_of_a_row_block_go_by_the_rows_of_a_sequence_and_the_work_list():
    rows = lambda **kw: _C.lib().pith_kv_attn_rows(ctypes.byref(_attn(**kw)))  # noqa: E731
    assert rows(T=0) == rows(B=0) == rows(H=3) == 0  # nothing to launch, or what pith_kv_attn rejects
    wide = dict(table_width=65536, table_rs=65536)
    assert rows(T=16, lse_hs=16, **wide) == 16  # sixteen rows a sequence and key-value head
    assert rows(T=17, lse_hs=17, **wide) == 32 and rows(T=32, lse_hs=32, **wide) == 32
    assert rows(T=33, lse_hs=33, **wide) == rows(T=72, lse_hs=72, **wide) == 64  # where that makes the row blocks fewer by a quarter
    assert rows(T=33, lse_hs=33, cache=_cache(**FP8), **wide) == 32 and rows(T=33, lse_hs=33, cache=_cache(dim=64, k_ps=64 * 128, v_ps=64 * 128), **wide) == 32
    assert rows(T=256, lse_hs=256, **wide) == 64 and rows(T=256, lse_hs=256, table_width=512, table_rs=512) == 32  # and there is so much to read
    assert rows(T=64, lse_hs=64, table_width=16, table_rs=16) == 16  # and a work list of some length


# ---------------------------------------------------------------------------------------------
# The Python entry points


def _zeros(*s, d=BF, dev="cpu"):
    return torch.zeros(*s, dtype=d, device=dev)


def _calls(dev):
    z = lambda *s, d=BF: _zeros(*s, d=d, dev=dev)  # noqa: E731
    i32, i64 = torch.int32, torch.int64
    cache = K.KVCache(z(4, 2, 16, 64), z(4, 2, 16, 64))
    pool = paging.PagePool(z(8, d=i32), z(1, d=i32))
    new = lambda: (z(3, 4, 64), z(3, 2, 64), z(3, 2, 64), z(64), z(64), z(8, 64), z(8, 64), z(3, d=i64), z(3, d=i64))  # noqa: E731
    where = lambda: (z(2, 2, d=i32), z(2, d=i32), z(3, d=i32))  # noqa: E731
    return {
        "plan": lambda: paging.plan_step(z(2, d=i32), z(2, d=i32), z(2, 4, d=i32), pool, 16, 5),
        "append": lambda: K.kv_cache_append(*new(), cache),
        "attention": lambda: K.kv_attention(z(3, 4, 64), cache, *where(), 0.1),
        "attention_of_heads": lambda: K.kv_attention(z(3, 4, 64), cache, z(3, 2, 5, d=i32), z(3, 2, d=i32), None, 0.1),
        "bounds": lambda: K.kv_page_bounds(cache, z(4, 2, 2, 64), *where(), 3),
        "select": lambda: K.kv_select_pages(z(3, 4, 64), z(4, 2, 2, 64), *where(), 16, 3),
        "decode": lambda: K.kv_decode(*new(), cache, *where(), 0.1, bounds=z(4, 2, 2, 64), keep=2),
    }


@pytest.mark.parametrize("name", _calls("cpu"))
def test_cpu_tensors_are_refused(name):
    with pytest.raises(RuntimeError, match="need tensors on a GPU"):
        _calls("cpu")[name]()


def test_shapes_propagate_without_a_device():
    calls = _calls("meta")
    plan = calls["plan"]()
    assert [tuple(t.shape) for t in plan] == [(3,), (2,), (5,), (5,), (2,), (1,)] and [t.dtype for t in plan] == [torch.int32] * 2 + [torch.int64] * 2 + [torch.int32] * 2
    assert calls["append"]().shape == (3, 4, 64) and calls["bounds"]() is None
    for name in ("attention", "attention_of_heads"):
        o, lse = calls[name]()
        assert (o.shape, o.dtype, lse.shape, lse.dtype) == ((3, 4, 64), BF, (4, 3), torch.float32)
    selected = calls["select"]()
    assert (selected.page_table.shape, selected.lengths.shape, selected.page_table.dtype) == ((3, 2, 3), (3, 2), torch.int32)
    assert calls["decode"]().shape == (3, 4, 64)


def test_arguments_that_require_a_gradient_are_refused():
    z, i32, i64 = _zeros, torch.int32, torch.int64
    cache = K.KVCache(z(4, 2, 16, 64), z(4, 2, 16, 64))
    where = (z(2, 2, d=i32), z(2, d=i32), z(3, d=i32))
    new = [z(3, 4, 64), z(3, 2, 64), z(3, 2, 64), z(64), z(64), z(8, 64), z(8, 64)]
    for i in range(5):
        one = [t.clone().requires_grad_() if i == j else t for j, t in enumerate(new)]
        with pytest.raises(RuntimeError, match="kv_append has no backward"):
            K.kv_cache_append(*one, z(3, d=i64), z(3, d=i64), cache)
        with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError, match="kv_append has no forward-mode derivative"):
            one[i] = torch.autograd.forward_ad.make_dual(new[i], new[i])
            K.kv_cache_append(*one, z(3, d=i64), z(3, d=i64), cache)
    q = z(3, 4, 64).requires_grad_()
    with pytest.raises(RuntimeError, match="kv_attention has no backward"):
        K.kv_attention(q, cache, *where, 0.1)
    with pytest.raises(RuntimeError, match="kv_attention has no backward"):
        K.kv_attention(q.detach(), K.KVCache(cache.k.clone().requires_grad_(), cache.v), *where, 0.1)
    with pytest.raises(RuntimeError, match="kv_select has no backward"):
        K.kv_select_pages(q, z(4, 2, 2, 64), *where, 16, 3)
    with pytest.raises(RuntimeError, match="kv_bounds has no backward"):
        K.kv_page_bounds(cache, z(4, 2, 2, 64).requires_grad_(), *where, 3)
    for given in (q, z(3, 4, 64)):
        with pytest.raises(RuntimeError, match="has no backward"):
            K.kv_attention_into(given, cache, *where, 0.1, None, z(3, 4, 64) if given is q else z(3, 4, 64).requires_grad_(), z(4, 3, d=torch.float32))
    with torch.no_grad(), pytest.raises(RuntimeError, match="need tensors on a GPU"):
        K.kv_attention(q, cache, *where, 0.1)
