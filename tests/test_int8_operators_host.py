"""Host-side checks of the norm, the int8 rows and the int8 products that need no GPU: struct layouts, sizes and arguments that the launchers and the C ABI
refuse before anything reaches a device."""
import ctypes
import os
import subprocess

import pytest

from int8_cuts import CASES
from memfabric_hybrid_amd import capi

INC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
INVALID = capi.Z_INVALID_PARAM


@pytest.fixture(scope="module")
def lib():
    return capi.load()


def test_struct_layouts(tmp_path):
    src, exe = tmp_path / "t.c", tmp_path / "t"
    src.write_text('#include "zbal.h"\n#include "zbal_hip_kernels.h"\n#include <stdio.h>\n'
                   'int main(void){printf("%zu %zu %zu %zu %zu %zu", sizeof(zbalhip_rms_norm_t), __builtin_offsetof(zbalhip_rms_norm_t, eps),'
                   'sizeof(zbalhip_quantize_rows_t), __builtin_offsetof(zbalhip_quantize_rows_t, width),'
                   'sizeof(zbalhip_expert_linear_int8_t), __builtin_offsetof(zbalhip_expert_linear_int8_t, rows));return 0;}\n')
    subprocess.check_call(["gcc", "-I", INC, str(src), "-o", str(exe)])
    got = [int(v) for v in subprocess.check_output([str(exe)]).split()]
    assert got == [ctypes.sizeof(capi.RmsNorm), capi.RmsNorm.eps.offset, ctypes.sizeof(capi.QuantizeRows), capi.QuantizeRows.width.offset,
                   ctypes.sizeof(capi.ExpertLinearInt8), capi.ExpertLinearInt8.rows.offset]


def norm(**kw):
    d = dict(x=4096, residual=None, weight=4096, dtype=capi.DT_BF16, weight_is_f32=0, tokens=4, hidden=64, eps=1e-6)
    d.update(kw)
    return capi.RmsNorm(**d)


NORM_SIZES = [dict(tokens=-1), dict(tokens=(1 << 24) + 1), dict(hidden=0), dict(hidden=65537), dict(dtype=capi.DT_INT8), dict(eps=0.0), dict(eps=-1.0),
              dict(eps=float("nan")), dict(eps=float("inf"))]


@pytest.mark.parametrize("kw", NORM_SIZES + [dict(x=None)])
def test_norm_refusals(lib, kw):
    d = ctypes.byref(norm(**kw))
    assert lib.zbalhip_rms_norm(d, 4096, None, None, None, None) == INVALID
    assert lib.zbalhip_rms_norm_backward(d, 4096, None, 4096, None, 0, None, 0, None) == INVALID
    if kw in NORM_SIZES:
        assert lib.zbalhip_rms_norm_backward_workspace(d) == -1


def test_norm_null_pointers(lib):
    d = ctypes.byref(norm())
    assert lib.zbalhip_rms_norm(None, 4096, None, None, None, None) == INVALID
    assert lib.zbalhip_rms_norm(d, None, None, None, 4096, None) == INVALID                    # no output
    assert lib.zbalhip_rms_norm(d, None, None, 4096, None, None) == INVALID                    # int8 without scales
    assert lib.zbalhip_rms_norm_backward_workspace(d) == 0                                     # so few rows that one workgroup has them all
    many = ctypes.byref(norm(tokens=4096))
    need = lib.zbalhip_rms_norm_backward_workspace(many)
    assert need > 0
    for of, grad, gx, gw, ws, size in ((d, None, 4096, None, None, 0), (d, 4096, None, None, None, 0), (many, 4096, 4096, 4096, None, need), (many, 4096, 4096, 4096, 4096, need - 1)):
        assert lib.zbalhip_rms_norm_backward(of, grad, None, gx, gw, 0, ws, size, None) == INVALID
    none = ctypes.byref(norm(tokens=0, x=None))
    assert lib.zbalhip_rms_norm(none, None, None, None, None, None) == 0
    assert lib.zbalhip_rms_norm_backward(none, None, None, None, None, 0, None, 0, None) == 0


def test_norm_workspace_is_bounded(lib):
    for tokens in (0, 1, 61, 16384, 1 << 24):
        for hidden in (1, 64, 2048, 7168, 65536):
            b = lib.zbal_moe_rms_norm_workspace_size(tokens, hidden)
            assert 0 <= b <= 1 << 30 and (tokens > 0 or b == 0)
    assert lib.zbal_moe_rms_norm_workspace_size(4, 65537) == lib.zbal_moe_rms_norm_workspace_size(-1, 64) == -1


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(rows=(1 << 24) + 1), dict(width=0), dict(width=65537), dict(dtype=capi.DT_INT8), dict(activation=-1), dict(activation=6),
                                dict(activation=5, width=63), dict(counts=4096, experts=0), dict(counts=4096, experts=1025), dict(x=None), dict(q=None), dict(scales=None)])
def test_quantize_refusals(lib, kw):
    a = dict(x=4096, q=4096, scales=4096)
    a.update({k: kw[k] for k in kw if k in a})
    d = dict(counts=None, counts_are_i64=0, dtype=capi.DT_BF16, activation=0, rows=4, width=64, experts=0)
    d.update({k: kw[k] for k in kw if k in d})
    assert lib.zbalhip_quantize_rows(ctypes.byref(capi.QuantizeRows(**d)), a["x"], a["q"], a["scales"], None) == INVALID
    assert lib.zbalhip_quantize_rows(None, 4096, 4096, 4096, None) == INVALID


def linear(**kw):
    d = dict(weight=4096, weight_scales=4096, weight_scales_are_f32=1, counts_are_i64=0, counts=4096, activation=0, y_dtype=capi.DT_BF16, rows=16, k=64, n=64, experts=2)
    d.update(kw)
    return capi.ExpertLinearInt8(**d)


SIZES = [dict(rows=-1), dict(rows=(1 << 24) + 1), dict(k=0), dict(n=0), dict(k=65537), dict(n=65537), dict(experts=0), dict(experts=1025), dict(y_dtype=capi.DT_INT8),
         dict(activation=-1), dict(activation=6), dict(activation=5, n=63)]


@pytest.mark.parametrize("kw", SIZES + [dict(weight=None), dict(weight_scales=None), dict(counts=None)])
def test_linear_refusals(lib, kw):
    d = ctypes.byref(linear(**kw))
    assert lib.zbalhip_expert_linear_int8(d, 4096, 4096, None, 0, None, 4096, None, 0, None) == INVALID
    if kw in SIZES:
        assert lib.zbalhip_expert_linear_int8_workspace(d) == -1


def test_linear_null_pointers(lib):
    d = ctypes.byref(linear())
    assert lib.zbalhip_expert_linear_int8(None, 4096, 4096, None, 0, None, 4096, None, 0, None) == INVALID
    for x, xs, y in ((None, 4096, 4096), (4096, None, 4096), (4096, 4096, None)):
        assert lib.zbalhip_expert_linear_int8(d, x, xs, None, 0, None, y, None, 0, None) == INVALID
    assert lib.zbalhip_expert_linear_int8(ctypes.byref(linear(rows=0)), None, None, None, 0, None, None, None, 0, None) == 0


def test_linear_workspace_sizes(lib):
    for rows, k, n, e in ((0, 64, 64, 1), (1, 7168, 256, 1), (4096, 7168, 256, 1), (500, 8192, 128, 1), (32768, 2048, 4096, 32), (1 << 24, 65536, 65536, 1), (5, 1, 1, 1), (7, 15, 3, 2)):
        b = lib.zbal_moe_expert_linear_int8_workspace_size(rows, k, n, e, 0)
        assert 0 <= b < 1 << 32
        assert b == 0 or e == 1
    assert lib.zbal_moe_expert_linear_int8_workspace_size(16, 64, 63, 1, 5) == -1
    # unaligned rows are copied where that is sooner, never past 512 MiB
    assert lib.zbal_moe_expert_linear_int8_workspace_size(4093, 4099, 4093, 1, 0) == 2 * 4093 * 4112
    assert lib.zbal_moe_expert_linear_int8_workspace_size(16, 4001, 1531, 32, 0) == 0
    assert lib.zbal_moe_expert_linear_int8_workspace_size(1 << 20, 4099, 4093, 1, 0) == 0


def plan(lib, rows, experts, k, n, act):
    parts, copied = ctypes.c_int32(-1), ctypes.c_int32(-1)
    name = lib.zbalhip_expert_linear_int8_plan(ctypes.byref(linear(rows=rows, experts=experts, k=k, n=n, activation=capi.ACTIVATIONS[act])), ctypes.byref(parts), ctypes.byref(copied))
    return name and (name.decode(), parts.value, copied.value)


@pytest.mark.parametrize("cut,rows,experts,k,n,act", CASES)
def test_linear_plans(lib, cut, rows, experts, k, n, act):
    """the sizes that the tests on the GPU have for each kind of tiles are cut into them"""
    assert plan(lib, rows, experts, k, n, act) == cut
    wide = (k + 15) // 16 * 16
    cols = -(-n // 8) * 8 if act == "swiglu" and n % 8 else -(-n // 4) * 4            # either half of a swiglu's sums starts at a multiple of four
    size = lib.zbal_moe_expert_linear_int8_workspace_size(rows, k, n, experts, capi.ACTIVATIONS[act])
    assert size == (cut[2] and (rows + experts * n) * wide) + (cut[1] > 1 and cut[1] * rows * cols * 4)


def test_linear_plans_reach_every_kind(lib):
    kinds = {name for (name, _, _), *_ in CASES}
    assert len(kinds) == 14
    for name in kinds - {"short"}:
        of = [(c, size) for c, *size in CASES if c[0] == name]
        assert {size[1] > 1 for _, size in of} == {True, False} and {size[4] for _, size in of} == {"none", "swiglu"}
        aligned = not name.endswith("any")
        assert {c[2] for c, _ in of} == ({0, 1} if aligned else {0})
        parts = {c[1] for c, _ in of}
        assert 1 in parts and (parts == {1}) == (name in ("256x256", "rows") or name.endswith("flat"))
    assert plan(lib, 0, 2, 64, 64, "none") is None and plan(lib, 4, 2, 65537, 64, "none") is None
    assert lib.zbalhip_expert_linear_int8_plan(None, None, None) is None
    assert lib.zbalhip_expert_linear_int8_plan(ctypes.byref(linear()), None, None)


def test_outer_calls_check_their_arguments_first(lib):
    t = capi.TensorInfo()
    ok = ctypes.byref(t)
    assert lib.zbal_moe_rms_norm(None, None, None, 1e-6, ok, None, None, None, None, None, 0) == INVALID
    assert "x is null" in capi.last_error()
    assert lib.zbal_moe_rms_norm(ok, None, None, 1e-6, ok, None, None, None, None, None, 0) == INVALID
    assert "comm is null" in capi.last_error()
    for args, name in (((None, ok, None, None, 1e-6, ok), "grad"), ((ok, None, None, None, 1e-6, ok), "x"), ((ok, ok, None, None, 1e-6, None), "gradX")):
        assert lib.zbal_moe_rms_norm_backward(*args, None, None, None, None, 0) == INVALID
        assert name + " is null" in capi.last_error()
    for args, name in (((None, None, 0, ok, ok), "x"), ((ok, None, 0, None, ok), "quantized"), ((ok, None, 0, ok, None), "scales")):
        assert lib.zbal_moe_quantize_rows(*args, None, None, 0) == INVALID
        assert name + " is null" in capi.last_error()
    assert lib.zbal_moe_quantize_rows(ok, None, 6, ok, ok, None, None, 0) == INVALID
    assert "activation" in capi.last_error()
    for i, name in enumerate(("x", "xScales", "weight", "weightScales")):
        four = [ok] * 4
        four[i] = None
        assert lib.zbal_moe_expert_linear_int8(*four, None, None, 0, None, ok, None, None, None, 0) == INVALID
        assert name + " is null" in capi.last_error()
    assert lib.zbal_moe_expert_linear_int8(ok, ok, ok, ok, None, None, 9, None, ok, None, None, None, 0) == INVALID
    assert "activation" in capi.last_error()
