"""Host-side checks of the group router, the experts' products and the combine's gradient that need no GPU: struct layouts, sizes and
arguments that the launchers and the C ABI refuse before anything reaches a device."""
import ctypes
import os
import subprocess

import pytest

from memfabric_hybrid_amd import capi

INC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
INVALID = capi.Z_INVALID_PARAM


@pytest.fixture(scope="module")
def lib():
    return capi.load()


def test_struct_layouts(tmp_path):
    src, exe = tmp_path / "t.c", tmp_path / "t"
    src.write_text('#include "zbal.h"\n#include "zbal_hip_kernels.h"\n#include <stdio.h>\n'
                   'int main(void){printf("%zu %zu %zu %zu", sizeof(zbalhip_group_route_t), __builtin_offsetof(zbalhip_group_route_t, bias),'
                   'sizeof(zbalhip_expert_linear_t), __builtin_offsetof(zbalhip_expert_linear_t, rows));return 0;}\n')
    subprocess.check_call(["gcc", "-I", INC, str(src), "-o", str(exe)])
    got = [int(v) for v in subprocess.check_output([str(exe)]).split()]
    assert got == [ctypes.sizeof(capi.GroupRoute), capi.GroupRoute.bias.offset, ctypes.sizeof(capi.ExpertLinear), capi.ExpertLinear.rows.offset]


def route(**kw):
    d = dict(logits=4096, dtype=capi.DT_FP32, score=0, group_score=0, renormalize=1, scale=1.0, bias=None, tokens=4, experts=64, topk=8, groups=8,
             kept_groups=4)
    d.update(kw)
    return capi.GroupRoute(**d)


@pytest.mark.parametrize("kw", [dict(tokens=-1), dict(tokens=1 << 31), dict(tokens=1 << 24), dict(experts=0), dict(experts=1032), dict(topk=0), dict(topk=33), dict(groups=0),
                                dict(groups=5), dict(groups=128, experts=1024), dict(kept_groups=0), dict(kept_groups=9), dict(topk=9, kept_groups=1),
                                dict(score=2), dict(score=-1), dict(group_score=2), dict(dtype=capi.DT_INT32), dict(logits=None)])
def test_route_refusals(lib, kw):
    assert lib.zbalhip_group_route(ctypes.byref(route(**kw)), 4096, 1, 4096, None) == INVALID
    if not set(kw) & {"groups", "kept_groups", "group_score"}:
        assert lib.zbalhip_group_route_backward(ctypes.byref(route(**kw)), 4096, 4096, 1, 4096, None) == INVALID


def test_route_null_pointers_and_empty_batches(lib):
    d = route()
    assert lib.zbalhip_group_route(None, 4096, 1, 4096, None) == INVALID
    assert lib.zbalhip_group_route(ctypes.byref(d), None, 1, 4096, None) == INVALID
    assert lib.zbalhip_group_route(ctypes.byref(d), 4096, 1, None, None) == INVALID
    for args in ((None, 4096, 4096), (4096, None, 4096), (4096, 4096, None)):
        assert lib.zbalhip_group_route_backward(ctypes.byref(d), args[0], args[1], 1, args[2], None) == INVALID
    none = route(tokens=0, logits=None)
    assert lib.zbalhip_group_route(ctypes.byref(none), None, 1, None, None) == 0
    assert lib.zbalhip_group_route_backward(ctypes.byref(none), None, None, 1, None, None) == 0


def linear(**kw):
    d = dict(weight=4096, weight_is_nk=0, dtype=capi.DT_BF16, counts=4096, counts_are_i64=0, activation=0, rows=16, k=64, n=64, experts=2)
    d.update(kw)
    return capi.ExpertLinear(**d)


SIZES = [dict(rows=-1), dict(rows=(1 << 24) + 1), dict(k=0), dict(n=0), dict(k=65537), dict(n=65537), dict(experts=0), dict(experts=1025), dict(dtype=capi.DT_FP32),
         dict(activation=-1), dict(activation=6), dict(activation=5, n=63)]


@pytest.mark.parametrize("kw", SIZES + [dict(weight=None), dict(counts=None)])
def test_linear_refusals(lib, kw):
    d = ctypes.byref(linear(**kw))
    assert lib.zbalhip_expert_linear(d, 4096, None, 0, None, 4096, 0, None, None, 0, None) == INVALID
    assert lib.zbalhip_expert_linear_backward(d, 4096, 0, 4096, 4096, 4096, 4096, None, 0, 4096, None, 0, None) == INVALID
    if kw in SIZES:
        assert lib.zbalhip_expert_linear_workspace(d, 0) == lib.zbalhip_expert_linear_workspace(d, 1) == -1


def test_linear_null_pointers(lib):
    d, silu = ctypes.byref(linear()), ctypes.byref(linear(activation=2))
    assert lib.zbalhip_expert_linear(None, 4096, None, 0, None, 4096, 0, None, None, 0, None) == INVALID
    assert lib.zbalhip_expert_linear(d, None, None, 0, None, 4096, 0, None, None, 0, None) == INVALID
    assert lib.zbalhip_expert_linear(d, 4096, None, 0, None, None, 0, None, None, 0, None) == INVALID
    back = lib.zbalhip_expert_linear_backward
    assert back(d, None, 0, 4096, None, 4096, 4096, None, 0, None, None, 0, None) == INVALID          # no gradient
    assert back(d, 4096, 0, None, None, 4096, 4096, None, 0, None, None, 0, None) == INVALID          # no rows for the weights' gradient
    assert back(silu, 4096, 0, 4096, None, 4096, 4096, None, 0, 4096, None, 0, None) == INVALID       # no pre-activation
    assert back(silu, 4096, 0, 4096, 4096, 4096, 4096, None, 0, None, None, 0, None) == INVALID       # nowhere to put its gradient
    assert back(d, 4096, 1, 4096, None, 4096, 4096, None, 0, None, None, 0, None) == INVALID          # nor that of 32 bits, rounded
    assert back(d, 4096, 0, 4096, None, 4096, None, 4096, 0, None, None, 0, None) == INVALID          # the bias's alone
    assert back(d, 4096, 0, 4096, None, None, None, None, 0, None, None, 0, None) == 0                # nothing asked for
    none = ctypes.byref(linear(rows=0))
    assert lib.zbalhip_expert_linear(none, None, None, 0, None, None, 0, None, None, 0, None) == 0


def test_workspace_sizes(lib):
    f = lib.zbal_moe_expert_linear_workspace_size
    for backward in (0, 1):
        for rows, k, n, e in ((0, 64, 64, 1), (1, 7168, 256, 1), (4096, 7168, 256, 1), (32768, 2048, 4096, 32), (1 << 24, 65536, 65536, 1)):
            b = f(rows, k, n, e, 0, capi.DT_BF16, capi.WEIGHT_FORMAT_ND, backward)
            assert 0 <= b < 1 << 32
            assert b == 0 or e == 1
        assert f(16, 64, 64, 1, 0, capi.DT_BF16, capi.WEIGHT_FORMAT_PREPACKED, backward) == -1
        assert f(16, 64, 63, 1, 5, capi.DT_BF16, capi.WEIGHT_FORMAT_ND, backward) == -1


@pytest.mark.parametrize("kw", [dict(dtype=capi.DT_FP32), dict(tokens=-1), dict(tokens=1 << 24), dict(hidden=0), dict(hidden=20), dict(topk=0), dict(topk=33), dict(experts=0), dict(rows=-1),
                                dict(grad=None), dict(y=None), dict(out=None)])
def test_combine_refusals(lib, kw):
    d = dict(grad=4096, y=4096, rows=8, dtype=capi.DT_BF16, tokens=4, hidden=64, topk=2, experts=8, out=4096)
    d.update(kw)
    assert lib.zbalhip_combine_backward(d["grad"], d["y"], d["rows"], d["dtype"], 4096, 4096, 4096, 0, 4096, d["tokens"], d["hidden"], d["topk"], d["experts"],
                                        d["out"], 4096, None) == INVALID


def test_outer_calls_check_their_arguments_first(lib):
    t = capi.TensorInfo()
    ok = ctypes.byref(t)
    assert lib.zbal_moe_group_route(None, None, 2, 1, 1, 0, 0, 1, 1.0, ok, ok, None, None, 0) == INVALID
    assert "logits is null" in capi.last_error()
    for topk, groups, kept, score, by, text in ((0, 1, 1, 0, 0, "topkNum"), (2, 0, 1, 0, 0, "groupNum"), (2, 2, 3, 0, 0, "topkGroupNum"), (2, 1, 1, 2, 0, "score"),
                                                (2, 1, 1, 0, 7, "groupScore")):
        assert lib.zbal_moe_group_route(ok, None, topk, groups, kept, score, by, 1, 1.0, ok, ok, None, None, 0) == INVALID
        assert text in capi.last_error()
    assert lib.zbal_moe_group_route(ok, None, 2, 1, 1, 0, 0, 1, 1.0, ok, ok, None, None, 0) == INVALID
    assert "comm is null" in capi.last_error()
    assert lib.zbal_moe_group_route_backward(ok, ok, ok, 5, 1, 1.0, ok, None, None, 0) == INVALID
    assert lib.zbal_moe_expert_linear(ok, None, None, None, 0, None, ok, None, None, None, None, 0) == INVALID
    assert lib.zbal_moe_expert_linear(ok, ok, None, None, 9, None, ok, None, None, None, None, 0) == INVALID
    assert lib.zbal_moe_expert_linear_backward(ok, ok, None, None, 0, None, None, None, None, None, None, None, None, 0) == INVALID
    assert lib.zbal_moe_expert_linear_backward(ok, ok, ok, None, 6, None, None, None, None, None, None, None, None, 0) == INVALID
    assert lib.zbal_combine_normal_backward(ok, ok, ok, ok, ok, None, 8, ok, ok, None, None, 0) == INVALID
    assert lib.zbal_combine_normal_backward(ok, ok, ok, ok, ok, ok, 0, ok, ok, None, None, 0) == INVALID
