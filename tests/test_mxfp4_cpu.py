"""Refusals of the routing and MXFP4 entry points, without a GPU."""
import ctypes as C
import os
import subprocess

import pytest
import torch

import moe_ascend_opt_b200  # noqa: F401
from moe_ascend_opt_b200 import capi

P = 1 << 20  # never dereferenced: the calls are refused on their arguments


def refused(name, *args, match):
    with pytest.raises(capi.MoeError, match=match) as e:
        capi.call(name, *args)
    assert e.value.code == capi.MOE_ERR_INVALID


def route(**kw):
    a = dict(logits=P, dtype=2, bias=None, T=4, E=64, K=8, score=0, groups=1, topk_groups=1, group_top=1, renorm=1, scale=1.0, ids=P, w=P)
    a.update(kw)
    return [a[k] for k in ("logits", "dtype", "bias", "T", "E", "K", "score", "groups", "topk_groups", "group_top", "renorm", "scale", "ids", "w")] + [None]


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=3), "logits must be"), (dict(T=-1), "num_tokens"), (dict(E=0), "num_experts"), (dict(E=1025), "num_experts"),
    (dict(score=2), "score"), (dict(groups=0), "num_groups"), (dict(groups=5), "num_groups"), (dict(groups=64), "num_groups"),
    (dict(groups=4, topk_groups=5), "topk_groups"), (dict(topk_groups=0), "topk_groups"), (dict(group_top=3), "group_top"),
    (dict(K=0), "top_k"), (dict(K=33), "top_k"), (dict(E=4, K=5), "top_k"), (dict(groups=32, topk_groups=2, K=5), "top_k"),
    (dict(scale=float("nan")), "scale"), (dict(logits=None), "null"), (dict(ids=None), "null"), (dict(w=None), "null")])
def test_route_refusals(kw, match):
    refused("moe_route_scored", *route(**kw), match=match)


def test_route_of_nothing():
    capi.call("moe_route_scored", *route(T=0, logits=None, ids=None, w=None))


def test_quantize_refusals():
    refused("moe_quantize_rows_mxfp4", P, 1, 4, 33, 0, P, P, None, match="multiple of 32")
    refused("moe_quantize_rows_mxfp4", P, 1, 4, 0, 0, P, P, None, match="multiple of 32")
    refused("moe_quantize_rows_mxfp4", P, 1, -1, 32, 0, P, P, None, match="multiple of 32")
    refused("moe_quantize_rows_mxfp4", P, 5, 4, 32, 0, P, P, None, match="dtype")
    refused("moe_quantize_rows_mxfp4", None, 1, 4, 32, 0, P, P, None, match="null")
    refused("moe_quantize_rows_mxfp4", P + 2, 1, 4, 32, 0, P, P, None, match="aligned")
    refused("moe_quantize_rows_mxfp4", P, 1, 4, 32, 1, P, P + 4, None, match="aligned")
    refused("moe_dequantize_rows_mxfp4", P, P, 4, 32, 0, P, 7, None, match="dtype")
    refused("moe_dequantize_rows_mxfp4", P, P, 4, 32, 0, P + 8, 1, None, match="aligned")
    refused("moe_dequantize_rows_mxfp4", P, None, 4, 32, 0, P, 1, None, match="null")
    refused("moe_mxfp4_tile_scales", P, 4, 40, P, None, match="multiple of 32")
    refused("moe_mxfp4_tile_scales", P, 4, 32, None, None, match="null")
    refused("moe_mxfp4_tile_scales", P, 4, 32, P + 1, None, match="aligned")
    capi.call("moe_quantize_rows_mxfp4", None, 1, 0, 32, 0, None, None, None)


def test_product_refusals():
    def mm(a=P, sa=P, b=P, sb=P, M=4, N=8, K=64, y=P, dt=1):
        return ("moe_mxfp4_matmul", a, sa, b, sb, M, N, K, y, dt, None)
    refused(*mm(K=48), match="multiple of 32")
    refused(*mm(K=0), match="multiple of 32")
    refused(*mm(N=0), match="positive")
    refused(*mm(M=-1), match="K must be")
    refused(*mm(M=1 << 31), match="too large")
    refused(*mm(dt=9), match="output dtype")
    refused(*mm(b=None), match="null")
    for k in ("a", "sa", "b", "sb", "y"):
        refused(*mm(**{k: P + 8}), match="aligned")
    capi.call(*mm(M=0, a=None, y=None))


def test_engine_refusals():
    L = capi.lib()
    assert L.moe_engine_load_mxfp4(None, None, None, None, None, 0, None) == capi.MOE_ERR_INVALID
    cfg = capi.MoeConfig(8, 100, 64, capi.MXFP4, 0, 0, 0)
    assert L.moe_engine_create(C.byref(cfg), C.byref(C.c_void_p())) == capi.MOE_ERR_INVALID


def test_handle_checks_before_device_work():
    h = torch.classes.nanovllm.MoEInfer(8, 256, 128, 3)
    assert h.get_quant_type() == "MXFP4"

    def z(*s, dtype=torch.uint8):
        return torch.zeros(s, dtype=dtype)
    good = [z(8, 256, 128), z(8, 256, 8), z(8, 256, 64), z(8, 256, 4)]
    with pytest.raises(RuntimeError, match="use store_mxfp4"):
        h.store_quantized_repack(*good)
    for i, name in enumerate(("w13", "w13_scales", "w2", "w2_scales")):
        bad = list(good)
        bad[i] = good[i][:, :, 1:]
        with pytest.raises(RuntimeError, match=name + " must be"):
            h.store_mxfp4(*bad)
        bad[i] = good[i].to(torch.int32)
        with pytest.raises(RuntimeError, match=name + " must be uint8"):
            h.store_mxfp4(*bad)
    with pytest.raises(RuntimeError, match="needs quant_type 3"):
        torch.classes.nanovllm.MoEInfer(8, 256, 128, 1).store_mxfp4(*good)


def test_ops_have_no_cpu_form():
    x = torch.zeros(4, 64)
    for call in (lambda: torch.ops.nanovllm.moe_route_scored(x, None, 2, "softmax"), lambda: torch.ops.nanovllm.quantize_rows_mxfp4(x),
                 lambda: torch.ops.nanovllm.mxfp4_tile_scales(torch.zeros(4, 2, dtype=torch.uint8))):
        with pytest.raises(NotImplementedError):
            call()


PLAN = r"""
#include "mx_plan.h"
using namespace moe::layer;
extern "C" int64_t layout_bytes(int64_t E, int64_t H, int64_t I, int64_t T, int64_t K) { return layout_of({E, H, I}, T, K).bytes; }
extern "C" int64_t call_size(int64_t E, int64_t H, int64_t I, int64_t T, int64_t K) { return call_bytes({E, H, I}, T, K); }
extern "C" int64_t reserve_size(int64_t E, int64_t H, int64_t I, int64_t T, int64_t K) { return reserve_bytes({E, H, I}, T, K); }
extern "C" int64_t slice(int64_t T, int64_t K) { return slice_tokens(T, K); }
extern "C" int64_t runs(int64_t T, int64_t K) { return ceil_div(T, prep_tokens(T, K, 148)); }
extern "C" int64_t runs_most(int64_t T, int64_t K) { return runs_bound(T, K); }
// the first t in [lo, hi] whose layout is larger than `bytes`, or 0
extern "C" int64_t first_above(int64_t E, int64_t H, int64_t I, int64_t K, int64_t lo, int64_t hi, int64_t bytes) {
    for (int64_t t = lo; t <= hi; ++t)
        if ((int64_t)layout_of({E, H, I}, t, K).bytes > bytes) return t;
    return 0;
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """The host arithmetic of the expert layer's workspace, compiled by itself."""
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(PLAN)
    csrc = os.path.join(os.path.dirname(moe_ascend_opt_b200.__file__), "csrc")
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I", csrc, str(d / "plan.cpp"), "-o", str(d / "plan.so")])
    lib = C.CDLL(str(d / "plan.so"))
    for f in ("layout_bytes", "call_size", "reserve_size", "slice", "runs", "runs_most", "first_above"):
        getattr(lib, f).restype = C.c_int64
    return lambda name, *a: getattr(lib, name)(*[C.c_int64(v) for v in a])


SHAPES = [(128, 2048, 768, 8), (1024, 32, 32, 51), (1024, 32, 32, 1), (1, 32, 32, 1), (3, 8224, 32, 2), (64, 2048, 768, 64), (8, 64, 32, 9)]


@pytest.mark.parametrize("E,H,I,K", SHAPES)
def test_reserve_covers_every_shorter_call(plan, E, H, I, K):
    """What is reserved for T tokens holds every call of fewer: runs of the token kernel, plans and slices that change."""
    S = plan("slice", 1 << 40, K)
    ends = {1, 2, 8 // K, (56 * E - 1) // K, 56 * E // K, 4096 // K, 4096 // K + 1, S, S + 1, 3 * S}
    ends |= {512 * n * max(1, 256 // K) + d for n in (1, 2) for d in (-1, 0, 1)} | {16384, 16385, 20000}
    for T in sorted(t for t in ends if 0 < t):
        assert plan("first_above", E, H, I, K, 1, min(T, S), plan("reserve_size", E, H, I, T, K)) == 0, T


@pytest.mark.parametrize("E,H,I,K", SHAPES)
def test_every_slice_of_a_call_fits(plan, E, H, I, K):
    """The last slice of a long call is shorter and may need more than the others."""
    S = plan("slice", 1 << 40, K)
    for T in list(range(1, 400, 7)) + [S - 1, S, S + 1, 2 * S - 1] + [S + n for n in range(1, S, max(1, S // 700))]:
        size = plan("call_size", E, H, I, T, K)
        for t in {min(T, S), T % min(T, S)} - {0}:
            assert plan("layout_bytes", E, H, I, t, K) <= size, (T, t)
            if t * K > 4096:
                assert plan("runs", t, K) <= plan("runs_most", t, K)
    if (E, H, I, K) == (1024, 32, 32, 51):
        assert plan("layout_bytes", E, H, I, 5120, K) <= plan("call_size", E, H, I, 10260, K)


RANK = r"""
#include "mx_plan.h"
using namespace moe::layer;
extern "C" int64_t plan(int64_t E, int64_t all, int64_t T, int64_t K) { return plan_of({E, 2048, 768, all}, T, K); }
extern "C" int64_t reserve_size(int64_t E, int64_t all, int64_t T, int64_t K) { return reserve_bytes({E, 2048, 768, all}, T, K); }
extern "C" int64_t call_size(int64_t E, int64_t all, int64_t T, int64_t K) { return call_bytes({E, 2048, 768, all}, T, K); }
"""
FUSED, SLIM, WIDE = 0, 1, 2


@pytest.fixture(scope="module")
def rank_plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("rank")
    (d / "rank.cpp").write_text(RANK)
    csrc = os.path.join(os.path.dirname(moe_ascend_opt_b200.__file__), "csrc")
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I", csrc, str(d / "rank.cpp"), "-o", str(d / "rank.so")])
    lib = C.CDLL(str(d / "rank.so"))
    for f in ("plan", "reserve_size", "call_size"):
        getattr(lib, f).restype = C.c_int64
    return lambda name, *a: getattr(lib, name)(*[C.c_int64(v) for v in a])


@pytest.mark.parametrize("W", [1, 2, 8])
def test_plan_of_a_rank(rank_plan, W):
    """A rank of W is given every rank's pairs and keeps a W-th: its tiles are those of the rows that its experts get."""
    E, K = 128, 8
    assert rank_plan("plan", E // W, E, 1, K) == FUSED
    for rows in (1, 7, 55):
        assert rank_plan("plan", E // W, E, rows * E // K, K) == SLIM
    for rows in (56, 57, 400):
        assert rank_plan("plan", E // W, E, rows * E // K, K) == WIDE
    assert rank_plan("plan", E, 0, 1000, K) == WIDE and rank_plan("plan", E, 0, 800, K) == SLIM


@pytest.mark.parametrize("E,all_", [(1, 1), (2, 0), (3, 24), (16, 128), (128, 0)])
def test_reserve_of_a_rank(rank_plan, E, all_):
    """It covers the routed calls and the dense ones, whose pairs are all the rank's."""
    for K in (1, 2, 8):
        if K <= max(E, all_):
            for T in (1, 8, 9, 55, 56, 57, 500, 3000):
                size = rank_plan("reserve_size", E, all_, T, K)
                assert all(rank_plan("call_size", E, 0, t, 1) <= size and rank_plan("call_size", E, all_, t, K) <= size
                           for t in range(1, T + 1)), (T, K)
