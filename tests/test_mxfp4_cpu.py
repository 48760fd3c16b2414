"""Refusals of the routing and MXFP4 entry points, without a GPU."""
import ctypes as C

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
