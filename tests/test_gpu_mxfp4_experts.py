"""The expert layer on MXFP4 weights against a 64-bit reference, and its entry points."""
import numpy as np
import pytest
import torch

from tests import mx_reference as R

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import moe_ascend_opt_b200  # noqa: F401
    from moe_ascend_opt_b200 import capi

ops = torch.ops.nanovllm
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def weights(E, H, I, seed):
    rng = np.random.default_rng(seed)
    c13, s13 = R.quantize(0.02 * rng.standard_normal((E, 2 * I, H)))
    c2, s2 = R.quantize(0.02 * rng.standard_normal((E, H, I)))
    return (R.pack(c13), s13, R.pack(c2), s2), R.decode(c13, s13), R.decode(c2, s2)


def handle(E, H, I, packed):
    h = torch.classes.nanovllm.MoEInfer(E, H, I, 3)
    h.store_mxfp4(*[torch.from_numpy(p) for p in packed])
    return h


def tokens(T, H, E, K, seed, dtype="bfloat16"):
    rng = np.random.default_rng(seed + 1)
    x = cuda(rng.standard_normal((T, H)) * np.exp(0.5 * rng.standard_normal(H))).to(TYPES[dtype])
    ids = np.stack([rng.permutation(E)[:K] for _ in range(T)]).astype(np.int32).reshape(T, K)
    w = rng.random((T, K)).astype(np.float32) + 0.05
    return x, ids, w / w.sum(1, keepdims=True)


def close(y, want, tol):
    y = y.double().cpu().numpy()
    bad = ~(np.abs(y - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], np.abs(y - want).max(), bad.sum())


SHAPES = [(4, 64, 32, 2), (8, 256, 96, 3), (16, 512, 160, 8), (3, 96, 64, 3), (1, 128, 128, 1), (40, 320, 224, 6)]


@pytest.mark.parametrize("E,H,I,K", SHAPES)
@pytest.mark.parametrize("T", [1, 2, 7, 33, 150, 700])
def test_forward(E, H, I, K, T):
    packed, w13, w2 = weights(E, H, I, E + H)
    h = handle(E, H, I, packed)
    for dtype in ("bfloat16", "float16"):
        x, ids, w = tokens(T, H, E, K, T, dtype)
        y = ops.moe_forward(x, cuda(ids), cuda(w), h)
        assert h.device_error() == 0 and y.dtype == x.dtype
        want, tol = R.experts(x.double().cpu().numpy(), ids, w, w13, w2, dtype)
        close(y, want, tol)
    p = ops.moe_forward_partial(x, cuda(ids), cuda(w), h)
    close(p, want, R.experts(x.double().cpu().numpy(), ids, w, w13, w2, "float32")[1])


def test_one_expert_takes_all():
    """More than one tile of rows for an expert, others empty."""
    E, H, I, K, T = 6, 128, 64, 2, 300
    packed, w13, w2 = weights(E, H, I, 3)
    x, ids, w = tokens(T, H, E, K, 5)
    w *= 1e3  # parts of very different sizes in a sum
    ids[:, 0], ids[:, 1] = 4, np.where(np.arange(T) % 97 == 0, 2, 5)
    want, tol = R.experts(x.double().cpu().numpy(), ids, w, w13, w2, "bfloat16")
    close(ops.moe_forward(x, cuda(ids), cuda(w), handle(E, H, I, packed)), want, tol)


@pytest.mark.parametrize("T", [1, 5, 140])
def test_skipped_ids(T):
    """Ids outside the engine's experts are left out; a token that keeps none is zero; an id twice counts twice."""
    E, H, I, K = 8, 128, 96, 4
    packed, w13, w2 = weights(E, H, I, 4)
    h = handle(E, H, I, packed)
    x, ids, w = tokens(T, H, E, K, 6)
    ids[0] = [-1, E, 1 << 30, -(1 << 31)]
    if T > 2:
        ids[1], ids[2] = [3, 3, 3, -1], [7, -5, 7, 0]
        ids[T - 1] = -1
    y = torch.full((T, H), 7.0, device="cuda", dtype=x.dtype)
    ctx = torch.classes.nanovllm.MoEGraphContext(h, T, K, 1)
    ops.moe_forward_npu_graph_out(x, cuda(ids), cuda(w), h, ctx, y)
    want, tol = R.experts(x.double().cpu().numpy(), ids, w, w13, w2, "bfloat16")
    close(y, want, tol)
    assert not y[0].any() and (T < 3 or not y[T - 1].any())


def test_nan_tokens_stay_apart():
    E, H, I, K, T = 8, 256, 128, 4, 70
    packed, _, _ = weights(E, H, I, 7)
    h = handle(E, H, I, packed)
    x, ids, w = tokens(T, H, E, K, 8)
    clean = ops.moe_forward(x, cuda(ids), cuda(w), h)
    x2 = x.clone()
    x2[13, 40], x2[60, 3] = float("nan"), float("inf")
    y = ops.moe_forward(x2, cuda(ids), cuda(w), h)
    assert y[13].isnan().all() and y[60].isnan().all()
    keep = torch.ones(T, dtype=torch.bool, device="cuda")
    keep[13] = keep[60] = False
    assert torch.equal(y[keep], clean[keep])


def test_rows_do_not_depend_on_the_batch():
    """A token's row is the same whatever else is in the call, and from call to call."""
    E, H, I, K, T = 16, 256, 160, 4, 400
    packed, _, _ = weights(E, H, I, 9)
    h = handle(E, H, I, packed)
    x, ids, w = tokens(T, H, E, K, 10)
    idc, wc = cuda(ids), cuda(w)
    full = ops.moe_forward_partial(x, idc, wc, h)
    assert torch.equal(full, ops.moe_forward_partial(x, idc, wc, h))
    half = ops.moe_forward(x, idc, wc, h)
    assert torch.equal(half, ops.moe_forward(x, idc, wc, h))
    for n in (1, 3, 64, 129):
        assert torch.equal(full[:n], ops.moe_forward_partial(x[:n], idc[:n].contiguous(), wc[:n].contiguous(), h))


def test_long_call_in_slices():
    E, H, I, K, T = 8, 32, 32, 8, 40000
    packed, w13, w2 = weights(E, H, I, 12)
    h = handle(E, H, I, packed)
    x, ids, w = tokens(T, H, E, K, 13)
    y = ops.moe_forward(x, cuda(ids), cuda(w), h)
    some = np.concatenate([np.arange(20), np.arange(32760, 32780), np.arange(T - 20, T)])
    want, tol = R.experts(x.double().cpu().numpy()[some], ids[some], w[some], w13, w2, "bfloat16")
    close(y[torch.from_numpy(some).cuda()], want, tol)


def test_graph_growth_and_streams():
    """A captured call keeps its results when the workspace grows after the capture; eager calls on two streams."""
    E, H, I, K = 8, 256, 128, 4
    packed, _, _ = weights(E, H, I, 14)
    h = handle(E, H, I, packed)
    x, ids, w = tokens(9, H, E, K, 15)
    idc, wc = cuda(ids), cuda(w)
    ctx = torch.classes.nanovllm.MoEGraphContext(h, 9, K, 1)
    y = torch.empty_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.moe_forward_npu_graph_out(x, idc, wc, h, ctx, y)
    big, bids, bw = tokens(600, H, E, K, 16)
    bids, bw = cuda(bids), cuda(bw)
    first = ops.moe_forward(big, bids, bw, h)  # outgrows the captured workspace
    for seed in (1, 2):
        x.copy_(tokens(9, H, E, K, 20 + seed)[0])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.moe_forward(x, idc, wc, h))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for i in range(6):
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            outs.append(ops.moe_forward(big, bids, bw, h))
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)
    with pytest.raises(RuntimeError, match="before capture"):
        g2 = torch.cuda.CUDAGraph()
        huge, hids, hw = tokens(3000, H, E, K, 17)
        hids, hw = cuda(hids), cuda(hw)
        with torch.cuda.graph(g2):
            ops.moe_forward(huge, hids, hw, h)
    torch.cuda.synchronize()
    assert torch.equal(ops.moe_forward(big, bids, bw, h), first)


def test_expert_parallel_parts_sum_to_the_layer():
    E, H, I, K, T = 12, 128, 96, 4, 50
    packed, w13, w2 = weights(E, H, I, 18)
    x, ids, w = tokens(T, H, E, K, 19)
    idc, wc = cuda(ids), cuda(w)
    total = torch.zeros(T, H, device="cuda")
    for part in ([0, 3, 7, 11], [1, 2, 4, 5, 6, 8, 9, 10]):
        h = torch.classes.nanovllm.MoEInfer(E, H, I, 3)
        h.set_expert_placement(part)
        h.store_mxfp4(*[cuda(p) for p in packed])
        total += ops.moe_forward_partial(x, idc, wc, h)
    want, tol = R.experts(x.double().cpu().numpy(), ids, w, w13, w2, "float32")
    close(total, want, 2 * tol)
    rank = torch.classes.nanovllm.MoEInfer(E, H, I, 3)
    rank.set_expert_parallel(1, 3)
    rank.store_mxfp4(*[torch.from_numpy(p) for p in packed])
    mine = np.where((ids >= 4) & (ids < 8), ids, -1)
    want, tol = R.experts(x.double().cpu().numpy(), mine, w, w13, w2, "bfloat16")
    close(ops.moe_forward(x, idc, wc, rank), want, tol)


@pytest.mark.parametrize("H,I", [(128, 96), (96, 32), (256, 160)])
def test_load_export_quantize_file(H, I, tmp_path):
    """The three ways to fill an engine hold the same bytes and give the same results."""
    E, K, T = 4, 2, 11
    rng = np.random.default_rng(21)
    wg, wu, wd = (0.02 * rng.standard_normal(s).astype(np.float32) for s in ((E, I, H), (E, I, H), (E, H, I)))
    c13, s13 = R.quantize(np.concatenate([wg, wu], 1))
    c2, s2 = R.quantize(wd)
    packed = (R.pack(c13), s13, R.pack(c2), s2)
    a = handle(E, H, I, packed)
    b = torch.classes.nanovllm.MoEInfer(E, H, I, 3)
    for e in range(E):
        b.quantize_and_store_expert(e, "gate_proj", torch.from_numpy(wg[e]))
        b.quantize_and_store_expert(e, "up_proj", torch.from_numpy(wu[e]).cuda())
        b.quantize_and_store_expert(e, "down_proj", torch.from_numpy(wd[e]))
    a.save(str(tmp_path / "w"))
    c = torch.classes.nanovllm.MoEInfer(E, H, I, 3)
    c.load_file(str(tmp_path / "w"))
    x, ids, w = tokens(T, H, E, K, 22)
    first = ops.moe_forward(x, cuda(ids), cuda(w), a)
    for h in (a, b, c):
        for e in range(E):
            for which, (q, s) in enumerate(((packed[0], s13), (packed[2], s2))):
                got = h.export_expert(e, which)
                np.testing.assert_array_equal(got[0].numpy(), q[e])
                np.testing.assert_array_equal(got[1].numpy(), s[e])
        assert torch.equal(ops.moe_forward(x, cuda(ids), cuda(w), h), first)
    other = torch.classes.nanovllm.MoEInfer(E, H, I, 1)
    with pytest.raises(RuntimeError, match="differs"):
        other.load_file(str(tmp_path / "w"))


@pytest.mark.parametrize("T", [1, 40, 200])
def test_dense_forward(T):
    E, H, I = 3, 256, 128
    packed, w13, w2 = weights(E, H, I, 23)
    h = handle(E, H, I, packed)
    x, _, _ = tokens(T, H, E, 1, 24)
    for e in (2, 0):
        want, tol = R.experts(x.double().cpu().numpy(), np.full((T, 1), e, np.int32), np.ones((T, 1)), w13, w2, "bfloat16")
        close(ops.moe_dense_forward(x, e, h), want, tol)


def test_refusals():
    E, H, I, K = 4, 64, 32, 2
    packed, _, _ = weights(E, H, I, 25)
    h = handle(E, H, I, packed)
    x, ids, w = tokens(5, H, E, K, 26)
    idc, wc = cuda(ids), cuda(w)
    with pytest.raises(RuntimeError, match="aligned"):
        ops.moe_forward(torch.zeros(5 * H + 1, device="cuda", dtype=torch.bfloat16)[1:].view(5, H), idc, wc, h)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.moe_forward(x.repeat(1, 2)[:, ::2], idc, wc, h)
    with pytest.raises(RuntimeError, match="float16 or bfloat16"):
        ops.moe_forward(x.float(), idc, wc, h)
    assert ops.moe_forward(x[:0], idc[:0], wc[:0], h).shape == (0, H)
    eng = capi.Engine(E, H, I, capi.MXFP4)
    with pytest.raises(capi.MoeError, match="no weights"):
        eng.forward(x, x, idc, wc, capi.BF16, capi.BF16)
    eng.load_mxfp4(*[torch.from_numpy(p) for p in packed])
    y = torch.empty_like(x)
    with pytest.raises(capi.MoeError, match="no no-allocation"):
        eng.forward_noalloc(x, y, idc, wc, capi.BF16, capi.BF16)
    with pytest.raises(capi.MoeError, match="peer combine"):
        capi.call("moe_engine_p2p_mailbox", eng.h, 2, 4, y.data_ptr())
    with pytest.raises(capi.MoeError, match="load_mxfp4"):
        eng.load_quantized(x, x, x, x, capi.F16)
    with pytest.raises(capi.MoeError, match="at most 1024"):
        capi.Engine(1025, 32, 32, capi.MXFP4)
    eng.forward(x, y, idc, wc, capi.BF16, capi.BF16)
    assert torch.equal(y, ops.moe_forward(x, idc, wc, h))


@pytest.mark.parametrize("T", [1, 6, 90])
def test_router_to_output(T):
    """Route by scores, run the routed layer, then a quantised linear layer, as a model's step does."""
    E, H, I, K, N = 32, 256, 96, 4, 192
    packed, w13, w2 = weights(E, H, I, 27)
    h = handle(E, H, I, packed)
    rng = np.random.default_rng(28)
    x = cuda(rng.standard_normal((T, H))).bfloat16()
    logits = cuda(rng.standard_normal((T, E)).astype(np.float32))
    logits[T - 1] = -float("inf")  # a padding row
    bias = cuda((0.1 * rng.standard_normal(E)).astype(np.float32))
    lw, ls = ops.quantize_rows_mxfp4(cuda(0.05 * rng.standard_normal((N, H)).astype(np.float32)), True)
    ids, w = ops.moe_route_scored(logits, bias, K, "sigmoid", 4, 2, 2, True, 2.5)
    y = ops.moe_forward(x, ids, w, h)
    z = ops.mxfp4_matmul(*ops.quantize_rows_mxfp4(y, True), lw, ls, torch.float32)
    ri, rw = R.route(logits.double().cpu().numpy(), bias.double().cpu().numpy(), K, "sigmoid", 4, 2, 2, True, 2.5)
    np.testing.assert_array_equal(ids.cpu().numpy(), ri)
    want, tol = R.experts(x.double().cpu().numpy(), ri, w.double().cpu().numpy(), w13, w2, "bfloat16")
    close(y, want, tol)
    assert not y[T - 1].any() and (ri[T - 1] == -1).all()
    a = R.decode(*R.quantize(y.double().cpu().numpy()))
    b = ops.dequantize_rows_mxfp4(lw, ls, torch.float32).double().cpu().numpy()
    close(z, a @ b.T, R.product_error(a, b) + R.HALF["float32"] * np.abs(a @ b.T))


@pytest.mark.parametrize("T,K", [(1, 16), (2, 8), (1, 20), (3, 33), (40, 64)])
def test_same_expert_many_times(T, K):
    """More pairs of one expert in a token than a tile of few rows holds, and long lists of ids."""
    E, H, I = 80, 128, 96
    packed, w13, w2 = weights(E, H, I, 30)
    h = handle(E, H, I, packed)
    x, ids, w = tokens(T, H, E, K, 31)
    for same in (True, False):
        if same:
            ids[:, : K - K // 4] = 7
        want, tol = R.experts(x.double().cpu().numpy(), ids, w, w13, w2, "bfloat16")
        close(ops.moe_forward(x, cuda(ids), cuda(w), h), want, tol)
        ids = tokens(T, H, E, K, 32)[1]


@pytest.mark.parametrize("E,H,I,K,T", [(1024, 64, 32, 8, 1), (1024, 64, 32, 8, 37), (1024, 64, 32, 8, 5000), (3, 8224, 32, 2, 1),
                                       (3, 8224, 32, 2, 5), (3, 64, 4128, 2, 2), (2, 32, 32, 1, 1), (2, 32, 32, 1, 513)])
def test_largest_and_smallest_sizes(E, H, I, K, T):
    packed, w13, w2 = weights(E, H, I, 33)
    h = handle(E, H, I, packed)
    x, ids, w = tokens(T, H, E, K, 34)
    y = ops.moe_forward(x, cuda(ids), cuda(w), h)
    some = np.unique(np.linspace(0, T - 1, 300).astype(int))
    want, tol = R.experts(x.double().cpu().numpy()[some], ids[some], w[some], w13, w2, "bfloat16")
    close(y[torch.from_numpy(some).cuda()], want, tol)


def test_expert_parallel_module():
    from moe_ascend_opt_b200.ep import ExpertParallelMoE
    E, H, I, K, T = 8, 128, 96, 4, 9
    packed, _, _ = weights(E, H, I, 46)
    x, ids, w = tokens(T, H, E, K, 47)
    moe = ExpertParallelMoE(E, H, I, 3)
    moe.load_mxfp4(*[torch.from_numpy(p) for p in packed])
    want = ops.moe_forward(x, cuda(ids), cuda(w), handle(E, H, I, packed))
    assert torch.equal(moe.forward(x, cuda(ids), cuda(w)), want)


@pytest.mark.parametrize("T", [1, 3, 60, 300])
def test_replicated_experts(T):
    """Ranks that share hot experts compute each pair once."""
    from moe_ascend_opt_b200.ep import replicated_placement
    E, H, I, K, W = 14, 128, 96, 4, 3
    packed, w13, w2 = weights(E, H, I, 35)
    x, ids, w = tokens(T, H, E, K, 36)
    pl, hot = replicated_placement(np.bincount(ids.ravel(), minlength=E), W, 2)
    total = torch.zeros(T, H, device="cuda")
    for r in range(W):
        h = torch.classes.nanovllm.MoEInfer(E, H, I, 3)
        h.set_expert_parallel(r, W)
        h.set_expert_placement(pl[r])
        h.set_expert_replicas(hot)
        h.store_mxfp4(*[torch.from_numpy(p) for p in packed])
        total += ops.moe_forward_partial(x, cuda(ids), cuda(w), h)
    want, tol = R.experts(x.double().cpu().numpy(), ids, w, w13, w2, "float32")
    close(total, want, W * tol)


@pytest.mark.parametrize("T", [1, 12, 400])
def test_captured_step_follows_its_routing(T):
    """Routing, experts and a product in one graph, replayed with other tokens, equal the eager calls."""
    E, H, I, K, N = 8, 256, 128, 2, 96
    packed, _, _ = weights(E, H, I, 37)
    h = handle(E, H, I, packed)
    x = tokens(T, H, E, K, 38)[0]
    rng = np.random.default_rng(39)
    logits = cuda(rng.standard_normal((T, E)).astype(np.float32))
    lw, ls = ops.quantize_rows_mxfp4(cuda(rng.standard_normal((N, H)).astype(np.float32)), True)

    def step():
        ids, w = ops.moe_route_scored(logits, None, K, "softmax", 1, 1, 1, True, 1.0)
        q, s = ops.quantize_rows_mxfp4(ops.moe_forward(x, ids, w, h), True)
        return ops.mxfp4_matmul(q, s, lw, ls, torch.bfloat16)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = step()
    for seed in (1, 2, 3):
        x.copy_(tokens(T, H, E, K, 40 + seed)[0])
        logits.copy_(cuda(np.random.default_rng(seed).standard_normal((T, E)).astype(np.float32)))
        if seed == 2:
            logits[:, 1:] = -float("inf")  # one expert takes every token's first place
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(z, step())
    assert h.device_error() == 0


def test_threads_with_streams_of_their_own():
    import threading
    E, H, I, K, T = 8, 256, 128, 4, 150
    packed, _, _ = weights(E, H, I, 44)
    x, ids, w = tokens(T, H, E, K, 45)
    idc, wc = cuda(ids), cuda(w)
    shared = handle(E, H, I, packed)
    first = ops.moe_forward(x, idc, wc, shared)
    q, s = ops.quantize_rows_mxfp4(x, True)
    product = ops.mxfp4_matmul(q, s, q, s, torch.float32)
    torch.cuda.synchronize()
    bad = []

    def work(i):
        own = handle(E, H, I, packed) if i % 2 else shared
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                y = ops.moe_forward(x, idc, wc, own)
                z = ops.mxfp4_matmul(*ops.quantize_rows_mxfp4(x, True), q, s, torch.float32)
                if not (torch.equal(y, first) and torch.equal(z, product)):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_slices_of_different_runs():
    """A long call whose last slice has more runs of the token kernel than the others: each token's row is that of
    a call by itself."""
    E, H, I, K, T = 1024, 32, 32, 51, 10260
    packed, _, _ = weights(E, H, I, 52)
    h = handle(E, H, I, packed)
    x, ids, w = tokens(T, H, E, K, 53)
    idc, wc = cuda(ids), cuda(w)
    y = ops.moe_forward_partial(x, idc, wc, h)
    for a, b in ((0, 300), (5000, 5300), (T - 300, T)):
        assert torch.equal(y[a:b], ops.moe_forward_partial(x[a:b], idc[a:b].contiguous(), wc[a:b].contiguous(), h))
    assert h.device_error() == 0


def test_reserved_for_one_token_more():
    """A captured call of fewer tokens than were reserved is accepted where the token kernel's runs change."""
    E, H, I, K, T = 128, 64, 32, 8, 16384
    packed, _, _ = weights(E, H, I, 54)
    h = handle(E, H, I, packed)
    x, ids, w = tokens(T, H, E, K, 55)
    idc, wc = cuda(ids), cuda(w)
    ctx = torch.classes.nanovllm.MoEGraphContext(h, T + 1, K, 1)
    y = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.moe_forward_npu_graph_out(x, idc, wc, h, ctx, y)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, ops.moe_forward(x, idc, wc, h))


def test_dense_calls_in_graphs():
    """A captured dense call keeps its expert: other experts, captures and longer calls in between change nothing."""
    E, H, I, T = 4, 256, 128, 6
    packed, _, _ = weights(E, H, I, 50)
    h = handle(E, H, I, packed)
    x = tokens(T, H, E, 1, 51)[0]
    one = torch.ones(T, 1, device="cuda")

    def routed(e):
        return ops.moe_forward(x, torch.full((T, 1), e, device="cuda", dtype=torch.int32), one, h)

    want = [routed(e) for e in range(E)]
    assert torch.equal(ops.moe_dense_forward(x, 0, h), want[0])
    graphs, outs = [], []
    for e in (0, 2):  # an expert that was called before, and a new one
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(ops.moe_dense_forward(x, e, h))
    assert torch.equal(ops.moe_dense_forward(x, 2, h), want[2])  # not replayed yet
    for e in (1, 3, 1):
        assert torch.equal(ops.moe_dense_forward(x, e, h), want[e])
        for graph, out, of in zip(graphs, outs, (0, 2)):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[of])


def test_dense_calls_after_growth_and_on_streams():
    """A captured dense call outlives longer calls of its expert; dense calls of two experts queued on two streams, and
    from threads, each keep theirs."""
    import threading
    E, H, I, T = 3, 256, 128, 30
    packed, _, _ = weights(E, H, I, 56)
    h = handle(E, H, I, packed)
    x = tokens(T, H, E, 1, 57)[0]
    want = [ops.moe_dense_forward(x, e, h) for e in range(E)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.moe_dense_forward(x, 1, h)
    ops.moe_dense_forward(tokens(3000, H, E, 1, 58)[0], 1, h)  # outgrows the captured routing
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want[1])
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(ops.moe_dense_forward(x, i % E, h))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i % E]) for i, o in enumerate(outs))
    fresh, bad = handle(E, H, I, packed), []

    def work(e):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                if not torch.equal(ops.moe_dense_forward(x, e, fresh), want[e]):
                    bad.append(e)

    threads = [threading.Thread(target=work, args=(e,)) for e in range(E)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_streams_that_take_over_a_handle():
    """Calls on a stream that is destroyed with work pending, then on a new stream that may have its handle."""
    import ctypes
    E, H, I, K, T = 8, 512, 256, 4, 4096
    packed, _, _ = weights(E, H, I, 59)
    h = handle(E, H, I, packed)
    x, ids, w = tokens(T, H, E, K, 60)
    idc, wc = cuda(ids), cuda(w)
    short = (x[:2], idc[:2].contiguous(), wc[:2].contiguous())
    want = ops.moe_forward(x, idc, wc, h), ops.moe_forward(*short, h)
    torch.cuda.synchronize()
    rt = torch.cuda.cudart()

    def create():
        p = ctypes.c_void_p()
        assert int(rt.cudaStreamCreate(ctypes.addressof(p))) == 0
        return p.value

    outs = []
    for _ in range(12):
        a = create()
        with torch.cuda.stream(torch.cuda.ExternalStream(a)):
            outs.append([ops.moe_forward(*short, h)] + [ops.moe_forward(x, idc, wc, h) for _ in range(6)])
        assert int(rt.cudaStreamDestroy(a)) == 0
    torch.cuda.synchronize()
    for first, *rest in outs:
        assert torch.equal(first, want[1]) and all(torch.equal(o, want[0]) for o in rest)


def test_branches_of_one_graph():
    """Calls that one capture takes from two streams without an order between them do not share the workspace at once."""
    E, H, I, K = 8, 512, 256, 4
    packed, _, _ = weights(E, H, I, 61)
    h = handle(E, H, I, packed)
    calls = []
    for T in (2000, 30, 2):
        x, ids, w = tokens(T, H, E, K, 62 + T)
        calls.append((x, cuda(ids), cuda(w)))
    want = [ops.moe_forward(*c, h) for c in calls] + [ops.moe_dense_forward(calls[0][0], 1, h)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    outs = []
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        for i in range(5):
            outs.append((0, ops.moe_forward(*calls[0], h)))
            with torch.cuda.stream(side):
                outs.append((3, ops.moe_dense_forward(calls[0][0], 1, h)))
                outs.append((1 + i % 2, ops.moe_forward(*calls[1 + i % 2], h)))
        main.wait_stream(side)
    for _ in range(3):
        for _, o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want[i]) for i, o in outs)
    again = torch.cuda.CUDAGraph()  # another capture does not wait for the first one's event
    with torch.cuda.graph(again, stream=side):
        o = ops.moe_forward(*calls[1], h)
    again.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, want[1]) and torch.equal(ops.moe_forward(*calls[0], h), want[0])


@pytest.mark.parametrize("T", [1, 20, 300])
def test_largest_gate(T):
    """SiLU of a gate near the largest float is the gate: g = 6 * 2^125, h = .75 g, y = 4 * 2^125 * 2^-120."""
    H = I = 32
    c13, s13 = np.zeros((1, 2 * I, H), np.uint8), np.full((1, 2 * I, 1), 127, np.uint8)
    c13[0, :I, 0], c13[0, I:, 0], s13[0, I:] = 2, 1, 0  # gate weight 1, up weight 2^-128
    c2, s2 = np.zeros((1, H, I), np.uint8), np.full((1, H, 1), 7, np.uint8)
    c2[0, :, 0] = 2
    h = handle(1, H, I, (R.pack(c13), s13, R.pack(c2), s2))
    x = torch.zeros(T, H, device="cuda", dtype=torch.bfloat16)
    x[:, 0] = 2.5e38
    y = ops.moe_forward(x, torch.zeros(T, 1, device="cuda", dtype=torch.int32), torch.ones(T, 1, device="cuda"), h)
    assert (y == 128).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("T", [8, 40, 300])
def test_columns_beside_a_large_one(T, dtype):
    """An output column 2^12 times its neighbours takes no bits from them, however many rows the call has: parts
    and sums hold 32 bits, the output is rounded once."""
    E, H, I, K = 4, 96, 64, 2
    rng = np.random.default_rng(48)
    c13, s13 = R.quantize(0.05 * rng.standard_normal((E, 2 * I, H)))
    w2 = 0.02 * rng.standard_normal((E, H, I))
    w2[:, 5] *= 4096.0
    w2[:, 70] *= 4096.0
    c2, s2 = R.quantize(w2)
    h = handle(E, H, I, (R.pack(c13), s13, R.pack(c2), s2))
    x, ids, w = tokens(T, H, E, K, 49, dtype)
    want, tol = R.experts(x.double().cpu().numpy(), ids, w, R.decode(c13, s13), R.decode(c2, s2), "float32")
    tol = tol + R.HALF[dtype] * (np.abs(want) + tol) + (2.0 ** -25 if dtype == "float16" else 0.0)
    close(ops.moe_forward(x, cuda(ids), cuda(w), h), want, tol)


def test_sixteen_bit_rows_do_not_depend_on_the_batch():
    """As for fp32 outputs: the plan that a call of many rows takes gives the bits of the plan for few."""
    E, H, I, K, T = 4, 256, 160, 2, 400
    packed, _, _ = weights(E, H, I, 63)
    h = handle(E, H, I, packed)
    for dtype in ("bfloat16", "float16"):
        x, ids, w = tokens(T, H, E, K, 64, dtype)
        idc, wc = cuda(ids), cuda(w)
        full = ops.moe_forward(x, idc, wc, h)
        for n in (1, 3, 64, 129):
            assert torch.equal(full[:n], ops.moe_forward(x[:n], idc[:n].contiguous(), wc[:n].contiguous(), h))


@pytest.mark.parametrize("T", [20, 300, 1000])
def test_a_ranks_rows_are_the_layers(T):
    """A rank's fp32 part has the bits of the whole engine's with the other ranks' pairs left out, whatever tiles
    either takes; the C engine with its number of experts told, too."""
    E, H, I, K, W = 64, 128, 96, 4, 8
    packed, _, _ = weights(E, H, I, 65)
    whole = handle(E, H, I, packed)
    x, ids, w = tokens(T, H, E, K, 66)
    idc, wc = cuda(ids), cuda(w)
    for r in (0, 5):
        lo, hi = r * E // W, (r + 1) * E // W
        want = ops.moe_forward_partial(x, cuda(np.where((ids >= lo) & (ids < hi), ids, -1)), wc, whole)
        rank = torch.classes.nanovllm.MoEInfer(E, H, I, 3)
        rank.set_expert_parallel(r, W)
        rank.store_mxfp4(*[torch.from_numpy(p) for p in packed])
        assert torch.equal(ops.moe_forward_partial(x, idc, wc, rank), want)
        eng = capi.Engine(E // W, H, I, capi.MXFP4, expert_offset=lo)
        eng.load_mxfp4(*[torch.from_numpy(p[lo:hi].copy()) for p in packed])
        for n in (E, E // W):
            eng.set_layer_experts(n)
            y = torch.empty(T, H, device="cuda")
            eng.forward(x, y, idc, wc, capi.BF16, capi.F32)
            assert torch.equal(y, want)
        with pytest.raises(capi.MoeError, match="at least the engine"):
            eng.set_layer_experts(E // W - 1)
    one = torch.ones(T, 1, device="cuda")
    for e in (0, 9):
        want = ops.moe_forward(x, torch.full((T, 1), e, device="cuda", dtype=torch.int32), one, whole)
        assert torch.equal(ops.moe_dense_forward(x, e, whole), want)


@pytest.mark.parametrize("T", [5, 100])
def test_dense_call_of_a_replicated_expert(T):
    """It takes every token on the rank that makes it, not the rank's share of routed pairs."""
    E, H, I, W = 6, 128, 96, 3
    packed, _, _ = weights(E, H, I, 67)
    whole = handle(E, H, I, packed)
    x, _, _ = tokens(T, H, E, 1, 68)
    h = torch.classes.nanovllm.MoEInfer(E, H, I, 3)
    h.set_expert_parallel(1, W)
    h.set_expert_placement([4, 0, 5])
    h.set_expert_replicas([0])
    h.store_mxfp4(*[torch.from_numpy(p) for p in packed])
    for e in (4, 0, 5):
        assert torch.equal(ops.moe_dense_forward(x, e, h), ops.moe_dense_forward(x, e, whole))
    with pytest.raises(RuntimeError, match="not held"):
        ops.moe_dense_forward(x, 1, h)
