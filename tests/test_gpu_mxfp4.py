"""MXFP4 quantisation and the product of MXFP4 matrices against 64-bit references."""
import numpy as np
import pytest
import torch

from tests import mx_reference as R

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import moe_ascend_opt_b200  # noqa: F401

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
ops = torch.ops.nanovllm


def cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def special_values(rows, cols, seed):
    """Normal rows of very different sizes, blocks of zeros, ties, subnormals, the largest floats."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, cols)) * 2.0 ** rng.integers(-12, 12, (rows, cols // 32)).repeat(32, 1)
    flat = x.reshape(-1, 32)
    n = len(flat)
    flat[0] = 0.0
    mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.5, 7.0, 7.9])
    flat[n // 2] = np.concatenate([mids, -mids, [4.0], GRID_ALL(11)])[:32]
    flat[n // 3] = -0.0
    flat[-1, 0] = 2.0 ** -14
    return x


def GRID_ALL(n):
    return np.resize(R.GRID, n)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (257, 2048), (128, 128), (130, 160), (1, 4096), (1000, 64)])
def test_quantize_exact(rows, cols, dtype):
    x = cuda(special_values(rows, cols, rows + cols)).to(TYPES[dtype])
    codes, scales = R.quantize(x.double().cpu().numpy())
    q, s = ops.quantize_rows_mxfp4(x)
    np.testing.assert_array_equal(q.cpu().numpy(), R.pack(codes))
    np.testing.assert_array_equal(s.cpu().numpy(), scales)
    q2, t = ops.quantize_rows_mxfp4(x, True)
    assert torch.equal(q, q2)
    np.testing.assert_array_equal(t.cpu().numpy(), R.tile(scales))
    assert torch.equal(ops.mxfp4_tile_scales(s), t)
    want = R.decode(codes, scales)
    for out in sorted(TYPES):
        for sc in (s, t):
            y = ops.dequantize_rows_mxfp4(q, sc, TYPES[out])
            assert torch.equal(y.double().cpu(), torch.from_numpy(want).to(TYPES[out]).double()), out


def test_quantize_extremes():
    """Subnormals, the largest floats, infinities and NaN; every exponent of fp32."""
    f = np.finfo(np.float32)
    x = np.zeros((300, 32), np.float32)
    for i in range(254):
        x[i] = np.float32(2.0) ** (i - 126) * np.linspace(-1.999, 1.999, 32, dtype=np.float32)
    x[254] = f.max
    x[255, 0] = f.smallest_subnormal
    x[256] = np.arange(32) * f.smallest_subnormal
    x[257, 5] = f.tiny
    x[258, 3], x[259, 3], x[260, 3] = np.inf, -np.inf, np.nan
    x[261, 30], x[261, 31] = 1e-30, np.nan
    codes, scales = R.quantize(x.astype(np.float64))
    q, s = ops.quantize_rows_mxfp4(cuda(x))
    np.testing.assert_array_equal(s.cpu().numpy(), scales)
    good = scales[:, 0] != 255
    np.testing.assert_array_equal(q.cpu().numpy()[good], R.pack(codes)[good])
    y = ops.dequantize_rows_mxfp4(q, s, torch.float32).cpu().numpy()
    assert np.isnan(y[258:262]).all() and not np.isnan(y[:258]).any()
    np.testing.assert_array_equal(y[good], R.decode(codes, scales)[good].astype(np.float32))


def test_views_streams_and_empty():
    x = torch.randn(64, 512, device="cuda").bfloat16()
    for v in (x[:, 32:96], x[::3], x.t()[:, :32], x.flatten()[1:1 + 64 * 32].view(64, 32)):
        q, s = ops.quantize_rows_mxfp4(v)
        qc, sc = ops.quantize_rows_mxfp4(v.clone(memory_format=torch.contiguous_format))
        assert torch.equal(q, qc) and torch.equal(s, sc)
    q, s = ops.quantize_rows_mxfp4(x[:0], True)
    assert q.shape == (0, 256) and s.shape == (0, 4, 512)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        q, s = ops.quantize_rows_mxfp4(x, True)
        y = ops.dequantize_rows_mxfp4(q, s)
    st.synchronize()
    assert torch.equal(y, ops.dequantize_rows_mxfp4(*ops.quantize_rows_mxfp4(x)))


def test_binding_refusals():
    x = torch.randn(64, 64, device="cuda")
    q, s = ops.quantize_rows_mxfp4(x)
    t = ops.mxfp4_tile_scales(s)
    with pytest.raises(RuntimeError, match="multiple of 32"):
        ops.quantize_rows_mxfp4(x[:, :40])
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        ops.quantize_rows_mxfp4(x.double())
    with pytest.raises(RuntimeError, match="scales must be"):
        ops.dequantize_rows_mxfp4(q, s[:, :1])
    with pytest.raises(RuntimeError, match="tiled scales"):
        ops.mxfp4_matmul(q, s, q, t)
    with pytest.raises(RuntimeError, match="tiled scales"):
        ops.mxfp4_matmul(q, t, q, t[:, :, :256])
    with pytest.raises(RuntimeError, match="agree in K"):
        ops.mxfp4_matmul(q, t, *ops.quantize_rows_mxfp4(x.repeat(1, 2), True))
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        ops.mxfp4_matmul(q, t, q, t, torch.float64)
    with pytest.raises(RuntimeError, match="codes must be"):
        ops.mxfp4_matmul(q.float(), t, q, t)


def operands(M, N, K, seed, spread=3):
    rng = np.random.default_rng(seed)
    a = rng.standard_normal((M, K)) * 2.0 ** rng.integers(-spread, spread + 1, (M, K // 32)).repeat(32, 1)
    b = rng.standard_normal((N, K)) * 2.0 ** rng.integers(-spread, spread + 1, (N, K // 32)).repeat(32, 1)
    (ca, sa), (cb, sb) = R.quantize(a), R.quantize(b)
    dev = [cuda(R.pack(ca)), ops.mxfp4_tile_scales(cuda(sa)), cuda(R.pack(cb)), ops.mxfp4_tile_scales(cuda(sb))]
    return dev, R.decode(ca, sa), R.decode(cb, sb)


def check_product(M, N, K, seed, dtypes=("bfloat16",), spread=3):
    dev, a, b = operands(M, N, K, seed, spread)
    want, lost = a @ b.T, R.product_error(a, b)
    for dt in dtypes:
        y = ops.mxfp4_matmul(*dev, TYPES[dt]).double().cpu().numpy()
        tol = lost + R.HALF[dt] * (np.abs(want) + lost) + (2.0 ** -25 if dt == "float16" else 0.0)
        bad = ~(np.abs(y - want) <= tol)
        assert not bad.any(), (dt, np.argwhere(bad)[:5], np.abs(y - want).max(), bad.sum())


@pytest.mark.parametrize("K", [32, 64, 96, 128, 160, 256, 288, 512, 2048])
def test_product_depths(K):
    check_product(5, 40, K, K, sorted(TYPES))
    check_product(130, 136, K, K + 1)


@pytest.mark.parametrize("M", [1, 2, 8, 9, 31, 127, 128, 129, 300])
@pytest.mark.parametrize("N", [1, 16, 31, 128, 200, 520])
def test_product_shapes(M, N):
    check_product(M, N, 320, 1000 * M + N, ("float32",))


@pytest.mark.parametrize("M,N,K", [(1000, 1000, 1024), (1, 4096, 2048), (3, 2049, 4096), (2000, 96, 512), (4100, 1288, 288), (2333, 2050, 64), (1300, 4104, 96),
                                   (2500, 2050, 320), (5, 40000, 96), (130, 38000, 64)])
def test_product_large(M, N, K):
    check_product(M, N, K, M, ("bfloat16", "float16", "float32") if K < 1024 else ("bfloat16", "float32"))


def test_product_scale_range():
    """Scales over many octaves: the accumulation bound holds against the sum of magnitudes."""
    check_product(70, 90, 512, 4, ("float32",), spread=12)


def test_product_nan_rows_stay_apart():
    dev, a, b = operands(200, 150, 256, 9)
    s = R.tile(np.full((200, 8), 127, np.uint8))
    s[:] = dev[1].cpu().numpy()
    s[130 // 128, 1, 16 * (130 % 32) + 4 * (130 % 128 // 32)] = 255  # row 130, block 4
    y = ops.mxfp4_matmul(dev[0], cuda(s), dev[2], dev[3], torch.float32).cpu().numpy()
    ref = ops.mxfp4_matmul(*dev, torch.float32).cpu().numpy()
    assert np.isnan(y[130]).all()
    keep = np.arange(200) != 130
    np.testing.assert_array_equal(y[keep], ref[keep])


def test_linear_layer_and_graph():
    """Quantise and multiply as a linear layer does, eager, on another stream and replayed from a graph."""
    M, N, K = 33, 512, 1024
    w = torch.randn(N, K, device="cuda") * 0.02
    wq, ws = ops.quantize_rows_mxfp4(w, True)
    wv = ops.dequantize_rows_mxfp4(wq, ws, torch.float32).double()

    def layer(x):
        return ops.mxfp4_matmul(*ops.quantize_rows_mxfp4(x, True), wq, ws)

    x = torch.randn(M, K, device="cuda").bfloat16()
    layer(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x)
    for seed in (1, 2):
        x.copy_(torch.randn(M, K, generator=torch.Generator("cuda").manual_seed(seed), device="cuda"))
        graph.replay()
        eager = layer(x)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        xv = ops.dequantize_rows_mxfp4(*ops.quantize_rows_mxfp4(x), torch.float32).double()
        want = (xv @ wv.t()).cpu().numpy()
        lost = R.product_error(xv.cpu().numpy(), wv.cpu().numpy())
        assert (np.abs(out.double().cpu().numpy() - want) <= lost + R.HALF["bfloat16"] * (np.abs(want) + lost)).all()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        other = layer(x)
    st.synchronize()
    assert torch.equal(other, eager)
