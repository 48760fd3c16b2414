"""moe_route_scored against the definition in 64 bits: scores, biases, groups, masks, ties and near ties."""
import numpy as np
import pytest
import torch

from tests import mx_reference as R

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import moe_ascend_opt_b200  # noqa: F401

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def run(logits, bias, K, score, groups=1, topk_groups=1, group_top=1, renorm=True, scale=1.0):
    return torch.ops.nanovllm.moe_route_scored(logits, bias, K, score, groups, topk_groups, group_top, renorm, scale)


def check(logits, bias, K, score, groups=1, topk_groups=1, group_top=1, renorm=True, scale=1.0):
    ids, w = run(logits, bias, K, score, groups, topk_groups, group_top, renorm, scale)
    l = logits.double().cpu().numpy()
    ri, rw = R.route(l, None if bias is None else bias.double().cpu().numpy(), K, score, groups, topk_groups, group_top, renorm, scale)
    assert ids.dtype == torch.int32 and w.dtype == torch.float32
    np.testing.assert_array_equal(ids.cpu().numpy(), ri)
    # fp32 scores: exp within 2 units in the last place and an argument rounded to 2^-24 of |l - max| (softmax), a sum
    # of at most 1024 terms over a tree, a quotient, a product: (16 + |l - max|) 2^-23 of the value covers them
    fin = np.where(np.isfinite(l), l, 0.0)
    d = 16.0 if score == "sigmoid" else 16.0 + np.clip(fin.max(1) - fin.min(1), 0, 104)[:, None]
    err = np.abs(w.double().cpu().numpy() - rw)
    assert (err <= d * 2.0 ** -23 * np.abs(rw) + 1e-37).all(), err.max()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,K", [(1, 1, 1), (1, 8, 8), (3, 33, 5), (257, 128, 8), (64, 250, 16), (5, 1024, 32), (2, 31, 31), (9, 200, 30), (40, 64, 1)])
@pytest.mark.parametrize("biased", [False, True])
def test_plain(T, E, K, score, biased):
    g = torch.Generator("cuda").manual_seed(T + E)
    logits = 2 * torch.randn(T, E, generator=g, device="cuda")
    bias = 0.2 * torch.randn(E, generator=g, device="cuda") if biased else None
    check(logits, bias, K, score)
    check(logits, bias, K, score, renorm=False, scale=1.7)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("E,groups,topk_groups,group_top,K", [(256, 8, 4, 2, 8), (256, 8, 1, 1, 8), (160, 5, 2, 2, 6), (24, 8, 3, 2, 9),
                                                            (32, 32, 7, 1, 7), (96, 2, 2, 2, 10), (60, 4, 3, 1, 8), (1024, 32, 9, 2, 32)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_groups(E, groups, topk_groups, group_top, K, score, dtype):
    g = torch.Generator("cuda").manual_seed(E + groups)
    logits = torch.randn(130, E, generator=g, device="cuda").to(TYPES[dtype])  # 16-bit logits tie often
    for bias in (None, 0.1 * torch.randn(E, generator=g, device="cuda")):
        check(logits, bias, K, score, groups, topk_groups, group_top, True, 2.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,topk_groups,group_top", [(1, 1, 1), (4, 2, 2), (4, 2, 1)])
@pytest.mark.parametrize("biased", [False, True])
def test_masks(score, groups, topk_groups, group_top, biased):
    """Masked experts, rows of which nothing or less than top_k is left, NaN, infinities, the type's lowest value."""
    E, K = 64, 6
    g = torch.Generator("cuda").manual_seed(11)
    logits = torch.randn(40, E, generator=g, device="cuda")
    logits[torch.rand(40, E, generator=g, device="cuda") < 0.5] = -float("inf")
    logits[0] = -float("inf")
    logits[1] = float("nan")
    logits[2, 3:] = -float("inf")  # three experts left
    logits[3, :16] = -float("inf")  # a whole group masked
    logits[4, 5] = float("nan")
    logits[5, 7] = float("inf")
    logits[6, 7:9] = float("inf")
    logits[7] = torch.finfo(torch.float32).min
    logits[8, 10:] = torch.finfo(torch.float32).min
    logits[9] = 0.0
    bias = None
    if biased:
        bias = 0.3 * torch.randn(E, generator=g, device="cuda")
        bias[2], bias[9], bias[33], bias[34] = -float("inf"), float("nan"), float("inf"), -1e30
    check(logits, bias, K, score, groups, topk_groups, group_top)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_near_ties(score):
    """Neighbouring floats and choices whose 32-bit forms coincide keep the order of the definition."""
    E = 128
    base = torch.full((16, E), 0.37, device="cuda")
    up = base.clone()
    for i in range(16):
        up[i, 5 * i + 3] = torch.nextafter(base[i, 0], torch.tensor(1.0, device="cuda"))
        up[i, 5 * i + 9] = torch.nextafter(base[i, 0], torch.tensor(-1.0, device="cuda"))
    check(up, None, 8, score)
    g = torch.Generator("cuda").manual_seed(3)
    logits = 0.5 * torch.randn(256, E, generator=g, device="cuda")
    # biases that bring every choice of row 0 near 0.6: they differ by the rounding of the bias only
    s = torch.sigmoid(logits[0].double()) if score == "sigmoid" else torch.softmax(logits[0].double(), -1)
    check(logits, (0.6 - s).float(), 8, score)
    check(logits[:1].expand(9, E), (0.6 - s).float(), 8, score, 8, 3, 2)


@pytest.mark.parametrize("E,groups", [(128, 1), (256, 8), (512, 4)])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_clusters_of_near_ties(score, biased, E, groups):
    """Pairs and triples of choices that differ by a few units in the last place, at every rank and at the border
    of the top-k and of the groups."""
    g = torch.Generator("cuda").manual_seed(E)
    logits = torch.randn(64, E, generator=g, device="cuda")
    for t in range(64):
        order = torch.randperm(E, generator=g, device="cuda")
        for r in range(2 + t % 3):
            a, b, c = order[3 * r], order[3 * r + 1], order[3 * r + 2]
            logits[t, a] = 2.0 - 0.1 * r
            logits[t, b] = logits[t, a] * (1 + (t % 5 - 2) * 2.0 ** -23)
            if t % 2:
                logits[t, c] = logits[t, a] * (1 - (t % 7 - 3) * 2.0 ** -23)
    bias = torch.zeros(E, device="cuda") if biased else None
    if biased:
        bias += 0.25
    for K in (1, 4, 8):
        check(logits, bias, K, score, groups, max(1, groups // 2), 2 if groups > 1 else 1)
    check(torch.zeros(5, E, device="cuda"), bias, 8, score, groups, max(1, groups // 2), 1)


def test_strides_streams_and_graph():
    g = torch.Generator("cuda").manual_seed(5)
    wide = torch.randn(64, 512, generator=g, device="cuda")
    bias = torch.randn(512, generator=g, device="cuda")
    check(wide[:, ::2], bias[::2], 8, "sigmoid", 8, 4, 2)
    check(wide.t()[:64], None, 4, "softmax")
    check(wide[1:, :250], None, 4, "softmax")
    assert run(wide[:0], None, 4, "softmax")[0].shape == (0, 4)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        check(wide, bias, 8, "sigmoid")
    graph = torch.cuda.CUDAGraph()
    x = wide.clone()
    run(x, bias, 8, "sigmoid", 8, 4, 2)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = run(x, bias, 8, "sigmoid", 8, 4, 2)
    for seed in (1, 2):
        x.copy_(torch.randn(64, 512, generator=torch.Generator("cuda").manual_seed(seed), device="cuda"))
        graph.replay()
        want = run(x, bias, 8, "sigmoid", 8, 4, 2)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_agrees_with_softmax_router():
    """The unbiased softmax case selects and weighs as moe_route does."""
    logits = torch.randn(300, 128, generator=torch.Generator("cuda").manual_seed(8), device="cuda")
    for renorm in (False, True):
        a, b = torch.ops.nanovllm.moe_route(logits, 8, renorm), run(logits, None, 8, "softmax", renorm=renorm)
        assert torch.equal(a[0], b[0])
        torch.testing.assert_close(a[1], b[1], rtol=1e-5, atol=0)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("E,groups,topk_groups,K", [(32, 1, 1, 16), (64, 1, 1, 30), (128, 4, 2, 24), (256, 8, 3, 8), (1024, 1, 1, 30), (60, 4, 2, 20)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_signed_zeros_tie(score, E, groups, topk_groups, K, dtype):
    """-0 and +0 are the same logit: logits times a 0/1 mask, rows of zeros and negatives, and rows whose last choice
    is between one -0 and one +0, tie to the lower index."""
    g = torch.Generator("cuda").manual_seed(E + K)
    logits = torch.randn(80, E, generator=g, device="cuda")
    logits[20:40] = -logits[20:40].abs()
    logits[:40] *= torch.rand(40, E, generator=g, device="cuda") < 0.4
    logits[40:60] = torch.where(torch.rand(20, E, generator=g, device="cuda") < 0.5, 0.0, -0.0)
    per = E // groups
    for t in range(60, 80):
        logits[t] = -1.0 - logits[t].abs()
        mine = torch.cat([gr * per + torch.randperm(per, generator=g, device="cuda") for gr in range(topk_groups)])
        order = mine[torch.randperm(len(mine), generator=g, device="cuda")][:K + 1]
        logits[t, order[:K - 1]] = 1.0 + torch.rand(K - 1, generator=g, device="cuda")
        a, b = sorted(order[K - 1:].tolist())
        logits[t, a], logits[t, b] = -0.0, 0.0
    logits = logits.to(TYPES[dtype])
    assert (logits.eq(0) & logits.signbit()).any()
    check(logits, None, K, score, groups, topk_groups)
    if groups > 1:
        check(logits, None, K, score, groups, topk_groups, 2)
        alone = torch.full((2, E), -1.0, device="cuda").to(TYPES[dtype])  # groups whose best are -0 and +0
        alone[:, ::per] = 0.0
        alone[:, :per * (groups // 2):per] = -0.0
        check(alone, None, min(K, per), score, groups, 1)
    check(logits, torch.zeros(E, device="cuda"), K, score, groups, topk_groups)


@pytest.mark.parametrize("per", [4, 8])
@pytest.mark.parametrize("low,high", [(-5, 3), (-45, -30), (-86, -45), (-110, -86)])
def test_sums_of_small_scores(low, high, per):
    """Groups by the sum of two sigmoid scores, the last that is kept and the first that is not nearly equal in it: far
    below zero a score's relative error grows with its logit."""
    T, G = 2000, 8
    rng = np.random.default_rng(per - low)
    l = low + (high - low) * rng.random((T, 1, 1)) - 3.0 - rng.random((T, G, per))
    l[..., 0] += 3.0
    l[..., 1] += 3.0
    l = l.astype(np.float32).astype(np.float64)
    s = 1 / (1 + np.exp(-l))
    a, b = s[:, 0::2, :2].sum(-1), s[:, 1::2, 0]  # group 2j + 1 takes its second score from the sum of group 2j
    rest = np.where(a > 1.1 * b, a - b, a / 2)
    l[:, 1::2, 1] = np.log(rest / (1 - np.minimum(rest, 0.9)))
    logits = torch.from_numpy(l.astype(np.float32).reshape(T, G * per)).cuda()
    ids, _ = run(logits, None, 3 * per, "sigmoid", G, 3, 2)
    ri, _ = R.route(logits.double().cpu().numpy(), None, 3 * per, "sigmoid", G, 3, 2)
    np.testing.assert_array_equal(ids.cpu().numpy(), ri)


@pytest.mark.parametrize("shift", [0.0, -10.0, -40.0, -70.0, -100.0])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E", [32, 256, 1024])
def test_biases_that_level_small_scores(E, score, shift):
    """Biases that bring pairs of choices to the same value, with scores far below one: all of a sigmoid's, and a
    softmax's where the bias hides the largest logit.  A pair differs by the rounding of its biases."""
    for seed in range(40):
        g = torch.Generator("cuda").manual_seed(seed)
        logits = shift + 0.05 * torch.randn(1, E, generator=g, device="cuda")
        if score == "softmax":
            logits[0, 3] = 1.0
        s = torch.sigmoid(logits[0].double()) if score == "sigmoid" else torch.softmax(logits[0].double(), -1)
        most = s[torch.arange(E, device="cuda") != 3].max()
        level = 3.0 - 0.1 * (torch.randperm(E, generator=g, device="cuda") // 2).clamp(max=20)
        bias = (level * most - s).float()
        bias[3] = -float("inf")
        ids, _ = run(logits, bias, 8, score)
        ri, _ = R.route(logits.double().cpu().numpy(), bias.double().cpu().numpy(), 8, score)
        np.testing.assert_array_equal(ids.cpu().numpy(), ri)
