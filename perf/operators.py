"""What the routing and MXFP4 operators are measured on.

Four operators of one path, the routed expert layer with 4-bit floating-point weights:

* ``route``     routing to experts from given logits: softmax or sigmoid scores, a balance bias, expert
                groups, top-k, renormalised and scaled weights;
* ``quantize``  rows to MXFP4 (blocks of 32 along a row: 4-bit e2m1 elements, one e8m0 scale) and back;
* ``product``   y = a b^T of two MXFP4 matrices, and the linear layer that quantises its input first;
* ``experts``   the expert layer on MXFP4 weights: quantise, gate_up, SiLU * up, quantise, down, weighted sum.

``own`` False computes them with elementary torch operations, True with the framework's calls.
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # one decode token through the router of a 128-expert layer: latency
        {"name": "route-decode", "op": "route", "T": 1, "E": 128, "K": 8, "score": "softmax", "bias": False, "groups": 1,
         "topk_groups": 1, "group_top": 1, "renorm": True, "scale": 1.0, "dtype": "float32", "padded": 0},
        # a ragged batch with padding rows, sigmoid scores, balance bias, 8 groups of 32 experts
        {"name": "route-grouped", "op": "route", "T": 257, "E": 256, "K": 8, "score": "sigmoid", "bias": True, "groups": 8,
         "topk_groups": 4, "group_top": 2, "renorm": True, "scale": 2.5, "dtype": "float32", "padded": 31},
        # a prefill batch, bf16 logits
        {"name": "route-prefill", "op": "route", "T": 16384, "E": 256, "K": 8, "score": "sigmoid", "bias": True, "groups": 8,
         "topk_groups": 4, "group_top": 2, "renorm": True, "scale": 2.5, "dtype": "bfloat16", "padded": 0},
        # activations of a decode batch
        {"name": "quantize-decode", "op": "quantize", "rows": 8, "cols": 2048, "dtype": "bfloat16"},
        # one expert group's weights at load, an odd number of rows
        {"name": "quantize-weights", "op": "quantize", "rows": 24577, "cols": 768, "dtype": "float32"},
        # a linear layer on one decode token
        {"name": "linear-decode", "op": "product", "M": 1, "N": 4096, "K": 2048, "quantised": False, "dtype": "bfloat16"},
        # a ragged prefill chunk against a gate_up matrix
        {"name": "product-chunk", "op": "product", "M": 333, "N": 1536, "K": 2048, "quantised": True, "dtype": "bfloat16"},
        # a large dense layer
        {"name": "product-large", "op": "product", "M": 8192, "N": 4096, "K": 4096, "quantised": True, "dtype": "bfloat16"},
        # one decode token through 8 of 128 experts
        {"name": "experts-decode", "op": "experts", "T": 1, "E": 128, "K": 8, "H": 2048, "I": 768, "skew": 0.0, "skip": 0.0,
         "dtype": "bfloat16"},
        # a decode batch with hot experts
        {"name": "experts-batch", "op": "experts", "T": 8, "E": 128, "K": 8, "H": 2048, "I": 768, "skew": 1.2, "skip": 0.0,
         "dtype": "bfloat16"},
        # one rank's share of a ragged batch: half the pairs belong to other ranks
        {"name": "experts-ragged", "op": "experts", "T": 201, "E": 64, "K": 8, "H": 2048, "I": 768, "skew": 0.0, "skip": 0.5,
         "dtype": "float16"},
        # a prefill step
        {"name": "experts-prefill", "op": "experts", "T": 4096, "E": 128, "K": 8, "H": 2048, "I": 768, "skew": 0.0, "skip": 0.0,
         "dtype": "bfloat16"},
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "quantize", "product", "experts"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        per = rng.randint(4, 256 // groups)
        topk_groups = rng.randint(1, groups)
        T = _spread(rng, 1, 16384)
        return {"op": op, "T": T, "E": groups * per, "K": rng.randint(1, min(16, topk_groups * per)),
                "score": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.5, "groups": groups,
                "topk_groups": topk_groups, "group_top": rng.choice([1, 2]), "renorm": rng.random() < 0.7,
                "scale": rng.choice([1.0, 2.5]), "dtype": rng.choice(sorted(TYPES)), "padded": rng.choice([0, T // 8])}
    if op == "quantize":
        cols = 32 * _spread(rng, 1, 128)
        return {"op": op, "rows": _spread(rng, 1, max(1, (24577 * 768) // cols)), "cols": cols, "dtype": rng.choice(sorted(TYPES))}
    if op == "product":
        N, K = _spread(rng, 16, 4096), 32 * _spread(rng, 2, 128)
        return {"op": op, "M": _spread(rng, 1, 8192), "N": N, "K": K, "quantised": rng.random() < 0.5,
                "dtype": rng.choice(sorted(TYPES))}
    E = rng.choice([8, 16, 40, 64, 128])
    return {"op": op, "T": _spread(rng, 1, 4096), "E": E, "K": rng.randint(1, min(8, E)), "H": 32 * rng.randint(8, 64),
            "I": 32 * rng.randint(2, 24), "skew": rng.choice([0.0, 0.0, 1.2]), "skip": rng.choice([0.0, 0.0, 0.5]),
            "dtype": rng.choice(["bfloat16", "float16"])}


# ------------------------------------------------------------------ MXFP4, plain
def _encode(x):
    """Codes (0..15, one a byte) and e8m0 scale bytes of the blocks of 32 along the last axis of an fp32 tensor."""
    b = x.float().unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1)
    exponent = (amax.view(torch.int32) >> 23).clamp(max=255)  # biased exponent of the block's largest magnitude
    code = (exponent - 2).clamp(min=0)
    code = torch.where(exponent == 255, torch.full_like(code, 255), code)  # infinity or NaN in the block
    m = b.abs() * ((254 - code).clamp(min=1) << 23).view(torch.float32).unsqueeze(-1)  # times 2^(127 - code)
    # the midpoints of 0 .5 1 1.5 2 3 4 6: a tie goes to the even code
    q = ((m > 0.25).to(torch.uint8) + (m >= 0.75).to(torch.uint8) + (m > 1.25).to(torch.uint8) + (m >= 1.75).to(torch.uint8)
         + (m > 2.5).to(torch.uint8) + (m >= 3.5).to(torch.uint8) + (m > 5.0).to(torch.uint8))
    return (q | (torch.signbit(b).to(torch.uint8) << 3)).flatten(-2), code.to(torch.uint8)


def _pack(codes):
    """Two codes a byte, the even element in the low half."""
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _decode(codes, scales):
    """fp32 values of codes (one a byte) with the e8m0 scales of their blocks."""
    half = (codes & 1).float()
    e = ((codes >> 1) & 3).int()
    m = torch.where(e == 0, 0.5 * half, (1.0 + 0.5 * half) * ((e + 126) << 23).view(torch.float32))
    m = torch.where((codes & 8) != 0, -m, m)
    power = torch.where(scales == 0, 1 << 22, scales.int() << 23).view(torch.float32)  # 2^(scale - 127), the least is subnormal
    power = torch.where(scales == 255, math.nan, power)
    return (m.unflatten(-1, (-1, 32)) * power.unsqueeze(-1)).flatten(-2)


def _unpack(q):
    return torch.stack((q & 15, q >> 4), -1).flatten(-2)


def _tile(scales):
    """[rows, blocks] -> [ceil(rows / 128), ceil(blocks / 4), 512]: byte 16 (r % 32) + 4 (r / 32) + k of a 128 x 4 tile."""
    rows, blocks = scales.shape
    s = torch.nn.functional.pad(scales, (0, -blocks % 4, 0, -rows % 128))
    return s.view(s.shape[0] // 128, 4, 32, s.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).reshape(s.shape[0] // 128, s.shape[1] // 4, 512).contiguous()


def _untile(tiles, rows, blocks):
    rb, kb = tiles.shape[0], tiles.shape[1]
    return tiles.view(rb, kb, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rb * 128, kb * 4)[:rows, :blocks]


def _rounded(x):
    """The values that an fp32 tensor has after MXFP4."""
    return _decode(*_encode(x))


# ------------------------------------------------------------------ inputs
def _activations(g, rows, cols, dtype):
    """Hidden states: normal, with some channels that are larger than the others."""
    x = torch.randn(rows, cols, generator=g, device=DEVICE)
    return (x * torch.exp(0.5 * torch.randn(cols, generator=g, device=DEVICE))).to(dtype)


def _ids(g, case):
    """Top-k experts of normal logits, by a softmax over the selected; skew makes the low ids hot, skip gives pairs away."""
    T, E, K = case["T"], case["E"], case["K"]
    logits = torch.randn(T, E, generator=g, device=DEVICE) - case["skew"] * torch.log(torch.arange(1, E + 1, device=DEVICE))
    v, ids = logits.topk(K, dim=-1)
    ids = torch.where(torch.rand(T, K, generator=g, device=DEVICE) < case["skip"], torch.full_like(ids, -1), ids)
    return ids.int(), torch.softmax(v, -1)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    s = {"case": case}
    if case["op"] == "route":
        T, E = case["T"], case["E"]
        logits = 1.5 * torch.randn(T, E, generator=g, device=DEVICE)
        logits[T - case["padded"]:] = -math.inf  # padding rows
        s["logits"] = logits.to(TYPES[case["dtype"]])
        s["bias"] = 0.1 * torch.randn(E, generator=g, device=DEVICE) if case["bias"] else None
    elif case["op"] == "quantize":
        s["x"] = _activations(g, case["rows"], case["cols"], TYPES[case["dtype"]])
    elif case["op"] == "product":
        M, N, K = case["M"], case["N"], case["K"]
        x = _activations(g, M, K, torch.bfloat16)
        codes, scales = _encode(0.02 * torch.randn(N, K, generator=g, device=DEVICE))
        s["b"], s["b_scales"] = _pack(codes), _tile(scales)
        if case["quantised"]:
            codes, scales = _encode(x)
            s["a"], s["a_scales"] = _pack(codes), _tile(scales)
        else:
            s["x"] = x
    else:
        E, H, I = case["E"], case["H"], case["I"]
        s["x"] = _activations(g, case["T"], H, TYPES[case["dtype"]])
        s["ids"], s["weights"] = _ids(g, case)
        codes, s["w13_scales"] = _encode(0.02 * torch.randn(E, 2 * I, H, generator=g, device=DEVICE))
        s["w13"] = _pack(codes)
        codes, s["w2_scales"] = _encode(0.02 * torch.randn(E, H, I, generator=g, device=DEVICE))
        s["w2"] = _pack(codes)
        del codes
        # the most pairs that an expert has: the plain form's batch
        s["most"] = int(torch.bincount(s["ids"].flatten().clamp(min=-1).long() + 1, minlength=E + 1)[1:].max())
        if own:
            import moe_ascend_opt_b200  # noqa: F401
            s["handle"] = torch.classes.nanovllm.MoEInfer(E, H, I, 3)
            s["handle"].store_mxfp4(s["w13"], s["w13_scales"], s["w2"], s["w2_scales"])
    if own:
        import moe_ascend_opt_b200  # noqa: F401, F811
    return s


# ------------------------------------------------------------------ the plain forms
def _route(logits, bias, K, score, groups, topk_groups, group_top, renorm, scale):
    T, E = logits.shape
    l = logits.double()
    live = l > -math.inf
    l = torch.where(live, l, torch.zeros_like(l))
    if score == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-l))
    else:
        top = torch.where(live, l, torch.full_like(l, -math.inf)).amax(-1, keepdim=True).clamp(min=-1e300)
        e = torch.where(live, torch.exp(torch.where(live, l - top, torch.zeros_like(l))), torch.zeros_like(l))
        s = e / e.sum(-1, keepdim=True).clamp(min=1e-300)
    s = torch.where(live, s, torch.zeros_like(s))
    # without a bias the scores have the logits' order
    key = torch.where(live, l if bias is None else s + bias.double(), torch.full_like(l, -math.inf))
    if groups > 1:
        part = (key if group_top == 1 else torch.where(live, s if bias is None else key, torch.full_like(l, -math.inf))).view(T, groups, E // groups)
        best = part.topk(min(group_top, E // groups), dim=-1).values
        total = torch.where(best > -math.inf, best, torch.zeros_like(best)).sum(-1)
        total = torch.where(best[..., 0] > -math.inf, total, torch.full_like(total, -math.inf))
        order = torch.sort(total, dim=-1, descending=True, stable=True).indices[:, :topk_groups]
        keep = torch.zeros(T, groups, dtype=torch.bool, device=l.device).scatter_(1, order, True)
        key = torch.where(keep.repeat_interleave(E // groups, 1), key, torch.full_like(key, -math.inf))
    picked = torch.sort(key, dim=-1, descending=True, stable=True)
    ids = picked.indices[:, :K]
    found = picked.values[:, :K] > -math.inf
    w = torch.where(found, s.gather(1, ids), torch.zeros((), dtype=torch.float64, device=l.device))
    if renorm:
        w = w / (w.sum(-1, keepdim=True) + 1e-20)
    return torch.where(found, ids, torch.full_like(ids, -1)).int(), (w * scale).float()


def _experts(s):
    case = s["case"]
    T, E, K, H, I = (case[k] for k in "TEKHI")
    x, ids = _rounded(s["x"]), s["ids"].flatten().long()
    rows = torch.arange(T, device=x.device).repeat_interleave(K)
    held = (ids >= 0) & (ids < E)
    if T * K <= E:  # each pair with its own expert's weights
        pick = ids.clamp(0, E - 1)
        a = x[rows].unsqueeze(1)
    else:  # a batch of the experts, padded to the most pairs that one has
        pick = torch.arange(E, device=x.device)
        one = torch.nn.functional.one_hot(torch.where(held, ids, torch.full_like(ids, E)), E + 1)
        place = (one.cumsum(0) * one).sum(-1) - 1
        slot = torch.where(held, ids * s["most"] + place, torch.full_like(ids, E * s["most"]))
        a = torch.zeros(E * s["most"] + 1, H, device=x.device).index_copy_(0, slot, x[rows])[:-1].view(E, s["most"], H)
    w13 = _decode(_unpack(s["w13"][pick]), s["w13_scales"][pick])
    gu = torch.bmm(a, w13.transpose(1, 2))
    del w13
    h = _rounded(gu[..., :I] / (1.0 + torch.exp(-gu[..., :I])) * gu[..., I:])
    p = torch.bmm(h, _decode(_unpack(s["w2"][pick]), s["w2_scales"][pick]).transpose(1, 2))
    p = p.reshape(-1, H) if T * K <= E else p.reshape(-1, H)[slot.clamp(max=E * s["most"] - 1)]
    p = torch.where(held.unsqueeze(1), p, torch.zeros_like(p)).view(T, K, H)
    return (p * s["weights"].unsqueeze(-1)).sum(1).to(s["x"].dtype)


def run(s):
    case = s["case"]
    if case["op"] == "route":
        if own:
            return torch.ops.nanovllm.moe_route_scored(s["logits"], s["bias"], case["K"], case["score"], case["groups"],
                                                       case["topk_groups"], case["group_top"], case["renorm"], case["scale"])
        return _route(s["logits"], s["bias"], case["K"], case["score"], case["groups"], case["topk_groups"],
                      case["group_top"], case["renorm"], case["scale"])
    if case["op"] == "quantize":
        if own:
            q, scales = torch.ops.nanovllm.quantize_rows_mxfp4(s["x"])
            return torch.ops.nanovllm.dequantize_rows_mxfp4(q, scales)
        codes, scales = _encode(s["x"])
        q = _pack(codes)
        return _decode(_unpack(q), scales).bfloat16()
    if case["op"] == "product":
        out = TYPES[case["dtype"]]
        if own:
            a, a_scales = (s["a"], s["a_scales"]) if case["quantised"] else torch.ops.nanovllm.quantize_rows_mxfp4(s["x"], True)
            return torch.ops.nanovllm.mxfp4_matmul(a, a_scales, s["b"], s["b_scales"], out)
        blocks = case["K"] // 32
        a = _decode(_unpack(s["a"]), _untile(s["a_scales"], case["M"], blocks)) if case["quantised"] else _rounded(s["x"])
        return (a @ _decode(_unpack(s["b"]), _untile(s["b_scales"], case["N"], blocks)).t()).to(out)
    if own:
        return torch.ops.nanovllm.moe_forward(s["x"], s["ids"], s["weights"], s["handle"])
    return _experts(s)


def work(case):
    size = TYPES[case["dtype"]].itemsize
    mx = 17.0 / 32.0  # bytes of an MXFP4 element with its share of the scale
    if case["op"] == "route":
        T, E, K = case["T"], case["E"], case["K"]
        return {"bytes": T * E * size + (4 * E if case["bias"] else 0) + 8 * T * K, "flops": 5 * T * E}
    if case["op"] == "quantize":  # rows in, codes and scales out and in again, bf16 values out
        n = case["rows"] * case["cols"]
        return {"bytes": n * (size + 2 * mx + 2), "flops": 4 * n}
    if case["op"] == "product":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": N * K * mx + M * K * (mx if case["quantised"] else 2) + M * N * size, "flops": 2 * M * N * K}
    T, E, K, H, I = (case[k] for k in "TEKHI")
    pairs = T * K * (1 - case["skip"])
    active = E * (1 - (1 - K * (1 - case["skip"]) / E) ** T)  # experts that a uniform routing reaches
    return {"bytes": active * 3 * H * I * mx + 2 * T * H * size + 8 * T * K, "flops": 6 * pairs * H * I}


# ------------------------------------------------------------------ the definition in 64 bits
def _mx64(x):
    """Values after MXFP4, by the grid's step at each magnitude: .5 below 2, 1 below 4, 2 up to 6."""
    b = x.double().unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    shared = torch.where(amax > 0, torch.frexp(amax).exponent - 1 - 2, torch.full_like(amax, -127, dtype=torch.int32)).clamp(min=-127)
    unit = torch.pow(2.0, shared.double())
    v = (b / unit).clamp(-6.0, 6.0)
    step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0)).double()
    return (torch.round(v / step) * step * unit).flatten(-2)


def _values64(packed, scales):
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=packed.device)
    grid = torch.cat((grid, -grid))
    v = torch.stack((grid[(packed & 15).long()], grid[(packed >> 4).long()]), -1).flatten(-2)
    return v * torch.pow(2.0, scales.double() - 127).repeat_interleave(32, -1)


def _scales64(tiles, rows, blocks):
    r = torch.arange(rows, device=tiles.device).unsqueeze(1)
    k = torch.arange(blocks, device=tiles.device).unsqueeze(0)
    return tiles[r // 128, k // 4, 16 * (r % 32) + 4 * (r % 128 // 32) + k % 4]


def _route64(s):
    import numpy as np
    case = s["case"]
    l = s["logits"].double().cpu().numpy()
    T, E = l.shape
    live = np.isfinite(l)
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        if case["score"] == "sigmoid":
            p = np.where(live, 1 / (1 + np.exp(-np.where(live, l, 0))), 0)
        else:
            e = np.where(live, np.exp(l - l.max(1, keepdims=True, initial=-1e300, where=live)), 0)
            p = e / np.maximum(e.sum(1, keepdims=True), 1e-300)
    c = p if s["bias"] is None else p + s["bias"].double().cpu().numpy()
    order_key = l if s["bias"] is None else c
    ids = np.full((T, case["K"]), -1, np.int32)
    w = np.zeros((T, case["K"]))
    G, per = case["groups"], E // case["groups"]
    for t in range(T):
        mine = np.flatnonzero(live[t])
        if G > 1 and len(mine):
            of = order_key[t] if case["group_top"] == 1 else c[t]
            total = [sum(sorted(of[mine[mine // per == g]])[::-1][: case["group_top"]]) if (mine // per == g).any() else -np.inf for g in range(G)]
            good = sorted(range(G), key=lambda g: (-total[g], g))[: case["topk_groups"]]
            mine = mine[np.isin(mine // per, good)]
        take = mine[np.lexsort((mine, -order_key[t, mine]))][: case["K"]]
        ids[t, : len(take)] = take
        w[t, : len(take)] = p[t, take]
    if case["renorm"]:
        w = w / (w.sum(1, keepdims=True) + 1e-20)
    return torch.from_numpy(ids), torch.from_numpy(w * case["scale"])


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        return _route64(s)
    if case["op"] == "quantize":
        return _mx64(s["x"])
    if case["op"] == "product":
        blocks = case["K"] // 32
        a = _values64(s["a"], _scales64(s["a_scales"], case["M"], blocks)) if case["quantised"] else _mx64(s["x"])
        return a @ _values64(s["b"], _scales64(s["b_scales"], case["N"], blocks)).t()
    x, y = _mx64(s["x"]), torch.zeros(case["T"], case["H"], dtype=torch.float64, device=DEVICE)
    for e in range(case["E"]):
        t, k = (s["ids"] == e).nonzero(as_tuple=True)
        if len(t):
            gate, up = (x[t] @ _values64(s["w13"][e], s["w13_scales"][e]).t()).chunk(2, -1)
            h = _mx64(gate * torch.sigmoid(gate) * up)
            y.index_add_(0, t, (h @ _values64(s["w2"][e], s["w2_scales"][e]).t()) * s["weights"][t, k].double().unsqueeze(1))
    return y
