"""The measured cases of the expert-layer operators: FP8 products grouped by expert with their gradients, products of
4-bit weights with a few vectors, and the row quantiser that feeds the FP8 products.

``run`` computes them in their plain form with elementary torch operations, or, with ``own`` set, through this library's
entry points.  Every listed case says what it stands for in real use."""
import math

import numpy as np
import torch

own = False

F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
MOST8 = {"e4m3": 448.0, "e5m2": 57344.0}
FLOAT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LEAST = 2.0 ** -80          # a row's maximum counts as at least this, so that its scale is a normal number


def listed():
    return [
        # one token of a decode step: the latency of the call
        dict(name="quantize_one_token", op="quantize", tokens=1, top_k=1, k=8192, x="bf16", q="e4m3", gather=False),
        # a prefill's tokens, each sent to two experts, quantised as they are copied into expert order
        dict(name="quantize_to_experts", op="quantize", tokens=8192, top_k=2, k=4096, x="bf16", q="e4m3", gather=True),
        # 16 decoding sequences, two experts each: a few rows an expert, the weights' bytes decide
        dict(name="forward_decode", op="forward", rows=32, slack=0, experts=16, empty=True, k=4096, n=4096, a="e4m3", b="e4m3",
             d="bf16", bias=False, act="none"),
        # a prefill's up-projection with its activation, skewed groups, rows left over at the buffer's end
        dict(name="forward_prefill", op="forward", rows=16384, slack=384, experts=16, empty=False, k=4096, n=8192, a="e4m3",
             b="e4m3", d="bf16", bias=True, act="gelu_tanh"),
        # odd sizes, empty experts, e5m2 gradients, a small training step's input gradient
        dict(name="dgrad_ragged", op="dgrad", rows=1777, slack=33, experts=12, empty=True, k=1040, n=2064, a="e5m2", b="e4m3",
             d="f16"),
        # a training step's input gradient
        dict(name="dgrad_train", op="dgrad", rows=8192, slack=0, experts=8, empty=False, k=4096, n=8192, a="e5m2", b="e4m3",
             d="bf16"),
        # odd sizes, empty experts whose gradient is zero, an FP32 gradient for the optimiser
        dict(name="wgrad_ragged", op="wgrad", rows=1777, slack=33, experts=12, empty=True, k=1040, n=528, a="e5m2", b="e4m3",
             d="f32"),
        # a training step's weight gradient
        dict(name="wgrad_train", op="wgrad", rows=8192, slack=0, experts=8, empty=False, k=4096, n=4096, a="e5m2", b="e4m3",
             d="bf16"),
        # one decoding sequence
        dict(name="w4_one_token", op="w4", m=1, n=8192, k=8192, group=128, x="bf16", zeros=False),
        # eight sequences against a wide up-projection, groups of 64 with zero points
        dict(name="w4_eight_tokens", op="w4", m=8, n=28672, k=8192, group=64, x="f16", zeros=True),
        # one token, four small experts: the smallest call of its kind, an odd number of outputs
        dict(name="w4_experts_one_token", op="w4_experts", tokens=1, top_k=4, experts=64, n=1000, k=2048, group=32, x="bf16",
             zeros=False),
        # 16 sequences, eight experts each: most experts are hit, some several times
        dict(name="w4_experts_batch", op="w4_experts", tokens=16, top_k=8, experts=64, n=2048, k=4096, group=128, x="bf16",
             zeros=True),
    ]


def _spread(rng, low, high, step=1):
    """A multiple of `step` in [low, high], even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high))) / step)) * step))


def draw(rng):
    while True:
        op = rng.choice(["quantize", "forward", "dgrad", "wgrad", "w4", "w4_experts"])
        if op == "quantize":
            c = dict(op=op, tokens=_spread(rng, 1, 8192), top_k=rng.choice([1, 2, 4]), k=_spread(rng, 64, 16384, 16),
                     x=rng.choice(["bf16", "f16"]), q=rng.choice(["e4m3", "e5m2"]), gather=rng.random() < 0.7)
        elif op in ("forward", "dgrad", "wgrad"):
            c = dict(op=op, rows=_spread(rng, 1, 16384), slack=0, experts=_spread(rng, 1, 64), empty=rng.random() < 0.5,
                     k=_spread(rng, 64, 8192, 16), n=_spread(rng, 64, 8192, 1 if op == "forward" and rng.random() < 0.3 else 16),
                     a="e4m3" if op == "forward" else rng.choice(["e5m2", "e4m3"]), b=rng.choice(["e4m3", "e4m3", "e5m2"]),
                     d=rng.choice(["bf16", "f16", "f32"]))
            c["slack"] = rng.choice([0, 0, c["rows"] // 9])
            if op == "forward":
                c.update(bias=rng.random() < 0.5, act=rng.choice(["none", "relu", "gelu_tanh"]))
            if c["experts"] * c["n"] * c["k"] > 2 ** 29 or max(_sizes(c)) * c["experts"] > 40000:
                continue
        elif op == "w4":
            c = dict(op=op, m=_spread(rng, 1, 16), n=_spread(rng, 64, 28672, rng.choice([1, 16])), k=_spread(rng, 128, 8192, 128),
                     group=rng.choice([32, 64, 128]), x=rng.choice(["bf16", "f16"]), zeros=rng.random() < 0.5)
        else:
            c = dict(op=op, tokens=_spread(rng, 1, 32), top_k=rng.choice([1, 2, 4, 8]), experts=_spread(rng, 8, 64),
                     n=_spread(rng, 64, 4096, rng.choice([1, 16])), k=_spread(rng, 128, 4096, 128), group=rng.choice([32, 64, 128]),
                     x=rng.choice(["bf16", "f16"]), zeros=rng.random() < 0.5)
            if c["experts"] * c["n"] * c["k"] > 2 ** 29:
                continue
        if work(c)["flops"] <= (1.05e12 if op == "forward" else 6e11):
            return c


def _sizes(case):
    """Rows of each expert: a skewed split of the rows in use, every fourth expert without rows where the case has empty ones."""
    e, used = case["experts"], case["rows"] - case["slack"]
    w = np.array([0.0 if case["empty"] and i % 4 == 3 else 1.0 / (1.0 + 0.15 * (i % 11)) for i in range(e)])
    cum = np.floor(np.cumsum(w) / w.sum() * used + 0.5).astype(np.int64)
    return [int(v) for v in np.diff(np.concatenate([[0], cum]))]


def _expert_pattern(case):
    """Which experts the tokens take, as numbers that prepare() permutes: a popular few and a tail."""
    t, j = np.meshgrid(np.arange(case["tokens"]), np.arange(case["top_k"]), indexing="ij")
    return (t * t + 3 * t + 5 * j + j * j) % case["experts"]


def _normal(gen, shape, scale, dtype):
    """Normal values of this spread in a 16-bit or 8-bit type, made in pieces so that no large FP32 copy is needed."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat, piece = out.view(-1), 1 << 26
    for at in range(0, flat.numel(), piece):
        v = torch.randn(min(piece, flat.numel() - at), generator=gen, device="cuda") * scale
        if dtype in F8.values():
            v = v.clamp(-448.0, 448.0)
        flat[at:at + piece] = v.to(dtype)
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = np.random.RandomState(seed % (1 << 32))
    s = dict(case)
    uniform = lambda *shape: torch.rand(shape, generator=gen, device="cuda") * 1.5 + 0.5
    if case["op"] == "quantize":
        s["src"] = _normal(gen, (case["tokens"], case["k"]), 1.0, FLOAT[case["x"]])
        s["src"] *= uniform(case["tokens"], 1).to(s["src"].dtype)          # tokens of different size
        s["src"][:, :: max(1, case["k"] // 7)] *= 12                       # and a few strong channels
        rows = case["tokens"] * case["top_k"] if case["gather"] else case["tokens"]
        s["rows"] = torch.from_numpy((host.permutation(rows) // case["top_k"]).astype(np.int32)).cuda() if case["gather"] else None
        s["out"] = torch.empty((rows, case["k"]), dtype=torch.uint8, device="cuda").view(F8[case["q"]])
        s["scale"] = torch.empty(rows, device="cuda")
    elif case["op"] in ("forward", "dgrad", "wgrad"):
        sizes = [_sizes(case)[i] for i in host.permutation(case["experts"])]
        s["sizes"], s["most"] = sizes, max(1, max(sizes))                  # a capacity that the program has set
        s["ends"] = torch.from_numpy(np.cumsum(sizes).astype(np.int32)).cuda()
        e, rows, k, n = case["experts"], case["rows"], case["k"], case["n"]
        wide = {"forward": (k, (e, n, k), n, k), "dgrad": (n, (e, n, k), k, n), "wgrad": (n, (rows, k), k, max(1, rows // e))}[case["op"]]
        s["A"] = _normal(gen, (rows, wide[0]), 48.0, F8[case["a"]])
        s["B"] = _normal(gen, wide[1], 48.0, F8[case["b"]])
        unit = 1.0 / 48.0 / math.sqrt(wide[3])
        if case["op"] == "wgrad":
            s["a_scale"], s["b_scale"] = uniform(1) / 48.0, uniform(1) * unit
            s["D"] = torch.zeros((e, n, k), dtype=FLOAT[case["d"]], device="cuda")
        else:
            s["a_row"], s["b_row"] = uniform(rows) / 48.0, uniform(e, wide[2]) * unit
            s["bias_row"] = _normal(gen, (e, wide[2]), 0.5, torch.bfloat16) if case.get("bias") else None
            s["D"] = torch.zeros((rows, wide[2]), dtype=FLOAT[case["d"]], device="cuda")
        s["new"] = torch.zeros_like(s["D"])
    else:
        e = (case["experts"],) if case["op"] == "w4_experts" else ()
        n, k, groups = case["n"], case["k"], case["k"] // case["group"]
        s["codes"] = torch.randint(0, 256, (*e, n, k // 2), generator=gen, device="cuda", dtype=torch.uint8)
        s["scales"] = (uniform(*e, n, groups) / (4.0 * math.sqrt(k))).to(FLOAT[case["x"]])
        s["zero"] = torch.randint(6, 11, (*e, n, groups), generator=gen, device="cuda", dtype=torch.uint8) if case["zeros"] else None
        s["vec"] = _normal(gen, (case["tokens"] if e else case["m"], k), 1.0, FLOAT[case["x"]])
        if e:
            ids = host.permutation(case["experts"])[_expert_pattern(case)].reshape(-1).astype(np.int32)
            s["expert"] = torch.from_numpy(ids).cuda()
        s["y"] = torch.zeros((len(ids) if e else case["m"], n), dtype=FLOAT[case["x"]], device="cuda")
    return s


_library = None


def _own(s):
    global _library
    if _library is None:
        from __graft_entry__ import load_package
        _library = load_package().gemm
    g = _library
    if s["op"] == "quantize":
        g.quantize_rows(s["src"], s["out"], s["scale"], rows=s["rows"])
        return {"q": s["out"], "scale": s["scale"]}
    if s["op"] == "forward":
        return g.gemm_grouped(s["A"], s["B"], s["new"], s["ends"], a_row_scale=s["a_row"], b_row_scale=s["b_row"], bias=s["bias_row"],
                              activation=s["act"])
    if s["op"] == "dgrad":
        return g.gemm_grouped_dgrad(s["A"], s["B"], s["new"], s["ends"], a_row_scale=s["a_row"], b_row_scale=s["b_row"])
    if s["op"] == "wgrad":
        return g.gemm_grouped_wgrad(s["A"], s["B"], s["new"], s["ends"], a_scale=s["a_scale"], b_scale=s["b_scale"])
    if s["op"] == "w4":
        return g.gemv_w4(s["codes"], s["scales"], s["vec"], s["y"], zeros=s["zero"])
    return g.gemv_w4_experts(s["codes"], s["scales"], s["vec"], s["y"], s["expert"], zeros=s["zero"])


def run(s):
    if own:
        return _own(s)
    if s["op"] == "quantize":
        return _plain_quantize(s)
    if s["op"] in ("w4", "w4_experts"):
        return _plain_w4(s)
    return _plain_products(s)


def _plain_quantize(s):
    x = s["src"].double()
    if s["rows"] is not None:
        x = x[s["rows"].long()]
    most = x.abs().amax(dim=1).clamp_min(LEAST)
    top = MOST8[s["q"]]
    return {"q": (x * top / most[:, None]).clamp(-top, top).to(F8[s["q"]]), "scale": (most / top).float()}


def _in_groups(x, ends, most):
    """Rows by expert in a padded block [experts][most][...], zeros behind an expert's last row."""
    start = torch.cat([ends.new_zeros(1), ends[:-1]])
    at = start[:, None] + torch.arange(most, device=x.device)
    return torch.where((at < ends[:, None])[..., None], x[at.clamp(max=x.shape[0] - 1)].float(), 0.0)


def _plain_products(s):
    ends, most = s["ends"].long(), s["most"]
    a = _in_groups(s["A"], ends, most)
    if s["op"] == "wgrad":
        return (torch.bmm(a.transpose(1, 2), _in_groups(s["B"], ends, most)) * (s["a_scale"] * s["b_scale"])).to(s["D"].dtype)
    b = s["B"].float()
    t = torch.bmm(a, b.transpose(1, 2) if s["op"] == "forward" else b)
    t = t * s["b_row"][:, None, :]
    row = torch.arange(s["rows"], device=ends.device)
    of = torch.searchsorted(ends, row, right=True).clamp(max=s["experts"] - 1)
    start = torch.cat([ends.new_zeros(1), ends[:-1]])
    t = t[of, (row - start[of]).clamp(0, most - 1)] * s["a_row"][:, None]
    if s["bias_row"] is not None:
        t = t + s["bias_row"].float()[of]
    if s.get("act") == "relu":
        t = t.clamp_min(0.0)
    elif s.get("act") == "gelu_tanh":
        t = 0.5 * t * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (t + 0.044715 * t * t * t)))
    return torch.where((row < ends[-1])[:, None], t.to(s["D"].dtype), s["D"])


def _weights(s, dtype):
    """The matrix that the 4-bit codes stand for."""
    c = torch.stack([s["codes"] & 15, s["codes"] >> 4], dim=-1).reshape(*s["scales"].shape, s["group"]).to(dtype)
    z = 8.0 if s["zero"] is None else s["zero"].to(dtype)[..., None]
    return ((c - z) * s["scales"].to(dtype)[..., None]).flatten(-2)


def _plain_w4(s):
    x = s["vec"].float()
    if s["op"] == "w4":
        return (x @ _weights(s, torch.float32).transpose(0, 1)).to(s["vec"].dtype)
    expert = s["expert"].long()
    token = torch.arange(expert.shape[0], device=x.device) // s["top_k"]
    if expert.shape[0] <= s["experts"]:                                    # few rows: only their experts' matrices
        of_rows = {**s, **{key: s[key][expert] for key in ("codes", "scales", "zero") if s[key] is not None}}
        return torch.bmm(_weights(of_rows, torch.float32), x[token][..., None])[..., 0].to(s["vec"].dtype)
    y = torch.matmul(x, _weights(s, torch.float32).transpose(1, 2))        # every expert's answer to every token
    return y[expert, token].to(s["vec"].dtype)


def work(case):
    if case["op"] == "quantize":
        rows = case["tokens"] * (case["top_k"] if case["gather"] else 1)
        return {"bytes": case["k"] * (2 * case["tokens"] + rows) + rows * (8 if case["gather"] else 4), "flops": 4 * rows * case["k"]}
    if case["op"] in ("w4", "w4_experts"):
        n, k, groups = case["n"], case["k"], case["k"] // case["group"]
        if case["op"] == "w4":
            mats, xs, ys = 1, case["m"], case["m"]
        else:
            mats, xs, ys = len(np.unique(_expert_pattern(case))), case["tokens"], case["tokens"] * case["top_k"]
        return {"bytes": mats * n * (k // 2 + groups * (3 if case["zeros"] else 2)) + 2 * xs * k + 2 * ys * n, "flops": 2 * ys * n * k}
    sizes, n, k = _sizes(case), case["n"], case["k"]
    used, active, size = sum(sizes), sum(v > 0 for v in sizes), {"f32": 4, "bf16": 2, "f16": 2}[case["d"]]
    if case["op"] == "wgrad":
        got = used * (n + k) + case["experts"] * n * k * size
    else:
        wide, out = (k, n) if case["op"] == "forward" else (n, k)
        got = used * wide + active * n * k + used * out * size + 4 * used + active * out * (6 if case.get("bias") else 4)
    return {"bytes": got, "flops": 2 * used * n * k}


def _nearest8(v, kind):
    """The nearest 8-bit float, ties to the even one, by the spacing of the numbers at this size."""
    fraction, lowest = (3, -6) if kind == "e4m3" else (2, -14)
    _, up = torch.frexp(v)
    step = torch.exp2((up - 1).clamp_min(lowest).double() - fraction)
    return (torch.round(v / step) * step).clamp(-MOST8[kind], MOST8[kind])


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        x = s["src"].double()
        if case["gather"]:
            x = x.index_select(0, s["rows"].long())
        largest = torch.maximum(x.max(dim=1).values, -x.min(dim=1).values).clamp_min(LEAST)
        return {"q": _nearest8(x * MOST8[case["q"]] / largest.unsqueeze(1), case["q"]), "scale": largest / MOST8[case["q"]]}
    if case["op"] == "w4":
        return s["vec"].double() @ _weights(s, torch.float64).mT
    if case["op"] == "w4_experts":
        y, token = torch.empty(s["y"].shape, dtype=torch.float64, device="cuda"), 0
        for r, e in enumerate(s["expert"].tolist()):
            of_one = {**s, "codes": s["codes"][e], "scales": s["scales"][e], "zero": None if s["zero"] is None else s["zero"][e]}
            y[r] = _weights(of_one, torch.float64) @ s["vec"][r // case["top_k"]].double()
        return y
    out, at = s["D"].double(), 0
    for e, size in enumerate(s["sizes"]):
        a = s["A"][at:at + size].double()
        if case["op"] == "wgrad":
            out[e] = (a.mT @ s["B"][at:at + size].double()) * (s["a_scale"].double() * s["b_scale"].double())
        elif size:
            b = s["B"][e].double()
            t = (a @ (b.mT if case["op"] == "forward" else b)) * s["a_row"][at:at + size, None].double() * s["b_row"][e].double()
            if s["bias_row"] is not None:
                t = t + s["bias_row"][e].double()
            if case.get("act") == "relu":
                t = torch.relu(t)
            elif case.get("act") == "gelu_tanh":
                t = t / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (t + 0.044715 * t ** 3)))
            out[at:at + size] = t
        at += size
    return out
