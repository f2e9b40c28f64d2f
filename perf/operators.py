"""The quantised linear path, operator by operator: rows and weights in 8 bits with scales, weights in 4 bits with group scales.

Five operators, each beside its bf16 sibling in ``llm_steadyinfer_b200.csrc.ops``:

* ``norm``: residual add, RMS norm, rows out in e4m3 with a scale a row (``add_rmsnorm_q8``);
* ``swiglu``: the gated activation, rows out in e4m3 with a scale a row (``swiglu_q8``);
* ``quantize``: rows to e4m3 with a scale a row (``quantize_q8``);
* ``gemm_q8``: product of such rows with weights in e4m3 with a scale an output channel;
* ``gemm_w4``: product of bf16 rows with 4-bit weights, a scale (and a zero point) a group of input channels.

Sizes are those of the shapes the package's configurations and benchmark sections name (widths 1,024, 2,048 and 4,096 with their
feed-forwards), at the row counts of decode steps, decode batches and prompt portions.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
EPS = 1e-5
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
LEAST = 2.0 ** -100               # the least maximum that a row's scale is made of
# an int32 word holds eight entries; entry i of the eight lies at bit SHIFTS[i]: neighbours (2i, 2i + 1) sixteen bits apart
SHIFTS = (0, 16, 4, 20, 8, 24, 12, 28)


def listed():
    return [
        # a decode step of eight requests: the norm before a layer's products
        {"name": "norm 8x4096", "op": "norm", "rows": 8, "width": 4096, "deltas": 1, "dtype": "bf16"},
        # a prompt portion; two sublayers' results join the stream at once
        {"name": "norm 2048x4096 two", "op": "norm", "rows": 2048, "width": 4096, "deltas": 2, "dtype": "bf16"},
        # one request's decode step, gates and ups interleaved as the package stacks them
        {"name": "swiglu 1x8192", "op": "swiglu", "rows": 1, "inter": 8192, "group": 8, "dtype": "bf16"},
        # a prompt portion
        {"name": "swiglu 2048x14336", "op": "swiglu", "rows": 2048, "inter": 14336, "group": 8, "dtype": "bf16"},
        # the heads' results of an odd decode batch, rows of a wider buffer
        {"name": "quantize 61x4096", "op": "quantize", "rows": 61, "width": 4096, "stride": 6144, "dtype": "bf16"},
        # a weight at load: its rows become output channels with a scale each
        {"name": "quantize 4096x14336", "op": "quantize", "rows": 4096, "width": 14336, "stride": 14336, "dtype": "bf16"},
        # decode: the stacked gate/up projection of eight requests
        {"name": "q8 8x28672x4096", "op": "gemm_q8", "rows": 8, "n": 28672, "k": 4096, "out": "bf16"},
        # a large decode batch: the down projection
        {"name": "q8 61x4096x14336", "op": "gemm_q8", "rows": 61, "n": 4096, "k": 14336, "out": "bf16"},
        # a prompt portion
        {"name": "q8 2048x28672x4096", "op": "gemm_q8", "rows": 2048, "n": 28672, "k": 4096, "out": "bf16"},
        # one request's decode step: the output projection
        {"name": "w4 1x4096x4096", "op": "gemm_w4", "rows": 1, "n": 4096, "k": 4096, "group": 128, "zeros": False, "out": "bf16"},
        # decode: the stacked gate/up projection of eight requests, with zero points
        {"name": "w4 8x28672x4096 zeros", "op": "gemm_w4", "rows": 8, "n": 28672, "k": 4096, "group": 128, "zeros": True, "out": "bf16"},
        # an odd prompt portion through the down projection, groups of 64
        {"name": "w4 937x4096x14336", "op": "gemm_w4", "rows": 937, "n": 4096, "k": 14336, "group": 64, "zeros": False, "out": "bf16"},
    ]


def _spread(rng, low, high, multiple=1):
    """A whole number between the two, even over its logarithm, rounded to a multiple."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(multiple, int(round(v / multiple)) * multiple)


def draw(rng):
    op = rng.choice(["norm", "swiglu", "quantize", "gemm_q8", "gemm_q8", "gemm_w4", "gemm_w4"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    if op == "norm":
        return {"op": op, "rows": _spread(rng, 1, 2048), "width": _spread(rng, 96, 4096, rng.choice([1, 8])), "deltas": rng.choice([0, 1, 1, 2]),
                "dtype": dtype}
    if op == "swiglu":
        group = rng.choice([0, 8])
        return {"op": op, "rows": _spread(rng, 1, 2048), "inter": _spread(rng, 96, 14336, 8 if group else 1), "group": group, "dtype": dtype}
    if op == "quantize":
        width = _spread(rng, 64, 14336, rng.choice([1, 8]))
        return {"op": op, "rows": _spread(rng, 1, 4096), "width": width, "stride": width + rng.choice([0, 0, 8, 1024]), "dtype": dtype}
    n, k = rng.choice([(2048, 2048), (4096, 4096), (6144, 4096), (28672, 4096), (4096, 14336), (16384, 2048), (2048, 8192), (11264, 2048),
                       (2048, 5632), (1024, 2816), (_spread(rng, 64, 8192), _spread(rng, 64, 8192, 8))])
    rows = _spread(rng, 1, 2048)
    out = rng.choice(["bf16", "bf16", "fp32"]) if op == "gemm_q8" else "bf16"
    if op == "gemm_q8":
        return {"op": op, "rows": rows, "n": n, "k": k, "out": out}
    return {"op": op, "rows": rows, "n": n, "k": k, "group": rng.choice([32, 64, 128, 128, 256]), "zeros": rng.random() < 0.5, "out": out}


def _dtype(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _codes(x):
    """Rows in e4m3 and their scales, for inputs that a program has in hand."""
    s = x.abs().amax(1).clamp_min(LEAST) / E4M3_MAX
    return (x / s.unsqueeze(1)).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3), s


def _pack(q):
    """[N, K] entries 0 .. 15 -> int32 [N, K / 8]."""
    q = q.view(q.shape[0], -1, 8)
    w = torch.zeros(q.shape[:2], dtype=torch.int64, device=q.device)
    for i, s in enumerate(SHIFTS):
        w |= q[:, :, i].long() << s
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def _activations(g, rows, width):
    """Rows as a layer's products meet them: normal entries, a few channels far larger than the others."""
    x = torch.randn(rows, width, generator=g, device=DEVICE)
    return x * torch.where(torch.rand(width, generator=g, device=DEVICE) < 0.005, 12.0, 1.0)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    c, op, R = dict(case), case["op"], case["rows"]
    randn = lambda *shape: torch.randn(*shape, generator=g, device=DEVICE)
    empty = lambda *shape, dtype: torch.empty(*shape, dtype=dtype, device=DEVICE)
    s = {"case": c, "status": torch.zeros(1, dtype=torch.int32, device=DEVICE)}
    if op in ("norm", "swiglu", "quantize"):
        dt = _dtype(c["dtype"])
        width = c["inter"] if op == "swiglu" else c["width"]
        s["out"], s["scale"] = empty(R, width, dtype=E4M3), empty(R, dtype=torch.float32)
        if op == "norm":
            s["resid"] = _activations(g, R, width)
            s["deltas"] = [(0.3 * randn(R, width)).to(dt) for _ in range(c["deltas"])]
            s["weight"] = (1.0 + 0.1 * randn(width)).to(torch.bfloat16)
            s["stream"] = empty(R, width, dtype=torch.float32)
        elif op == "swiglu":
            s["gu"] = _activations(g, R, 2 * width).to(dt)
        else:
            s["x"] = _activations(g, R, c["stride"]).to(dt)[:, :width]
        return s
    N, K = c["n"], c["k"]
    w = 0.02 * randn(N, K)
    s["out"] = empty(R, N, dtype=_dtype(c["out"]))
    if op == "gemm_q8":
        s["a"], s["a_scale"] = _codes(_activations(g, R, K))
        s["w"], s["w_scale"] = _codes(w)
        return s
    G = -(-K // c["group"])
    w = torch.nn.functional.pad(w, (0, G * c["group"] - K)).view(N, G, c["group"])
    if c["zeros"]:
        w = w + 0.01 * randn(N, G, 1)                            # groups that do not lie around zero
        lo, hi = w.amin(2), w.amax(2)
        s["scales"] = ((hi - lo) / 15).to(torch.bfloat16)
        z = (-lo / s["scales"].float()).round().clamp(0, 15)
        s["zeros"] = z.to(torch.uint8)
    else:
        s["scales"] = (w.abs().amax(2) / 7.5).to(torch.bfloat16)
        z = torch.full((N, G), 8.0, device=DEVICE)
        s["zeros"] = None
    q = (w / s["scales"].float().unsqueeze(2) + z.unsqueeze(2)).round().clamp(0, 15)
    s["w"] = _pack(q.view(N, -1)[:, :K])
    s["x"] = _activations(g, R, K).to(torch.bfloat16)
    return s


def _gate_up(gu, group):
    """The gates and the ups of [T, 2F], interleaved in groups of columns (0: all gates, then all ups)."""
    T, F = gu.shape[0], gu.shape[1] // 2
    x = gu.view(T, -1, 2, group or F)
    return x[:, :, 0].reshape(T, F), x[:, :, 1].reshape(T, F)


def _q8_plain(y):
    s = y.abs().amax(1).clamp_min(LEAST) / E4M3_MAX
    return (y / s.unsqueeze(1)).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3), s


def _unpack(w, K):
    shifts = torch.tensor(SHIFTS, dtype=torch.int32, device=w.device)
    return ((w.unsqueeze(2) >> shifts) & 15).view(w.shape[0], K)


def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if own:
        from llm_steadyinfer_b200.csrc import ops
        if op == "norm":
            d = s["deltas"] + [None, None]
            ops.add_rmsnorm_q8(s["resid"], d[0], s["weight"], EPS, s["out"], s["scale"], delta2=d[1], dst=s["stream"])
            return {"codes": s["out"], "scale": s["scale"], "stream": s["stream"]}
        if op == "swiglu":
            ops.swiglu_q8(s["gu"], s["out"], s["scale"], c["group"] or None)
            return {"codes": s["out"], "scale": s["scale"]}
        if op == "quantize":
            ops.quantize_q8(s["x"], s["out"], s["scale"])
            return {"codes": s["out"], "scale": s["scale"]}
        if op == "gemm_q8":
            ops.gemm_q8(s["a"], s["a_scale"], s["w"], s["w_scale"], s["out"], s["status"])
            return {"out": s["out"]}
        ops.gemm_w4(s["x"], s["w"], s["scales"], s["zeros"], c["group"], s["out"], s["status"])
        return {"out": s["out"]}
    if op == "norm":
        h = s["resid"].clone()
        for d in s["deltas"]:
            h += d.float()
        y = s["weight"].float() * (h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS))
        codes, scale = _q8_plain(y)
        return {"codes": codes, "scale": scale, "stream": h}
    if op == "swiglu":
        gate, up = _gate_up(s["gu"].float(), c["group"])
        codes, scale = _q8_plain(gate / (1.0 + torch.exp(-gate)) * up)
        return {"codes": codes, "scale": scale}
    if op == "quantize":
        codes, scale = _q8_plain(s["x"].float())
        return {"codes": codes, "scale": scale}
    if op == "gemm_q8":
        y = torch.mm(s["a"].float(), s["w"].float().t()) * s["a_scale"].unsqueeze(1) * s["w_scale"]
        return {"out": y.to(s["out"].dtype)}
    K, group = c["k"], c["group"]
    zeros = 8.0 if s["zeros"] is None else s["zeros"].float().repeat_interleave(group, 1)[:, :K]
    w = (_unpack(s["w"], K).float() - zeros) * s["scales"].float().repeat_interleave(group, 1)[:, :K]
    return {"out": torch.mm(s["x"].float(), w.t()).to(s["out"].dtype)}


def work(case):
    c, op, R = case, case["op"], case["rows"]
    if op == "norm":
        e, d = (2 if c["dtype"] == "bf16" else 4), c["width"]
        return {"bytes": R * d * (4 + e * c["deltas"] + 4 + 1) + 2 * d + 4 * R, "flops": R * d * (8 + c["deltas"])}
    if op == "swiglu":
        e = 2 if c["dtype"] == "bf16" else 4
        return {"bytes": R * c["inter"] * (2 * e + 1) + 4 * R, "flops": R * c["inter"] * 8}
    if op == "quantize":
        e = 2 if c["dtype"] == "bf16" else 4
        return {"bytes": R * c["width"] * (e + 1) + 4 * R, "flops": R * c["width"] * 3}
    N, K = c["n"], c["k"]
    out = R * N * (2 if c["out"] == "bf16" else 4)
    if op == "gemm_q8":
        return {"bytes": R * K + N * K + 4 * (R + N) + out, "flops": 2 * R * N * K}
    groups = N * -(-K // c["group"])
    return {"bytes": 2 * R * K + N * K // 2 + groups * (3 if c["zeros"] else 2) + out, "flops": 2 * R * N * K}


def exact(case, seed):
    """What ``run`` returns in 64 bits, entry for entry from the definitions; the codes before they are rounded to eight bits."""
    s = prepare(case, seed)
    c, op = case, case["op"]

    def scaled(y):
        top = torch.maximum(y.abs().max(dim=1).values, torch.tensor(LEAST, dtype=torch.float64, device=y.device))
        scale = top / 448.0
        return {"codes": y / scale[:, None], "scale": scale}

    if op == "norm":
        h = sum((d.double() for d in s["deltas"]), s["resid"].double())
        y = h / torch.sqrt(h.pow(2).sum(1, keepdim=True) / c["width"] + EPS) * s["weight"].double()
        return {**scaled(y), "stream": h}
    if op == "swiglu":
        F, group = c["inter"], c["group"] or c["inter"]
        f = torch.arange(F, device=DEVICE)
        at = f // group * 2 * group + f % group                  # the column of output f's gate; its up lies a group further
        gate, up = s["gu"][:, at].double(), s["gu"][:, at + group].double()
        return scaled(gate * torch.sigmoid(gate) * up)
    if op == "quantize":
        return scaled(s["x"].double())
    if op == "gemm_q8":
        a, w = s["a"].double() * s["a_scale"].double()[:, None], s["w"].double() * s["w_scale"].double()[:, None]
        return {"out": a @ w.t()}
    N, K = c["n"], c["k"]
    k = torch.arange(K, device=DEVICE)
    words = s["w"].long() & 0xFFFFFFFF
    w = torch.empty(N, K, dtype=torch.float64, device=DEVICE)
    for i in range(8):                                           # entry i of every eight: bit 4 (i / 2), and 16 more where i is odd
        w[:, i::8] = ((words >> (4 * (i // 2) + 16 * (i % 2))) % 16).double()
    group = k // c["group"]
    w -= 8.0 if s["zeros"] is None else s["zeros"].double()[:, group]
    w *= s["scales"].double()[:, group]
    return {"out": s["x"].double() @ w.t()}
