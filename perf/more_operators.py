"""A layer in 8-bit floating point between the residual stream and back, measured as a serving program calls its operators.

Weights are e4m3 with a scale for each block of 128 x 128, activations e4m3 with a scale for each row's 128 columns (the last
group or block may be shorter). With `own` false `run` computes the operators in elementary torch operations in 32 bits,
rounded once at the end; with `own` true it calls the framework (`qengine_amd.ops`). A case is a dict of plain values; the
lengths of experts' segments follow from the case alone, values and indexes from the seed.

Kinds:
  norm     root-mean-square norm, with or without the residual's addition, to 16 bits or to 8 bits with scales (ops.rms_norm)
  act      silu(gate) * up, or a row as it is, to 8 bits with scales (ops.silu_mul_f8, ops.quant_f8)
  linear   one 8-bit matrix (ops.matmul_f8)
  experts  products grouped by expert over ragged segments, rows gathered by index or in order (ops.matmul_f8_grouped)
  combine  the experts' rows summed into tokens by routing weights (ops.moe_combine)

Quantized outputs are the e4m3 values and, beside them, their scales.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
F8 = torch.float8_e4m3fn
EPS = 1e-6
LOW = 448 * 2.0 ** -100  # the least that a group's largest value counts as


# ------------------------------------------------------------------------------------------------ cases
def listed():
    # hidden 5120 / intermediate 17408, and 512 experts of hidden 2048 / intermediate 512, 10 a token, are bench.py's layers
    return [
        # one sequence generating: a block's norm, the latency of a token
        {"name": "norm_1", "kind": "norm", "rows": 1, "d": 5120, "dtype": "bf16", "res": True, "f8": True},
        # a long prompt through the same norm
        {"name": "norm_8192", "kind": "norm", "rows": 8192, "d": 5120, "dtype": "bf16", "res": True, "f8": True},
        # a dozen sequences between the two products of an MLP
        {"name": "act_12", "kind": "act", "rows": 12, "d": 17408, "dtype": "bf16", "glu": True},
        # a prefill chunk there
        {"name": "act_4096", "kind": "act", "rows": 4096, "d": 17408, "dtype": "bf16", "glu": True},
        # one sequence generating: the second matrix of an MLP
        {"name": "linear_1", "kind": "linear", "rows": 1, "n": 5120, "k": 17408, "out": "bf16"},
        # a busy server's decode batch through the first (gate and up in one)
        {"name": "linear_48", "kind": "linear", "rows": 48, "n": 34816, "k": 5120, "out": "bf16"},
        # a chunk of a chunked prefill, ragged at its end
        {"name": "linear_1000", "kind": "linear", "rows": 1000, "n": 5120, "k": 17408, "out": "bf16"},
        # a long prompt in one call
        {"name": "linear_8192", "kind": "linear", "rows": 8192, "n": 17408, "k": 5120, "out": "bf16"},
        # 16 sequences decoded together, their experts' first product: most segments are empty, the others 1 to 4 rows
        {"name": "experts_16", "kind": "experts", "experts": 512, "topk": 10, "tokens": 16, "n": 1024, "k": 2048, "gather": True,
         "out": "bf16"},
        # a prompt through it: about 80 rows an expert
        {"name": "experts_4096", "kind": "experts", "experts": 512, "topk": 10, "tokens": 4096, "n": 1024, "k": 2048,
         "gather": True, "out": "bf16"},
        # the experts' results of those 16 sequences into the residual stream
        {"name": "combine_16", "kind": "combine", "tokens": 16, "topk": 10, "d": 2048, "dtype": "bf16", "add": True},
        # and of the prompt
        {"name": "combine_4096", "kind": "combine", "tokens": 4096, "topk": 10, "d": 2048, "dtype": "bf16", "add": True},
    ]


MOST_FLOPS = 2.0 * 8192 * 17408 * 5120
MOST_EXPERT_FLOPS = 2.0 * 40960 * 1024 * 2048
MOST_WEIGHTS = 512 * 1024 * 2048


def _log(rng, lo, hi, step=1):
    """a multiple of `step` in [lo, hi], spread over the logarithm"""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(hi, max(lo, step * round(v / step))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "act", "act", "linear", "linear", "linear", "experts", "experts", "combine"])
    while True:
        step = rng.choice([1, 8, 128])
        if kind == "norm":
            c = {"kind": kind, "rows": _log(rng, 1, 16384), "d": _log(rng, 128, 16384, step), "dtype": rng.choice(["bf16", "f16"]),
                 "res": rng.random() < 0.6, "f8": rng.random() < 0.6}
            if c["rows"] * c["d"] <= 8192 * 5120:
                return c
        elif kind == "act":
            c = {"kind": kind, "rows": _log(rng, 1, 16384), "d": _log(rng, 128, 17408, step), "dtype": rng.choice(["bf16", "f16"]),
                 "glu": rng.random() < 0.6}
            if c["rows"] * c["d"] <= 4096 * 17408:
                return c
        elif kind == "linear":
            c = {"kind": kind, "rows": _log(rng, 1, 8192), "n": _log(rng, 256, 34816, step), "k": _log(rng, 256, 17408, 16 * rng.choice([1, 8])),
                 "out": rng.choice(["bf16", "bf16", "f16"])}
            if work(c)["flops"] <= MOST_FLOPS:
                return c
        elif kind == "experts":
            c = {"kind": kind, "experts": rng.choice([8, 32, 60, 128, 256, 512]), "topk": rng.randint(1, 10), "tokens": _log(rng, 1, 4096),
                 "n": _log(rng, 256, 4096, step), "k": _log(rng, 256, 4096, 16 * rng.choice([1, 8])), "gather": rng.random() < 0.5,
                 "out": rng.choice(["bf16", "bf16", "f16"])}
            if c["topk"] <= c["experts"] and work(c)["flops"] <= MOST_EXPERT_FLOPS and c["experts"] * c["n"] * c["k"] <= MOST_WEIGHTS:
                return c
        else:
            c = {"kind": kind, "tokens": _log(rng, 1, 8192), "topk": rng.randint(1, 10), "d": _log(rng, 128, 8192, step),
                 "dtype": rng.choice(["bf16", "f16", "f32"]), "add": rng.random() < 0.5}
            if c["tokens"] * c["topk"] * c["d"] <= 40960 * 2048:
                return c


def _segments(case):
    """rows of each expert: every token goes to `topk` of them, some experts are chosen more often than others"""
    text = "/".join("%s=%s" % (k, case[k]) for k in ("experts", "topk", "tokens", "n", "k"))
    rng = random.Random(text)
    p = np.array([math.exp(rng.gauss(0, 0.4)) for _ in range(case["experts"])])
    return np.random.RandomState(rng.randrange(1 << 31)).multinomial(case["tokens"] * case["topk"], p / p.sum())


def work(case):
    kind, up = case["kind"], lambda v: -(-v // 128)
    size = {"bf16": 2, "f16": 2, "f32": 4}
    if kind == "norm":
        v = case["rows"] * case["d"]
        moved = 2 * v * (3 if case["res"] else 1) + 4 * case["d"]
        return {"bytes": moved + (v + 4 * case["rows"] * up(case["d"]) if case["f8"] else 2 * v), "flops": 5 * v}
    if kind == "act":
        v = case["rows"] * case["d"]
        return {"bytes": 2 * v * (2 if case["glu"] else 1) + v + 4 * case["rows"] * up(case["d"]), "flops": (8 if case["glu"] else 3) * v}
    if kind == "combine":
        t, k, d = case["tokens"], case["topk"], case["d"]
        return {"bytes": size[case["dtype"]] * t * d * (k + 1 + case["add"]) + 8 * t * k, "flops": 2 * t * k * d}
    n, k = case["n"], case["k"]
    if kind == "linear":
        x, rows, mats = case["rows"], case["rows"], 1
    else:
        rows = case["tokens"] * case["topk"]
        x, mats = case["tokens"] if case["gather"] else rows, int((_segments(case) > 0).sum())
    moved = mats * (n * k + 4 * up(n) * up(k)) + x * (k + 4 * up(k)) + rows * n * size[case["out"]]
    return {"bytes": moved + (4 * (case["experts"] + 1 + rows) if kind == "experts" else 0), "flops": 2.0 * rows * n * k}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _stream(g, rows, d, dtype, size=1.0):
    """activations: N(0, size) with some columns several times larger, as hidden states have"""
    wide = torch.exp(torch.randn(d, device=DEV, generator=g) * 0.6)
    return (torch.randn(rows, d, device=DEV, generator=g) * (wide * size)).to(dtype)


def _activations(g, rows, k):
    """e4m3 [rows][k] and scales [rows][groups] of such activations"""
    x, groups = torch.zeros(rows, -(-k // 128) * 128, device=DEV), -(-k // 128)
    x[:, :k] = _stream(g, rows, k, torch.float32)
    x = x.view(rows, groups, 128)
    top = x.abs().amax(-1).clamp_min(LOW)
    q = (x * (448 / top)[..., None]).view(rows, -1)[:, :k].to(F8).contiguous()
    return q, (top / 448).t().contiguous().t()


def _weights(g, lead, n, k):
    """e4m3 [lead..][n][k] of N(0, 1 / k) and scales [lead..][blocks of n][blocks of k]"""
    bn, bk = -(-n // 128), -(-k // 128)
    q = torch.empty(*lead, n, k, dtype=F8, device=DEV)
    s = torch.empty(*lead, bn, bk, device=DEV)
    parts = [(q, s)] if not lead else zip(q, s)
    for one, scales in parts:
        w = torch.zeros(bn * 128, bk * 128, device=DEV)
        w[:n, :k] = torch.randn(n, k, device=DEV, generator=g) * k ** -0.5
        w = w.view(bn, 128, bk, 128)
        top = w.abs().amax((1, 3))
        scales.copy_(top / 448)
        one.copy_((w * (448 / top)[:, None, :, None]).view(bn * 128, -1)[:n, :k].to(F8))
    return q, s


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    s = {"case": case}
    if kind == "norm":
        dtype = DT[case["dtype"]]
        s["x"] = _stream(g, case["rows"], case["d"], dtype, 0.3)
        s["w"] = 1 + 0.2 * torch.randn(case["d"], device=DEV, generator=g)
        if case["res"]:
            s["r"] = _stream(g, case["rows"], case["d"], dtype)
            s["h"] = torch.zeros_like(s["r"])  # the stream's next buffer
    elif kind == "act":
        s["x"] = _stream(g, case["rows"], case["d"] * (2 if case["glu"] else 1), DT[case["dtype"]])
    elif kind == "linear":
        s["x"], s["xs"] = _activations(g, case["rows"], case["k"])
        s["q"], s["qs"] = _weights(g, (), case["n"], case["k"])
    elif kind == "experts":
        lens = _segments(case)
        rows = int(lens.sum())
        s["off"] = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=DEV)
        s["most"] = int(lens.max())
        s["rows"] = None
        if case["gather"]:  # slots of a token: spread over the experts' segments
            s["rows"] = torch.randperm(rows, device=DEV, generator=g).int() % case["tokens"]
        s["x"], s["xs"] = _activations(g, case["tokens"] if case["gather"] else rows, case["k"])
        s["q"], s["qs"] = _weights(g, (case["experts"],), case["n"], case["k"])
    else:
        t, k, dtype = case["tokens"], case["topk"], DT[case["dtype"]]
        s["y"] = _stream(g, t * k, case["d"], dtype)
        s["inv"] = torch.randperm(t * k, device=DEV, generator=g).int()
        s["w"] = torch.softmax(torch.randn(t, k, device=DEV, generator=g), -1)
        s["add"] = _stream(g, t, case["d"], dtype) if case["add"] else None
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    return _run_own(s) if own else _PLAIN[s["case"]["kind"]](s)


def _run_own(s):
    from qengine_amd import ops
    c = s["case"]
    kind = c["kind"]
    if kind == "norm":
        r, h = s.get("r"), s.get("h")
        if c["f8"]:
            q, scales = ops.rms_norm(s["x"], s["w"], EPS, res=r, res_out=h, f8=True)
            out = {"q": q, "s": scales}
        else:
            out = {"y": ops.rms_norm(s["x"], s["w"], EPS, res=r, res_out=h)}
        return out if h is None else {**out, "h": h}
    if kind == "act":
        q, scales = ops.silu_mul_f8(s["x"]) if c["glu"] else ops.quant_f8(s["x"])
        return {"q": q, "s": scales}
    if kind == "combine":
        return ops.moe_combine(s["y"], s["inv"], s["w"], add=s["add"])
    if "handle" not in s:  # the weights as a server keeps them from its start on
        s["handle"] = ops.tile_f8(s["q"], s["qs"])
    if kind == "linear":
        return ops.matmul_f8(s["handle"], s["x"], s["xs"], dtype=DT[c["out"]])
    return ops.matmul_f8_grouped(s["handle"], s["x"], s["xs"], s["off"], rows=s["rows"], dtype=DT[c["out"]])


# ---- the plain forms
def _plain_quantized(v):
    rows, d = v.shape
    groups = -(-d // 128)
    v = torch.nn.functional.pad(v, (0, groups * 128 - d)).view(rows, groups, 128)
    top = v.abs().amax(-1).clamp_min(LOW)
    q = (v * (448 / top)[..., None]).view(rows, -1)[:, :d].to(F8)
    return {"q": q, "s": top / 448}


def _plain_norm(s):
    c, out = s["case"], {}
    h = s["x"]
    if c["res"]:
        h = s["h"].copy_((h.float() + s["r"].float()).to(h.dtype))
        out["h"] = h
    h = h.float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * s["w"]
    return {**out, **(_plain_quantized(y) if c["f8"] else {"y": y.to(s["x"].dtype)})}


def _plain_act(s):
    x = s["x"].float()
    if s["case"]["glu"]:
        gate, up = x.chunk(2, 1)
        x = gate / (1 + torch.exp(-gate)) * up
    return _plain_quantized(x)


def _spread(scales, n, k):
    """a block's scale for each of its values"""
    return scales.repeat_interleave(128, -2)[..., :n, :].repeat_interleave(128, -1)[..., :k]


def _plain_linear(s):
    c = s["case"]
    x = s["x"].float() * s["xs"].repeat_interleave(128, 1)[:, :c["k"]]
    w = s["q"].float() * _spread(s["qs"], c["n"], c["k"])
    return (x @ w.t()).to(DT[c["out"]])


def _plain_experts(s):
    c, off = s["case"], s["off"].long()
    x = s["x"].float() * s["xs"].repeat_interleave(128, 1)[:, :c["k"]]
    if s["rows"] is not None:
        x = x[s["rows"].long()]
    at = torch.arange(s["most"], device=DEV)
    live = at < (off[1:] - off[:-1])[:, None]        # [experts, most] places of a padded batch
    idx = torch.where(live, off[:-1, None] + at, torch.zeros_like(at))
    w = s["q"].view(torch.uint8).transpose(1, 2).contiguous().view(F8).float()
    w *= _spread(s["qs"].transpose(1, 2), c["k"], c["n"])
    y = torch.bmm(x[idx], w)
    out = torch.zeros(x.shape[0] + 1, c["n"], device=DEV)
    out[torch.where(live, idx, torch.full_like(idx, x.shape[0]))] = y  # places past a segment go to a row that is dropped
    return out[:-1].to(DT[c["out"]])


def _plain_combine(s):
    c = s["case"]
    y = s["y"].float()[s["inv"].long()].view(c["tokens"], c["topk"], c["d"])
    out = (y * s["w"][..., None]).sum(1)
    if c["add"]:
        out = out + s["add"].float()
    return out.to(DT[c["dtype"]])


_PLAIN = {"norm": _plain_norm, "act": _plain_act, "linear": _plain_linear, "experts": _plain_experts, "combine": _plain_combine}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_quantized(v):
    """e4m3 values before their rounding, and the scales"""
    q, scales = torch.empty_like(v), []
    for a in range(0, v.shape[1], 128):
        part = v[:, a:a + 128]
        top = torch.maximum(part.max(1).values, -part.min(1).values)
        top = torch.where(top < LOW, torch.full_like(top, LOW), top)
        scales.append(top / 448)
        q[:, a:a + 128] = part / scales[-1][:, None]
    return {"q": q, "s": torch.stack(scales, 1)}


def _exact_product(x, xs, q, qs):
    """sums of each block of 128 by themselves, scaled and added"""
    y = torch.zeros(x.shape[0], q.shape[0], dtype=torch.float64, device=DEV)
    block = torch.arange(q.shape[0], device=DEV) // 128
    for b, a in enumerate(range(0, q.shape[1], 128)):
        part = x[:, a:a + 128].double() @ q[:, a:a + 128].double().t().contiguous()
        y += part * xs[:, b:b + 1].double() * qs[block, b].double()
    return y


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "norm":
        h, out = s["x"], {}
        if case["res"]:
            h = (h.double() + s["r"].double()).to(h.dtype)  # the stream is held in 16 bits
            out["h"] = h
        h = h.double()
        y = s["w"].double() * h / (h.square().sum(1, keepdim=True) / case["d"] + EPS).sqrt()
        return {**out, **(_exact_quantized(y) if case["f8"] else {"y": y})}
    if kind == "act":
        x = s["x"].double()
        if case["glu"]:
            gate, up = x[:, :case["d"]], x[:, case["d"]:]
            x = gate * up * torch.sigmoid(gate)
        return _exact_quantized(x)
    if kind == "linear":
        return _exact_product(s["x"], s["xs"], s["q"], s["qs"])
    if kind == "experts":
        off = s["off"].tolist()
        x, xs = (s["x"], s["xs"]) if s["rows"] is None else (s["x"].view(torch.uint8)[s["rows"].long()].view(F8), s["xs"][s["rows"].long()])
        y = torch.zeros(off[-1], case["n"], dtype=torch.float64, device=DEV)
        for e, (a, z) in enumerate(zip(off[:-1], off[1:])):
            if z > a:
                y[a:z] = _exact_product(x[a:z], xs[a:z], s["q"][e], s["qs"][e])
        return y
    out = s["add"].double() if case["add"] else torch.zeros(case["tokens"], case["d"], dtype=torch.float64, device=DEV)
    inv = s["inv"].long().view(case["tokens"], -1)
    for j in range(case["topk"]):
        out += s["w"][:, j:j + 1].double() * s["y"][inv[:, j]].double()
    return out
