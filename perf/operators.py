"""The framework's 16- and 32-bit model operators and their gradients, as measured work.

Each case is one call of one operator: the embedding lookup and its gradient,
the per-head norm of queries, keys and values with the position rotation and
its gradient, and the gated feed-forward projection and its gradient.  With
``own`` false the operators run in a plain form of elementary torch operations
in 32 bits; with ``own`` true they run as the framework's kernels
(include/eg2_ops.h through ops.py).  ``exact`` gives the same outputs in
64 bits.
"""
import importlib
import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
EPS = 1e-6


def _ops():
    return importlib.import_module("embeddinggemma2-amdkfd_b200.ops")


# ---------------------------------------------------------------- cases
def listed():
    return [
        # One token entering the model: the latency of a lookup.
        {"name": "embed_token", "op": "embed", "n": 1, "vocab": 262144, "d": 512, "dtype": "fp16", "out": "fp16",
         "zipf": False, "pad": 0.0},
        # A training batch of packed text, natural token frequencies, some padding.
        {"name": "embed_batch", "op": "embed", "n": 61447, "vocab": 262144, "d": 512, "dtype": "bf16", "out": "bf16",
         "zipf": True, "pad": 0.05},
        # The gradient of one packed wave into the whole fp32 table.
        {"name": "embed_grad_wave", "op": "embed_grad", "n": 1999, "vocab": 262144, "d": 512, "dtype": "fp32",
         "out": "fp32", "zipf": False, "pad": 0.0},
        # The gradient of a large batch, natural frequencies: a few tokens hold a large share of the rows.
        {"name": "embed_grad_batch", "op": "embed_grad", "n": 100003, "vocab": 262144, "d": 512, "dtype": "bf16",
         "out": "bf16", "zipf": True, "pad": 0.05},
        # One token through a sliding-window layer's heads.
        {"name": "qkv_token", "op": "qkv", "n": 1, "hq": 4, "hkv": 2, "d": 256, "dtype": "bf16", "pad": 0.0},
        # A training batch, heads of 128 (generic).
        {"name": "qkv_batch", "op": "qkv", "n": 32771, "hq": 8, "hkv": 2, "d": 128, "dtype": "bf16", "pad": 0.05},
        # One packed wave through a sliding-window layer, trained in 32 bits.
        {"name": "qkv_grad_wave", "op": "qkv_grad", "n": 2011, "hq": 4, "hkv": 2, "d": 256, "dtype": "fp32",
         "pad": 0.0},
        # A training batch, many query heads on two key heads (generic).
        {"name": "qkv_grad_batch", "op": "qkv_grad", "n": 16411, "hq": 16, "hkv": 2, "d": 128, "dtype": "bf16",
         "pad": 0.05},
        # One token through the model's feed-forward projection: the weights are what there is to read.
        {"name": "glu_token", "op": "glu", "n": 1, "k": 512, "m": 2048, "dtype": "bf16", "act": "gelu_tanh"},
        # A training batch through a wider feed-forward block (generic).
        {"name": "glu_batch", "op": "glu", "n": 16411, "k": 2048, "m": 8192, "dtype": "bf16", "act": "silu"},
        # One packed wave through the model's own feed-forward block, backward.
        {"name": "glu_grad_wave", "op": "glu_grad", "n": 2048, "k": 512, "m": 2048, "dtype": "fp16",
         "act": "gelu_tanh"},
        # A training batch through a wider feed-forward block, backward (generic).
        {"name": "glu_grad_batch", "op": "glu_grad", "n": 8203, "k": 2048, "m": 8192, "dtype": "bf16",
         "act": "gelu_tanh"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "qkv", "qkv_grad", "glu", "glu_grad"])
    if op in ("embed", "embed_grad"):
        d = rng.randint(24, 1024)
        if rng.random() < 0.75:  # most models' widths are whole 16-byte vectors
            d = (d + 7) // 8 * 8
        case = {"op": op, "n": _log(rng, 1, 100003), "vocab": _log(rng, 1000, 262144), "d": d,
                "dtype": rng.choice(list(DTYPES)), "zipf": rng.random() < 0.6,
                "pad": rng.choice([0.0, 0.05, 0.4])}
        case["out"] = rng.choice([case["dtype"], "fp32"])
    elif op in ("qkv", "qkv_grad"):
        hkv = rng.choice([1, 2, 3, 4])
        case = {"op": op, "n": _log(rng, 1, 32771), "hq": hkv * rng.choice([1, 2, 4, 5]), "hkv": hkv,
                "d": rng.choice([48, 64, 80, 96, 128, 192, 256, 512]), "dtype": rng.choice(list(DTYPES)),
                "pad": rng.choice([0.0, 0.05, 0.4])}
    else:
        case = {"op": op, "n": _log(rng, 1, 16411), "k": 8 * _log(rng, 8, 256), "m": 8 * _log(rng, 8, 1024),
                "dtype": rng.choice(["bf16", "fp16"]), "act": rng.choice(["gelu_tanh", "silu"])}
    # No more bytes and operations than the operator's largest listed case.
    most = [work(c) for c in listed() if c["op"] == op]
    while any(work(case)[u] > max(w[u] for w in most) for u in ("bytes", "flops")):
        case["n"] = case["n"] * 3 // 4 + 1 if case["n"] > 3 else 1
        if "vocab" in case:
            case["vocab"] = case["vocab"] * 7 // 8
    return case


# ---------------------------------------------------------------- inputs
def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1000003 + salt)
    return g


def _ids(case, g):
    """Token ids: uniform, or with probability falling as 1/(rank + 1); -1 pads."""
    n, v = case["n"], case["vocab"]
    u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
    ids = (torch.exp(u * math.log(v)) - 1.0 if case["zipf"] else u * v).to(torch.int32).clamp_(0, v - 1)
    pads = torch.rand(n, generator=g, device=DEV) < case["pad"]
    return torch.where(pads, torch.full_like(ids, -1), ids)


def _rope_tables(d, positions):
    i = torch.arange(d // 2, dtype=torch.float64, device=DEV)
    angle = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * 10000.0 ** (-2.0 * i / d)
    return torch.cos(angle).float(), torch.sin(angle).float()


def _randn(shape, g, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def prepare(case, seed):
    op, n, dt = case["op"], case["n"], DTYPES[case["dtype"]]
    g = _gen(seed, 7)
    s = {"case": case}
    if op in ("embed", "embed_grad"):
        v, d = case["vocab"], case["d"]
        s["ids"], s["scale"] = _ids(case, g), math.sqrt(d)
        if op == "embed":
            s["table"] = _randn((v, d), g, dt, 1.0 / math.sqrt(d))
            s["out"] = torch.empty((n, d), dtype=DTYPES[case["out"]], device=DEV)
        else:
            s["dout"] = _randn((n, d), g, dt)
            s["dtable"] = torch.empty((v, d), dtype=DTYPES[case["out"]], device=DEV)
            if own:
                s["ws"] = torch.empty(_ops().embed_rows_grad_workspace(n, d), dtype=torch.uint8, device=DEV)
    elif op in ("qkv", "qkv_grad"):
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        heads = hq + 2 * hkv
        # The projection's output row holds a token's queries, keys and values side by side.
        qkv = _randn((n, heads, d), g, dt, 2.0)
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        s["qw"] = 1.0 + 0.1 * torch.randn(d, generator=g, device=DEV)
        s["kw"] = 1.0 + 0.1 * torch.randn(d, generator=g, device=DEV)
        s["cos"], s["sin"] = _rope_tables(d, 8192)
        # Packed sequences: each token's position in its own sequence; -1 pads.
        pos = (torch.arange(n, device=DEV) + int(seed) * 37) % 2039
        pads = torch.rand(n, generator=g, device=DEV) < case["pad"]
        s["pos"] = torch.where(pads, torch.full_like(pos, -1), pos).to(torch.int32)
        if op == "qkv":
            s["oq"] = torch.empty((n, hq, d), dtype=dt, device=DEV)
            s["ok"], s["ov"] = (torch.empty((n, hkv, d), dtype=dt, device=DEV) for _ in range(2))
        else:
            s["gq"], s["gk"], s["gv"] = _randn((n, hq, d), g, dt), _randn((n, hkv, d), g, dt), _randn((n, hkv, d), g, dt)
            s["dqkv"] = torch.empty((n, heads, d), dtype=dt, device=DEV)
            s["dqw"], s["dkw"] = torch.empty(d, device=DEV), torch.empty(d, device=DEV)
            if own:
                s["ws"] = torch.empty(_ops().qkv_norm_rope_grad_workspace(n, hq, hkv, d), dtype=torch.uint8,
                                      device=DEV)
    else:
        k, m = case["k"], case["m"]
        s["x"] = _randn((n, k), g, dt)
        s["wg"], s["wu"] = _randn((m, k), g, dt, 1.0 / math.sqrt(k)), _randn((m, k), g, dt, 1.0 / math.sqrt(k))
        if op == "glu":
            s["out"] = torch.empty((n, m), dtype=dt, device=DEV)
        else:
            s["dout"] = _randn((n, m), g, dt)
            s["dx"], s["dwg"], s["dwu"] = torch.empty_like(s["x"]), torch.empty_like(s["wg"]), torch.empty_like(s["wu"])
            if own:
                s["ws"] = torch.empty(_ops().glu_grad_workspace(n, k, m), dtype=torch.uint8, device=DEV)
    return s


# ---------------------------------------------------------------- the framework's calls
def _run_own(s):
    ops, op = _ops(), s["case"]["op"]
    if op == "embed":
        ops.embed_rows(s["out"], s["table"], s["ids"], s["scale"])
        return s["out"]
    if op == "embed_grad":
        ops.embed_rows_grad(s["dtable"], s["dout"], s["ids"], s["scale"], workspace=s["ws"])
        return s["dtable"]
    if op == "qkv":
        ops.qkv_norm_rope(s["oq"], s["ok"], s["ov"], s["q"], s["k"], s["v"], s["qw"], s["kw"], s["cos"], s["sin"],
                          s["pos"], EPS)
        return s["oq"], s["ok"], s["ov"]
    if op == "qkv_grad":
        hq, hkv, dqkv = s["case"]["hq"], s["case"]["hkv"], s["dqkv"]
        ops.qkv_norm_rope_grad(dqkv[:, :hq], dqkv[:, hq:hq + hkv], dqkv[:, hq + hkv:], s["dqw"], s["dkw"], s["gq"],
                               s["gk"], s["gv"], s["q"], s["k"], s["v"], s["qw"], s["kw"], s["cos"], s["sin"],
                               s["pos"], EPS, workspace=s["ws"])
        return dqkv, s["dqw"], s["dkw"]
    if op == "glu":
        ops.glu(s["out"], s["x"], s["wg"], s["wu"], s["case"]["act"])
        return s["out"]
    ops.glu_grad(s["dx"], s["dwg"], s["dwu"], s["dout"], s["x"], s["wg"], s["wu"], s["case"]["act"],
                 workspace=s["ws"])
    return s["dx"], s["dwg"], s["dwu"]


# ---------------------------------------------------------------- plain forms, 32 bits
def _norm(x):
    x = x.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)


def _act(g, act):
    u = g if act == "silu" else 2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g)
    return g / (1.0 + torch.exp(-u))


def _act_grad(g, act):
    if act == "silu":
        u, du = g, 1.0
    else:
        c = 2.0 * math.sqrt(2.0 / math.pi)
        u, du = c * (g + 0.044715 * g * g * g), c * (1.0 + 3.0 * 0.044715 * g * g)
    sg = 1.0 / (1.0 + torch.exp(-u))
    # 1 - sg as its own quotient: a subtraction would lose it where sg is near 1.
    return sg * (1.0 + g * du / (1.0 + torch.exp(u)))


def _run_plain(s):
    case = s["case"]
    op, dt = case["op"], DTYPES[case["dtype"]]
    if op == "embed":
        rows = s["table"][s["ids"].clamp(min=0).long()].float() * s["scale"]
        return torch.where((s["ids"] >= 0)[:, None], rows, 0.0).to(DTYPES[case["out"]])
    if op == "embed_grad":
        rows = torch.where((s["ids"] >= 0)[:, None], s["dout"].float(), 0.0)
        total = torch.zeros(s["dtable"].shape, device=DEV).index_add_(0, s["ids"].clamp(min=0), rows)
        return (total * s["scale"]).to(DTYPES[case["out"]])
    if op in ("qkv", "qkv_grad"):
        keep = (s["pos"] >= 0)[:, None, None]
        pos = s["pos"].clamp(min=0).long()
        c, sn = s["cos"][pos][:, None, :], s["sin"][pos][:, None, :]
    if op == "qkv":
        outs = []
        for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
            a, b = (_norm(x) * w).chunk(2, -1)
            outs.append(torch.cat([a * c - b * sn, b * c + a * sn], -1))
        outs.append(_norm(s["v"]))
        return tuple(torch.where(keep, o, 0.0).to(dt) for o in outs)
    if op == "qkv_grad":
        dxs, dws = [], []
        for x, w, go in ((s["q"], s["qw"], s["gq"]), (s["k"], s["kw"], s["gk"]), (s["v"], None, s["gv"])):
            x, go = x.float(), go.float()
            r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
            if w is not None:
                a, b = go.chunk(2, -1)
                go = torch.cat([a * c + b * sn, b * c - a * sn], -1)
                dws.append(torch.where(keep, go * (x * r), 0.0).sum((0, 1)))
                go = go * w
            dx = r * (go - x * r * (go * (x * r)).mean(-1, keepdim=True))
            dxs.append(torch.where(keep, dx, 0.0).to(dt))
        return torch.cat(dxs, 1), dws[0], dws[1]
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
    gate, up = x @ wg.t(), x @ wu.t()
    if op == "glu":
        return (_act(gate, case["act"]) * up).to(dt)
    dh = s["dout"].float()
    dgate, dup = dh * up * _act_grad(gate, case["act"]), dh * _act(gate, case["act"])
    return (dgate @ wg + dup @ wu).to(dt), (dgate.t() @ x).to(dt), (dup.t() @ x).to(dt)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------- what a pass cannot do without
def _distinct(case):
    """Expected number of table rows that the case's ids touch."""
    n, v = case["n"] * (1.0 - case["pad"]), case["vocab"]
    if not case["zipf"]:
        return v * -math.expm1(n * math.log1p(-1.0 / v))
    p = np.log1p(1.0 / np.arange(1.0, v)) / math.log(v)
    return float((-np.expm1(n * np.log1p(-p))).sum())


def work(case):
    op, n, e = case["op"], case["n"], BYTES[case["dtype"]]
    if op == "embed":
        d = case["d"]
        return {"bytes": 4 * n + _distinct(case) * d * e + n * d * BYTES[case["out"]], "flops": n * d}
    if op == "embed_grad":
        d = case["d"]
        return {"bytes": 4 * n + n * (1.0 - case["pad"]) * d * e + case["vocab"] * d * BYTES[case["out"]],
                "flops": 2 * n * d}
    if op in ("qkv", "qkv_grad"):
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        elems = n * (hq + 2 * hkv) * d
        table = min(n, 2039) * d * 4  # d / 2 cosines and d / 2 sines for each position that occurs
        if op == "qkv":
            return {"bytes": 2 * elems * e + table + 4 * n + 8 * d, "flops": 7 * elems}
        return {"bytes": 3 * elems * e + table + 4 * n + 16 * d, "flops": 16 * elems}
    k, m = case["k"], case["m"]
    if op == "glu":
        return {"bytes": (n * k + 2 * m * k + n * m) * e, "flops": 4 * n * k * m}
    # The two products forward (their outputs are not among the inputs), two for dx, two for the weights.
    return {"bytes": (2 * n * k + 4 * m * k + n * m) * e, "flops": 12 * n * k * m}


# ---------------------------------------------------------------- the definitions in 64 bits
def _f64(t):
    return t.to(torch.float64)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "embed":
        out = torch.zeros((case["n"], case["d"]), dtype=torch.float64, device=DEV)
        live = torch.nonzero(s["ids"] >= 0).flatten()
        out[live] = _f64(torch.index_select(s["table"], 0, s["ids"][live])) * s["scale"]
        return out
    if op == "embed_grad":
        # Rows in the order of their ids, summed between the places where the id changes.
        out = torch.zeros((case["vocab"], case["d"]), dtype=torch.float64, device=DEV)
        live = torch.nonzero(s["ids"] >= 0).flatten()
        if live.numel():
            ids, order = torch.sort(s["ids"][live].long(), stable=True)
            vocab_ids, counts = torch.unique_consecutive(ids, return_counts=True)
            ends = counts.cumsum(0)
            run_of = torch.repeat_interleave(torch.arange(counts.numel(), device=DEV), counts)
            for c in range(0, case["d"], 128):
                cols = _f64(s["dout"][live[order], c:c + 128])
                sums = torch.zeros((counts.numel(), cols.shape[1]), dtype=torch.float64, device=DEV)
                sums.scatter_add_(0, run_of[:, None].expand_as(cols), cols)
                out[vocab_ids, c:c + 128] = sums * s["scale"]
            assert int(ends[-1]) == live.numel()
        return out
    if op in ("qkv", "qkv_grad"):
        live = s["pos"] >= 0
        pos = torch.where(live, s["pos"], 0).long()
        half = case["d"] // 2
        # The rotation as a product of complex numbers.
        rot = torch.complex(_f64(s["cos"]), _f64(s["sin"]))[pos].unsqueeze(1)

        def turn(y, by):
            z = torch.complex(y[..., :half], y[..., half:]) * by
            return torch.cat([z.real, z.imag], -1)

        def scale(x):
            return 1.0 / torch.sqrt(torch.sum(x ** 2, -1, keepdim=True) / case["d"] + EPS)

        def mask(t):
            return t * live[:, None, None]
    if op == "qkv":
        q, k, v = _f64(s["q"]), _f64(s["k"]), _f64(s["v"])
        return (mask(turn(q * scale(q) * _f64(s["qw"]), rot)), mask(turn(k * scale(k) * _f64(s["kw"]), rot)),
                mask(v * scale(v)))
    if op == "qkv_grad":
        dx, dw = [], []
        for name, go in (("q", "gq"), ("k", "gk"), ("v", "gv")):
            x, dy = _f64(s[name]), _f64(s[go])
            r = scale(x)
            if name != "v":
                dy = turn(dy, rot.conj())
                dw.append(torch.einsum("nhd,nhd->d", mask(dy), x * r))
                dy = dy * _f64(s[name + "w"])
            # d(x r)/dx = r I - r^3 x x^T / d
            dx.append(mask(r * dy - r ** 3 * x * (torch.einsum("nhd,nhd->nh", x, dy) / case["d"])[..., None]))
        return torch.cat(dx, 1), dw[0], dw[1]
    x, wg, wu = _f64(s["x"]), _f64(s["wg"]), _f64(s["wu"])
    gate, up = torch.matmul(x, wg.T), torch.matmul(x, wu.T)
    if case["act"] == "silu":
        sg = torch.sigmoid(gate)
        a, da = gate * sg, sg + gate * sg * torch.sigmoid(-gate)
    else:
        c = math.sqrt(2.0 / math.pi)
        th = torch.tanh(c * (gate + 0.044715 * gate ** 3))
        a = 0.5 * gate * (1.0 + th)
        da = 0.5 * (1.0 + th) + 0.5 * gate * (1.0 - th ** 2) * c * (1.0 + 3.0 * 0.044715 * gate ** 2)
    if op == "glu":
        return a * up
    dh = _f64(s["dout"])
    dgate, dup = dh * up * da, dh * a
    del gate, up, a, da
    return (torch.matmul(dgate, wg) + torch.matmul(dup, wu), torch.matmul(dgate.T, x), torch.matmul(dup.T, x))
