"""The typed operators together, as a training step of the text graph uses them:
lookup, per-head norm and rotation, (torch) attention, gated projection, and back
through their gradients into the embedding table, captured in one CUDA graph.

Everything outside the gated projection is fp32 here; the projection takes and
gives bf16.  Against the same step in 64 bits the whole chain's results are off
by the bf16 roundings: the projection's input, its output and output gradient,
the two inner gradients and dx, each at most finfo.eps / 2 = 2^-8 of its value and
2^-8 of the norm, hence six of them along the longest path; products with the
activation's value or slope carry an error of G or U over with a factor below 2.2.
Every other map is linear with singular values of at most 1 or a mean over heads'
rows, except the rotation and softmax at a temperature where their slope is below
1.  The bound on the relative error in the 2-norm is 6 * 2.2 * 2^-8 = 0.052.
"""
import importlib
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BOUND = 6 * 2.2 * 2.0 ** -8
N, V, D, HQ, HKV, HD, M = 173, 400, 256, 2, 1, 64, 512
LENGTHS = (100, 1, 60)  # the last 12 rows are padding
EPS = 1e-6


@pytest.fixture(scope="module")
def ops(eg2):
    return importlib.import_module("embeddinggemma2-amdkfd_b200.ops")


def orthogonal(rows, cols, g):
    q, _ = torch.linalg.qr(torch.randn(max(rows, cols), max(rows, cols), generator=g, device=DEV))
    return q[:rows, :cols].contiguous()


def attend(q, k, v, seg):
    """Bidirectional attention inside each sequence, temperature 64; padding rows give zeros."""
    k, v = (t.expand(-1, HQ, -1) for t in (k, v))
    s = torch.einsum("ihd,jhd->hij", q, k) / 64.0
    same = (seg[:, None] == seg[None, :]) & (seg >= 0)[None, :]
    p = torch.softmax(s.masked_fill(~same[None], -1e30), -1) * same.any(1)[None, :, None]
    return torch.einsum("hij,jhd->ihd", p, v).reshape(N, HQ * HD)


def rotate(y, c, s):
    a, b = y.chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def reference(P, ids, pos, seg, dout):
    """Output and gradients of the step, in 64 bits by automatic differentiation."""
    W = {k: t.double().requires_grad_(k in ("table", "qw", "kw", "wg", "wu")) for k, t in P.items()}
    live = (pos >= 0)[:, None]
    x = torch.where(live, W["table"][ids.clamp(min=0).long()] * math.sqrt(D), 0.0)
    qkv = (x @ W["wqkv"].T).view(N, HQ + 2 * HKV, HD)
    p = pos.clamp(min=0).long()
    c, s = W["cos"][p][:, None], W["sin"][p][:, None]
    norm = lambda t: t * torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS)
    q = torch.where(live[:, None], rotate(norm(qkv[:, :HQ]) * W["qw"], c, s), 0.0)
    k = torch.where(live[:, None], rotate(norm(qkv[:, HQ:HQ + HKV]) * W["kw"], c, s), 0.0)
    v = torch.where(live[:, None], norm(qkv[:, HQ + HKV:]), 0.0)
    h = x + attend(q, k, v, seg) @ W["wo"].T
    gate, up = h @ W["wg"].T, h @ W["wu"].T
    out = torch.nn.functional.gelu(gate, approximate="tanh") * up
    grads = torch.autograd.grad((out * dout.double()).sum(), [W[k] for k in ("table", "qw", "kw", "wg", "wu")])
    return (out.detach(), *grads)


def test_training_step_against_64_bits(ops):
    g = torch.Generator(device=DEV)
    g.manual_seed(77)
    seg = torch.full((N,), -1, device=DEV, dtype=torch.int64)
    pos = torch.full((N,), -1, device=DEV, dtype=torch.int32)
    at = 0
    for i, n in enumerate(LENGTHS):
        seg[at:at + n] = i
        pos[at:at + n] = torch.arange(n, device=DEV, dtype=torch.int32)
        at += n
    i = torch.arange(HD // 2, dtype=torch.float64, device=DEV)
    angle = torch.arange(128, dtype=torch.float64, device=DEV)[:, None] * 10000.0 ** (-2.0 * i / HD)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)
    P = {"table": rand(V, D) / math.sqrt(D), "wqkv": orthogonal((HQ + 2 * HKV) * HD, D, g),
         "wo": orthogonal(D, HQ * HD, g), "qw": 1 + 0.1 * rand(HD), "kw": 1 + 0.1 * rand(HD),
         "wg": (rand(M, D) / math.sqrt(D)).bfloat16(), "wu": (rand(M, D) / math.sqrt(D)).bfloat16(),
         "cos": torch.cos(angle).float(), "sin": torch.sin(angle).float()}
    ids = torch.randint(0, V, (N,), generator=g, device=DEV, dtype=torch.int32)
    ids[pos < 0] = -1
    dout = rand(N, M).bfloat16()

    x, qkv = torch.empty(N, D, device=DEV), torch.empty(N, HQ + 2 * HKV, HD, device=DEV)
    rot, dqkv, drot = (torch.empty_like(qkv) for _ in range(3))
    out, dh = torch.empty(N, M, device=DEV, dtype=torch.bfloat16), torch.empty(N, D, device=DEV, dtype=torch.bfloat16)
    dtable = torch.empty(V, D, device=DEV)
    dqw, dkw = torch.empty(HD, device=DEV), torch.empty(HD, device=DEV)
    dwg, dwu = torch.empty(M, D, device=DEV), torch.empty(M, D, device=DEV)
    parts = lambda t: (t[:, :HQ], t[:, HQ:HQ + HKV], t[:, HQ + HKV:])

    def step():
        ops.embed_rows(x, P["table"], ids, math.sqrt(D))
        qkv.view(N, -1).copy_(x @ P["wqkv"].T)
        ops.qkv_norm_rope(*parts(rot), *parts(qkv), P["qw"], P["kw"], P["cos"], P["sin"], pos, EPS)
        r = rot.detach().requires_grad_()
        o = attend(*parts(r), seg)
        h = (x + o.detach() @ P["wo"].T).bfloat16()
        ops.glu(out, h, P["wg"], P["wu"])
        ops.glu_grad(dh, dwg, dwu, dout, h, P["wg"], P["wu"])
        (dr,) = torch.autograd.grad(o, r, dh.float() @ P["wo"])
        drot.copy_(dr)
        ops.qkv_norm_rope_grad(*parts(dqkv), dqw, dkw, *parts(drot), *parts(qkv), P["qw"], P["kw"], P["cos"],
                               P["sin"], pos, EPS)
        ops.embed_rows_grad(dtable, dh.float() + dqkv.view(N, -1) @ P["wqkv"], ids, math.sqrt(D))

    def check():
        got = (out, dtable, dqw, dkw, dwg, dwu)
        for name, a, b in zip(("out", "table", "qw", "kw", "wg", "wu"), got, reference(P, ids, pos, seg, dout)):
            err = float((a.double() - b).norm() / b.norm())
            assert err <= BOUND, (name, err)

    step()
    check()
    first = [t.clone() for t in (out, dtable, dqw, dkw, dwg, dwu)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    graph.replay()
    for a, b in zip((out, dtable, dqw, dkw, dwg, dwu), first):
        assert torch.equal(a, b)
    # Other weights, tokens and gradients through the same graph.
    P["table"].copy_(rand(V, D) / math.sqrt(D))
    P["wg"].copy_(rand(M, D) / math.sqrt(D))
    ids.copy_(torch.where(pos < 0, ids, torch.randint(0, V, (N,), generator=g, device=DEV, dtype=torch.int32)))
    dout.copy_(rand(N, M))
    graph.replay()
    check()
    assert ops.read_error() == 0


def test_two_threads_on_two_streams(ops):
    """Calls from two host threads at once, each on its stream with workspaces of its own (allocated by the call)."""
    import threading
    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)
    n, v, d, m = 5000, 3000, 128, 256
    cos, sin = rand(64, 32), rand(64, 32)
    w = rand(64)
    sets = []
    for _ in range(2):
        x = rand(n, d).bfloat16()
        sets.append(dict(x=x, ids=torch.randint(0, v, (n,), generator=g, device=DEV, dtype=torch.int32),
                         pos=torch.randint(0, 64, (n,), generator=g, device=DEV, dtype=torch.int32),
                         wg=(rand(m, d) / 8).bfloat16(), wu=(rand(m, d) / 8).bfloat16(), dout=rand(n, m).bfloat16()))

    def run(s):
        dtable, dx, rot = torch.empty(v, d, device=DEV), torch.empty_like(s["x"]), torch.empty_like(s["x"]).view(n, 2, 64)
        dwg, dwu, dw = torch.empty(m, d, device=DEV), torch.empty(m, d, device=DEV), torch.empty(64, device=DEV)
        out, drot = torch.empty_like(s["dout"]), torch.empty_like(rot)
        for _ in range(5):
            ops.glu(out, s["x"], s["wg"], s["wu"], "silu")
            ops.glu_grad(dx, dwg, dwu, s["dout"], s["x"], s["wg"], s["wu"], "silu")
            ops.qkv_norm_rope(rot, None, None, s["x"].view(n, 2, 64), None, None, w, None, cos, sin, s["pos"])
            ops.qkv_norm_rope_grad(drot, None, None, dw, None, dx.view(n, 2, 64), None, None, s["x"].view(n, 2, 64),
                                   None, None, w, None, cos, sin, s["pos"])
            ops.embed_rows_grad(dtable, drot.view(n, d), s["ids"])
        return out, dx, dwg, dwu, rot, drot, dw, dtable

    want = [run(s) for s in sets]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                got[i] = run(sets[i])
            stream.synchronize()
        except Exception as e:  # reported by the main thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(got, want):
        for x, y in zip(a, b):
            assert torch.equal(x, y)
    assert ops.read_error() == 0


def test_first_call_may_be_captured(tmp_path):
    """A process whose first calls are made under capture: nothing in them needs an uncaptured call before."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import importlib, torch
ops = importlib.import_module("embeddinggemma2-amdkfd_b200.ops")
dev = "cuda:0"
x = torch.randn(300, 64, device=dev).bfloat16()
w = torch.randn(128, 64, device=dev).bfloat16()
d = torch.randn(300, 128, device=dev).bfloat16()
ids = torch.arange(300, device=dev, dtype=torch.int32) % 7
out, dx, dw, table = torch.empty_like(d), torch.empty_like(x), torch.empty_like(w), torch.empty(7, 64, device=dev)
q, dq, c = torch.empty(300, 1, 64, device=dev, dtype=torch.bfloat16), torch.empty(300, 1, 64, device=dev, dtype=torch.bfloat16), torch.ones(7, 32, device=dev)
dn, n = torch.empty(64, device=dev), torch.ones(64, device=dev)
def step():
    ops.glu(out, x, w, w)
    ops.glu_grad(dx, dw, None, d, x, w, w)
    ops.qkv_norm_rope(q, None, None, x.view(300, 1, 64), None, None, n, None, c, c, ids)
    ops.qkv_norm_rope_grad(dq, None, None, dn, None, q, None, None, x.view(300, 1, 64), None, None, n, None, c, c, ids)
    ops.embed_rows_grad(table, dx, ids)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    step()
graph.replay()
got = [t.clone() for t in (out, dx, dw, q, dq, dn, table)]
step()
assert all(torch.equal(a, b) for a, b in zip(got, (out, dx, dw, q, dq, dn, table)))
assert ops.read_error() == 0
print("same")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]
