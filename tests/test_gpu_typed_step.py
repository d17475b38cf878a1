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
