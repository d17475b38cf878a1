"""The gated feed-forward projection and its gradient (include/eg2_ops.h part 3)
against their definitions in 64 bits.

Tolerances are worst-case bounds per element.  A sum of K products in fp32 is off
by at most K units of 2^-23 of the sum of the products' absolute values (an
addition in the tensor core may round or truncate); |gelu'|, |silu'| <= 1.13 and
|gelu''|, |silu''| <= 0.8 carry that through the activation; the approximate
2^x, reciprocal and the fp32 operations after them add 2^-19 relative; each
rounding to a 16-bit type adds finfo.eps / 2 relative or half its smallest
subnormal.
"""
import importlib
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
D1, D2, REL = 1.13, 0.8, 2.0 ** -19


@pytest.fixture(scope="module")
def ops(eg2):
    return importlib.import_module("embeddinggemma2-amdkfd_b200.ops")


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(shape, g, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def half_unit(ref, dtype):
    fi = torch.finfo(dtype)
    return ref.abs() * (fi.eps / 2) * (1 + 1e-6) + fi.tiny * fi.eps / 2


def assert_within(got, ref, bound, what=""):
    err = (got.double() - ref).abs()
    bad = ~(err <= bound)
    assert not bad.any(), (what, int(bad.sum()), float(err[bad].max()), float(bound[bad].min()),
                           torch.nonzero(bad)[:3].tolist())


def act64(g, act):
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * torch.sigmoid(-g))
    c = math.sqrt(2 / math.pi)
    th = torch.tanh(c * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + th), 0.5 * (1 + th) + 0.5 * g * (1 - th * th) * c * (1 + 3 * 0.044715 * g * g)


class Ref:
    """Values and error bounds of both directions, in 64 bits."""

    def __init__(self, x, wg, wu, act, dtype):
        self.x, self.wg, self.wu, self.dtype, self.act = x.double(), wg.double(), wu.double(), dtype, act
        k = x.shape[1]
        self.g, self.u = self.x @ self.wg.T, self.x @ self.wu.T
        self.eg = self.x.abs() @ self.wg.abs().T * k * 2.0 ** -23
        self.eu = self.x.abs() @ self.wu.abs().T * k * 2.0 ** -23
        self.a, self.da = act64(self.g, act)

    def forward(self):
        h = self.a * self.u
        # Second order (both factors off) is below 1 % of the first here.
        e = (D1 * self.eg * self.u.abs() + self.a.abs() * self.eu) * 1.01 + h.abs() * REL
        return h, e + half_unit(h, self.dtype)

    def backward(self, dout, dw_dtype):
        d = dout.double()
        dg, du = d * self.u * self.da, d * self.a
        eg = d.abs() * (self.da.abs() * self.eu + self.u.abs() * D2 * self.eg) * 1.01 + dg.abs() * REL
        # act' is a sum of terms of either sign: its fp32 error is relative to the terms, <= 2.2 together.
        eg = eg + d.abs() * self.u.abs() * 2.2 * REL + half_unit(dg, self.dtype)
        eu = d.abs() * D1 * self.eg * 1.01 + du.abs() * REL + half_unit(du, self.dtype)
        n, m = d.shape
        dx = dg @ self.wg + du @ self.wu
        ax = dg.abs() @ self.wg.abs() + du.abs() @ self.wu.abs()
        ex = eg @ self.wg.abs() + eu @ self.wu.abs() + ax * 1.01 * 2 * m * 2.0 ** -23 + half_unit(dx, self.dtype)
        out = [(dx, ex)]
        for v, e in ((dg, eg), (du, eu)):
            w = v.T @ self.x
            out.append((w, e.T @ self.x.abs() + v.abs().T @ self.x.abs() * 1.01 * n * 2.0 ** -23
                        + half_unit(w, dw_dtype)))
        return out


def inputs(n, k, m, dtype, seed):
    g = gen(seed)
    return (randn((n, k), g, dtype), randn((m, k), g, dtype, k ** -0.5), randn((m, k), g, dtype, k ** -0.5),
            randn((n, m), g, dtype))


SHAPES = [(1, 8, 8), (1, 512, 2048), (3, 200, 40), (8, 264, 72), (9, 8, 8), (9, 512, 2048), (64, 72, 264),
          (128, 64, 64), (129, 512, 96), (257, 136, 328), (300, 1032, 520), (513, 512, 2048), (2048, 512, 2048), (5, 40, 8200),
          (40, 264, 4104), (700, 2568, 136), (6000, 520, 2056), (9003, 1032, 264)]


@pytest.mark.parametrize("n,k,m", SHAPES)
@pytest.mark.parametrize("dtype,act", [(BF16, "gelu_tanh"), (F16, "silu")])
def test_glu(ops, n, k, m, dtype, act):
    x, wg, wu, _ = inputs(n, k, m, dtype, n + k + m)
    out = torch.full((n + 3, m), 7.0, dtype=dtype, device=DEV)
    ops.glu(out[:n], x, wg, wu, act)
    assert_within(out[:n], *Ref(x, wg, wu, act, dtype).forward())
    assert (out[n:] == 7.0).all()
    assert ops.read_error() == 0


@pytest.mark.parametrize("n,k,m", [(4, 512, 2048), (40, 512, 2048), (700, 512, 2048), (20000, 64, 512)])
def test_glu_other_types(ops, n, k, m):
    """The other pairing of type and activation, each tile width."""
    for dtype, act in ((F16, "gelu_tanh"), (BF16, "silu")):
        x, wg, wu, _ = inputs(n, k, m, dtype, n)
        out = torch.empty((n, m), dtype=dtype, device=DEV)
        ops.glu(out, x, wg, wu, act)
        assert_within(out, *Ref(x, wg, wu, act, dtype).forward())


@pytest.mark.parametrize("n,k,m", SHAPES)
@pytest.mark.parametrize("dtype,act,dw", [(BF16, "gelu_tanh", BF16), (F16, "silu", F32)])
def test_glu_grad(ops, n, k, m, dtype, act, dw):
    x, wg, wu, dout = inputs(n, k, m, dtype, 2 * n + k + m)
    dx = torch.full((n + 3, k), 7.0, dtype=dtype, device=DEV)
    dwg, dwu = (torch.full((m + 1, k), 7.0, dtype=dw, device=DEV) for _ in range(2))
    ops.glu_grad(dx[:n], dwg[:m], dwu[:m], dout, x, wg, wu, act)
    ref = Ref(x, wg, wu, act, dtype).backward(dout, dw)
    for name, got, (r, e) in zip(("dx", "dw_gate", "dw_up"), (dx[:n], dwg[:m], dwu[:m]), ref):
        assert_within(got, r, e, name)
    assert (dx[n:] == 7.0).all() and (dwg[m:] == 7.0).all() and (dwu[m:] == 7.0).all()
    assert ops.read_error() == 0


@pytest.mark.parametrize("dtype,act", [(F16, "gelu_tanh"), (BF16, "silu")])
def test_glu_grad_other_types_and_parts(ops, dtype, act):
    """The other pairings; each gradient alone has the same bits as all together."""
    n, k, m = 777, 264, 512
    x, wg, wu, dout = inputs(n, k, m, dtype, 5)
    dx, dwg, dwu = (torch.empty_like(t) for t in (x, wg, wu))
    ops.glu_grad(dx, dwg, dwu, dout, x, wg, wu, act)
    for got, (r, e) in zip((dx, dwg, dwu), Ref(x, wg, wu, act, dtype).backward(dout, dtype)):
        assert_within(got, r, e)
    for i, full in enumerate((dx, dwg, dwu)):
        part = [None] * 3
        part[i] = torch.full_like(full, 7.0)
        ops.glu_grad(*part, dout, x, wg, wu, act)
        assert torch.equal(part[i], full)
    again = [torch.empty_like(t) for t in (dx, dwg, dwu)]
    ops.glu_grad(*again, dout, x, wg, wu, act)
    for a, b in zip(again, (dx, dwg, dwu)):
        assert torch.equal(a, b)
    ops.glu_grad(None, None, None, dout, x, wg, wu, act)  # nothing wanted


def test_glu_grad_accumulates(ops):
    n, k, m = 300, 64, 136
    x, wg, wu, dout = inputs(n, k, m, BF16, 6)
    a, b = (torch.empty((m, k), device=DEV) for _ in range(2))
    ops.glu_grad(None, a, b, dout, x, wg, wu)
    old = randn((m, k), gen(7), F32)
    c, d = old.clone(), torch.zeros((m, k), device=DEV)
    ops.glu_grad(None, c, d, dout, x, wg, wu, accumulate=True)
    assert torch.equal(d, b) and torch.equal(c, old + a)
    # No tokens: zero, or as it was.
    e = lambda t: t[:0]
    ops.glu_grad(e(x), c, None, e(dout), e(x), wg, wu, accumulate=True)
    assert torch.equal(c, old + a)
    ops.glu_grad(e(x), c, None, e(dout), e(x), wg, wu)
    assert (c == 0).all()
    ops.glu(e(dout), e(x), wg, wu)


def test_glu_grad_against_differences(ops):
    """<dx, e> and <dW, e> against central differences of the operator in 64 bits."""
    n, k, m = 40, 64, 72
    x, wg, wu, dout = inputs(n, k, m, F16, 8)
    dx, dwg, dwu = torch.empty_like(x), torch.empty((m, k), device=DEV), torch.empty((m, k), device=DEV)
    ops.glu_grad(dx, dwg, dwu, dout, x, wg, wu)
    bounds = [e for _, e in Ref(x, wg, wu, "gelu_tanh", F16).backward(dout, F32)]
    args = [t.double() for t in (x, wg, wu)]

    def loss(x, wg, wu):
        return (act64(x @ wg.T, "gelu_tanh")[0] * (x @ wu.T) * dout.double()).sum()

    for i, grad in enumerate((dx, dwg, dwu)):
        e, h = randn(grad.shape, gen(20 + i), F32).double(), 1e-5
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + h * e, args[i] - h * e
        num = (loss(*up) - loss(*down)) / (2 * h)
        terms = (grad.double() * e).abs().sum()
        # The gradients' own bounds along e; truncation and cancellation below 1e-6 of the terms.
        assert abs(num - (grad.double() * e).sum()) <= (bounds[i] * e.abs()).sum() + 1e-6 * terms


def test_glu_strides_and_extremes(ops):
    n, k, m = 70, 64, 128
    g = gen(9)
    x = randn((n, k + 8), g, BF16)[:, :k]
    w = randn((m, 2, k), g, BF16, 0.125)  # gate and up rows interleaved
    whole = torch.full((n, m + 16), 7.0, dtype=BF16, device=DEV)
    ops.glu(whole[:, 8:8 + m], x, w[:, 0], w[:, 1])
    assert_within(whole[:, 8:8 + m], *Ref(x, w[:, 0], w[:, 1], "gelu_tanh", BF16).forward())
    assert (whole[:, :8] == 7).all() and (whole[:, 8 + m:] == 7).all()
    # Far out on both sides of the activation: g or 0, never NaN.
    for rows in (2, 70):
        xe = torch.zeros((rows, k), dtype=BF16, device=DEV)
        xe[0, 0], xe[1, 0] = 300.0, -300.0
        we = torch.zeros((m, k), dtype=BF16, device=DEV)
        we[:, 0] = 1.0
        for act in ("gelu_tanh", "silu"):
            out = torch.empty((rows, m), dtype=BF16, device=DEV)
            ops.glu(out, xe, we, we, act)
            assert (out[0] == 90112).all() and (out[1].abs() == 0).all() and (out[2:] == 0).all()
            dx, dw = torch.empty_like(xe), torch.empty_like(we)
            ops.glu_grad(dx, dw, None, torch.ones_like(out), xe, we, we, act)
            assert dx.isfinite().all() and dw.isfinite().all()
    # A row of NaN or infinity stays in its row.
    x2 = x.clone()
    x2[5], x2[60] = float("nan"), float("inf")
    out = torch.empty((n, m), dtype=BF16, device=DEV)
    ops.glu(out, x2, w[:, 0], w[:, 1])
    keep = torch.ones(n, dtype=torch.bool, device=DEV)
    keep[[5, 60]] = False
    assert out[5].isnan().all() and torch.equal(out[keep], whole[:, 8:8 + m][keep])


def test_glu_graph_replay_and_side_stream(ops):
    n, k, m = 300, 512, 256
    x, wg, wu, dout = inputs(n, k, m, BF16, 10)
    out, dx = torch.empty_like(dout), torch.empty_like(x)
    dwg, dwu = torch.empty((m, k), device=DEV), torch.empty((m, k), device=DEV)

    def step():
        ops.glu(out, x, wg, wu)
        ops.glu_grad(dx, dwg, dwu, out, x, wg, wu)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    x.copy_(randn((n, k), gen(11), BF16))
    graph.replay()
    got = [t.clone() for t in (out, dx, dwg, dwu)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for t in (out, dx, dwg, dwu):
            t.zero_()
        step()
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(got, (out, dx, dwg, dwu)):
        assert torch.equal(a, b)
    assert ops.read_error() == 0


def test_glu_refusals(ops):
    x, wg, wu, dout = inputs(16, 64, 32, BF16, 12)
    out = torch.full_like(dout, 7.0)
    for bad in (lambda: ops.glu(out, x, wg, wu, "relu"), lambda: ops.glu(out, x.float(), wg, wu),
                lambda: ops.glu(out, x, wg.half(), wu), lambda: ops.glu(out, x, wg, wu[:16]),
                lambda: ops.glu(out[:8], x, wg, wu), lambda: ops.glu(out, x[:, :60], wg[:, :60], wu[:, :60]),
                lambda: ops.glu(out[:, :28], x, wg[:28], wu[:28]), lambda: ops.glu(out.float(), x, wg, wu),
                lambda: ops.glu(out, x, wg.t().contiguous().t(), wu), lambda: ops.glu(out, x, wg.cpu(), wu),
                lambda: ops.glu_grad(None, torch.empty_like(wg), None, dout, x, wg, wu, accumulate=True),
                lambda: ops.glu_grad(None, wg.float(), wu, dout, x, wg, wu),
                lambda: ops.glu_grad(None, wg.half(), None, dout, x, wg, wu),
                lambda: ops.glu_grad(None, wg, None, dout, x, wg, wu, workspace=torch.empty(64, device=DEV))):
        with pytest.raises(ValueError):
            bad()
    flat = torch.zeros(17 * 64, dtype=BF16, device=DEV)
    with pytest.raises(RuntimeError):  # rows not 16-byte aligned
        ops.glu(out, flat[1:1 + 16 * 64].view(16, 64), wg, wu)
    with pytest.raises(RuntimeError):  # a row pitch that is not a multiple of 16 bytes
        ops.glu(out, torch.as_strided(flat, (16, 64), (65, 1)), wg, wu)
    with pytest.raises(RuntimeError):  # output rows on top of one another
        ops.glu(out[:1].expand(16, 32), x, wg, wu)
    assert (out == 7.0).all()
