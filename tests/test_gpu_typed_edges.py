"""The typed operators at the edges of what they accept, against their
definitions in 64 bits.  The references and their bounds are those of
test_gpu_typed_rows.py and test_gpu_glu.py."""
import importlib

import pytest

torch = pytest.importorskip("torch")
import test_gpu_glu as gated  # noqa: E402
import test_gpu_typed_rows as rows  # noqa: E402

pytestmark = pytest.mark.gpu

DEV, U = rows.DEV, rows.U
F32, F16, BF16 = rows.F32, rows.F16, rows.BF16


@pytest.fixture(scope="module")
def ops(eg2):
    return importlib.import_module("embeddinggemma2-amdkfd_b200.ops")


# ---------------------------------------------------------------- qkv_norm_rope
@pytest.mark.parametrize("n,hq,hkv,d", [(40, 1, 1, 128), (301, 3, 1, 64), (33, 5, 3, 96), (70, 3, 1, 512),
                                        (50, 3, 1, 34)])
@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (BF16, F32), (F16, F16)])
def test_qkv_norm_rope_grad_without_eps(ops, monkeypatch, n, hq, hkv, d, dtype, wdtype):
    """eps = 0 and head counts that do not fill the last block of heads: every row that is
    there is nonzero, so both gradients are finite and within the bounds of any eps."""
    monkeypatch.setattr(rows, "EPS", 0.0)
    q, k, v, qw, kw, cos, sin, pos, g = rows.qkv_inputs(n, hq, hkv, d, dtype, wdtype, 5 * n + d)
    gs = [rows.randn(t.shape, g, dtype) for t in (q, k, v)]
    dx = [torch.full_like(t, 7.0) for t in gs]
    dws = [torch.full((d,), 7.0, dtype=wdtype, device=DEV) for _ in range(2)]
    ops.qkv_norm_rope_grad(*dx, *dws, *gs, q, k, v, qw, kw, cos, sin, pos, 0.0)
    outs = [torch.full_like(t, 7.0) for t in gs]
    ops.qkv_norm_rope(*outs, q, k, v, qw, kw, cos, sin, pos, 0.0)
    rows.check_forward(outs, (q, k, v), (qw, kw, None), cos, sin, pos, dtype)
    keep, c, s = rows.rope_rows(cos, sin, pos)
    for kind, (x, w) in enumerate(((q, qw), (k, kw), (v, None))):
        ref, mag, terms, tmag = rows.qkv_grad_ref(x, w, c if kind < 2 else None, s, gs[kind])
        ref, mag = torch.where(keep, ref, 0.0), torch.where(keep, mag, 0.0)
        rows.assert_within(dx[kind], ref, mag * 80 * U + rows.half_unit(ref, dtype), f"dx {kind}")
        if kind < 2:
            total, bound = (torch.where(keep, t, 0.0).sum((0, 1)) for t in (terms, tmag))
            rows.assert_within(dws[kind], total,
                               bound * (n * x.shape[1] + 24) * U + rows.half_unit(total, wdtype), f"dw {kind}")


@pytest.mark.parametrize("n,d", [(5, 64), (9001, 512), (40, 34)])
def test_qkv_norm_rope_with_empty_tables(ops, n, d):
    """Tables without rows: every position is padding, so all is zero and nothing is read."""
    x = torch.full((n, 4, d), float("nan"), device=DEV)
    none = torch.empty((0, d // 2), device=DEV)
    pos = torch.arange(n, device=DEV, dtype=torch.int32) - 2
    w = torch.ones(d, device=DEV)
    parts = lambda t: (t[:, :2], t[:, 2:3], t[:, 3:])
    out, dx = torch.full_like(x, 7.0), torch.full_like(x, 7.0)
    dws = [torch.full((d,), 7.0, device=DEV) for _ in range(2)]
    ops.qkv_norm_rope(*parts(out), *parts(x), w, w, none, none, pos)
    ops.qkv_norm_rope_grad(*parts(dx), *dws, *parts(x), *parts(x), w, w, none, none, pos)
    for t in (out, dx, *dws):
        assert (t == 0).all()


@pytest.mark.parametrize("shape", [(1, 1), (1, 3), (150, 1)])
def test_qkv_norm_rope_grad_of_a_broadcast_gradient(ops, shape):
    """dout with token stride 0, head stride 0 or both: the bits of the same rows written out."""
    n, hq, hkv, d = 150, 3, 1, 64
    q, k, v, qw, kw, cos, sin, pos, g = rows.qkv_inputs(n, hq, hkv, d, BF16, F32, 12)
    gq = rows.randn((*shape, d), g, BF16).expand(n, hq, d)
    gk, gv = (rows.randn((1, hkv, d), g, BF16).expand(n, hkv, d) for _ in range(2))
    got, want = [], []
    for out, grads in ((got, (gq, gk, gv)), (want, tuple(t.contiguous() for t in (gq, gk, gv)))):
        out += [torch.full_like(t, 7.0, memory_format=torch.contiguous_format) for t in (q, k, v)]
        out += [torch.full((d,), 7.0, device=DEV) for _ in range(2)]
        ops.qkv_norm_rope_grad(*out, *grads, q, k, v, qw, kw, cos, sin, pos, 1e-6)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


# ---------------------------------------------------------------- glu
@pytest.mark.parametrize("n", [2, 14, 300])
@pytest.mark.parametrize("act", ["gelu_tanh", "silu"])
def test_glu_grad_of_large_gates(ops, n, act):
    """Gates up to 1e17, past where their cubes overflow fp32: the slope is 1 on one side and
    0 on the other.  Each projection is one product, so G and U are exact and only the
    roundings behind them are left of the bounds."""
    k, m, g = 64, 136, gated.gen(n)
    x = torch.zeros((n, k), dtype=BF16, device=DEV)
    big = torch.tensor([300.0, -300.0, 1e6, -1e6, 1e12, -1e12, 1.3e13, -1.3e13, 1e14, -1e14, 3e15, -3e15, 1e17, -1e17],
                       device=DEV)
    x[:, 0] = big[torch.arange(n, device=DEV) % 14 if n > 2 else slice(8, 10)].to(BF16)
    x[:, 1] = gated.randn((n,), g, BF16)
    wg, wu = torch.zeros((m, k), dtype=BF16, device=DEV), torch.zeros((m, k), dtype=BF16, device=DEV)
    wg[:, 0] = 1.0
    wu[:, 1] = gated.randn((m,), g, BF16)
    dout = gated.randn((n, m), g, BF16)
    got = [torch.full_like(t, 7.0) for t in (x, wg, wu)]
    ops.glu_grad(*got, dout, x, wg, wu, act)
    ref = gated.Ref(x, wg, wu, act, BF16)
    ref.eg, ref.eu = torch.zeros_like(ref.eg), torch.zeros_like(ref.eu)
    for name, a, (r, e) in zip(("dx", "dw_gate", "dw_up"), got, ref.backward(dout, BF16)):
        gated.assert_within(a, r, e, name)
    # A gate that is not a number stays one, in its row and column only.
    wg[5, 0] = float("nan")
    dw = torch.empty_like(wg)
    ops.glu_grad(None, dw, None, dout, x, wg, wu, act)
    assert dw[5, :2].isnan().all() and torch.equal(dw[:5], got[1][:5]) and torch.equal(dw[6:], got[1][6:])
    assert ops.read_error() == 0


def test_glu_grad_of_very_many_rows(ops):
    """600 million rows: a weight gradient's tile is 9.4 million K steps, near three seconds
    of products.  All rows but a few are zero, the last one not, so the sums are theirs."""
    n, k, m = 600_000_000, 8, 8
    if torch.cuda.mem_get_info()[0] < 48 << 30:
        pytest.skip("needs 48 GB")
    g = gated.gen(3)
    live = torch.tensor([0, 5, n // 2, n - 65, n - 1], device=DEV)
    x = torch.zeros((n, k), dtype=BF16, device=DEV)
    dout = torch.ones((n, m), dtype=BF16, device=DEV)
    x[live], dout[live] = gated.randn((5, k), g, BF16), gated.randn((5, m), g, BF16)
    wg, wu = gated.randn((m, k), g, BF16), gated.randn((m, k), g, BF16)
    dw = [torch.full((m, k), 7.0, device=DEV) for _ in range(2)]
    ops.glu_grad(None, *dw, dout, x, wg, wu)
    ref = gated.Ref(x[live], wg, wu, "gelu_tanh", BF16).backward(dout[live], F32)[1:]
    for name, a, (r, e) in zip(("dw_gate", "dw_up"), dw, ref):
        gated.assert_within(a, r, e, name)
    assert ops.read_error() == 0
    del x, dout
    torch.cuda.empty_cache()


def test_glu_grad_accumulates_with_frozen_weights(ops):
    """dx alone with accumulate: there is no weight gradient to be of a wrong type, and dx is written."""
    x, wg, wu, dout = gated.inputs(70, 64, 72, F16, 4)
    a, b = torch.full_like(x, 7.0), torch.full_like(x, -7.0)
    ops.glu_grad(a, None, None, dout, x, wg, wu, accumulate=True)
    ops.glu_grad(b, None, None, dout, x, wg, wu)
    assert torch.equal(a, b)
    r, e = gated.Ref(x, wg, wu, "gelu_tanh", F16).backward(dout, F32)[0]
    gated.assert_within(a, r, e)
    ops.glu_grad(None, None, None, dout, x, wg, wu, accumulate=True)  # nothing wanted


@pytest.mark.parametrize("n", [1, 2, 70, 700])
def test_glu_grad_of_a_broadcast_gradient(ops, n):
    """One row of dout for all tokens (row stride 0): the bits of the same rows written out."""
    x, wg, wu, dout = gated.inputs(n, 64, 136, BF16, n)
    row = dout[:1].expand(n, 136)
    got, want = ([torch.full_like(t, 7.0) for t in (x, wg, wu)] for _ in range(2))
    ops.glu_grad(*got, row, x, wg, wu)
    ops.glu_grad(*want, row.contiguous(), x, wg, wu)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    for a, (r, e) in zip(got, gated.Ref(x, wg, wu, "gelu_tanh", BF16).backward(row, BF16)):
        gated.assert_within(a, r, e)


@pytest.mark.parametrize("dw", [F16, F32])
def test_glu_grad_past_the_range_of_fp16(ops, dw):
    """A projection's gradient above 65504 shows: its token's row of dx and its row of dw_gate
    are not finite, never a wrong finite number, and all other rows keep their bits."""
    n, k, m, t, c = 70, 64, 136, 33, 77
    x, wg, wu, dout = gated.inputs(n, k, m, F16, 6)
    x[t], wg[c], wu[c] = 1.0, 0.25, 0.25                       # G = U = 16 there, act'(G) = 1
    got, want = ([torch.full_like(x, 7.0), *(torch.full((m, k), 7.0, dtype=dw, device=DEV) for _ in range(2))]
                 for _ in range(2))
    dout[t, c] = 0.0
    ops.glu_grad(*want, dout, x, wg, wu)
    dout[t, c] = 3900.0                                        # dG = 62400, dU = 62400: the last that fit
    ops.glu_grad(*got, dout, x, wg, wu)
    assert all(a.isfinite().all() for a in got)
    for a, (r, e) in zip(got, gated.Ref(x, wg, wu, "gelu_tanh", F16).backward(dout, dw)):
        gated.assert_within(a, r, e)
    dout[t, c] = 4200.0                                        # 67200
    ops.glu_grad(*got, dout, x, wg, wu)
    dx, dwg, dwu = got
    assert not (dx[t].isfinite().any() or dwg[c].isfinite().any() or dwu[c].isfinite().any())
    other, rest = torch.arange(n, device=DEV) != t, torch.arange(m, device=DEV) != c
    assert torch.equal(dx[other], want[0][other])
    assert torch.equal(dwg[rest], want[1][rest]) and torch.equal(dwu[rest], want[2][rest])


def test_one_tensor_for_two_gradients_is_refused(ops):
    """Queries and keys (or gate and up) that share a weight still have a gradient each."""
    n, hq, hkv, d = 20, 2, 1, 64
    q, k, v, w, _, cos, sin, pos, g = rows.qkv_inputs(n, hq, hkv, d, F32, F32, 3)
    gs = [rows.randn(t.shape, g) for t in (q, k)]
    dx, dw = [torch.full_like(t, 7.0) for t in gs], torch.full((d,), 7.0, device=DEV)
    call = lambda a, b: ops.qkv_norm_rope_grad(*dx, None, a, b, *gs, None, q, k, None, w, w, cos, sin, pos, accumulate=True)
    with pytest.raises(ValueError, match="same memory"):
        call(dw, dw)
    x, wg, _, dout = gated.inputs(20, 64, 72, BF16, 4)
    dwg = torch.full((72, 64), 7.0, device=DEV)
    with pytest.raises(ValueError, match="same memory"):
        ops.glu_grad(None, dwg, dwg, dout, x, wg, wg, accumulate=True)
    assert (dw == 7).all() and (dwg == 7).all() and all((t == 7).all() for t in dx)
    call(dw.zero_(), torch.zeros_like(dw))  # apart: taken, with the weight itself shared
    ops.glu_grad(None, dwg, torch.zeros_like(dwg), dout, x, wg, wg, accumulate=True)


def backward_with_rests(ref, dout, dw_dtype):
    """gated.Ref.backward with the inner gradients as a rounded value and its rounded rest:
    what is left is half a unit of the rest, (eps / 2)^2 of the value, or half the smallest
    subnormal."""
    fi = torch.finfo(ref.dtype)
    kept = lambda v: v.abs() * (fi.eps / 2) ** 2 * (1 + 1e-6) + fi.tiny * fi.eps / 2
    d = dout.double()
    dg, du = d * ref.u * ref.da, d * ref.a
    eg = d.abs() * (ref.da.abs() * ref.eu + ref.u.abs() * gated.D2 * ref.eg) * 1.01 + dg.abs() * gated.REL
    eg = eg + d.abs() * ref.u.abs() * 2.2 * gated.REL + kept(dg)
    eu = d.abs() * gated.D1 * ref.eg * 1.01 + du.abs() * gated.REL + kept(du)
    n, m = d.shape
    dx = dg @ ref.wg + du @ ref.wu
    ax = dg.abs() @ ref.wg.abs() + du.abs() @ ref.wu.abs()
    # Twice the terms: values and rests, the latter's absolute values far below 1 % of the former's.
    ex = eg @ ref.wg.abs() + eu @ ref.wu.abs() + ax * 1.01 * 4 * m * 2.0 ** -23 + gated.half_unit(dx, ref.dtype)
    out = [(dx, ex)]
    for v, e in ((dg, eg), (du, eu)):
        w = v.T @ ref.x
        out.append((w, e.T @ ref.x.abs() + v.abs().T @ ref.x.abs() * 1.01 * 2 * n * 2.0 ** -23
                    + gated.half_unit(w, dw_dtype)))
    return out


@pytest.mark.parametrize("n,k,m", [(1, 8, 8), (1, 512, 2048), (2, 80, 392), (3, 144, 1280), (15, 72, 264), (63, 136, 64),
                                   (64, 520, 56), (65, 64, 56), (127, 64, 32), (500, 40, 8), (1, 64, 4088), (3, 2056, 1360),
                                   (1, 136, 6520), (3, 80, 8200), (31, 8, 520), (1, 1016, 8192),
                                   (4, 88, 5616), (766, 40, 8), (11, 88, 552)])
@pytest.mark.parametrize("dtype,act,dw", [(BF16, "gelu_tanh", BF16), (F16, "silu", F32), (BF16, "silu", F32)])
def test_glu_grad_of_few_elements(ops, n, k, m, dtype, act, dw):
    """Few elements: the inner gradients keep what their roundings left, and the results are
    within their own rounding and 2^-16 or so, not two roundings, of the definition."""
    assert n * m < 6144 or n * k < 1024
    x, wg, wu, dout = gated.inputs(n, k, m, dtype, n + 2 * k + m)
    dx = torch.full((n + 3, k), 7.0, dtype=dtype, device=DEV)
    dws = [torch.full((m + 1, k), 7.0, dtype=dw, device=DEV) for _ in range(2)]
    ws = torch.full((ops.glu_grad_workspace(n, k, m) + 256,), 255, dtype=torch.uint8, device=DEV)  # NaN in any type
    ops.glu_grad(dx[:n], dws[0][:m], dws[1][:m], dout, x, wg, wu, act, workspace=ws[:-256])
    ref = backward_with_rests(gated.Ref(x, wg, wu, act, dtype), dout, dw)
    for name, got, (r, e) in zip(("dx", "dw_gate", "dw_up"), (dx[:n], dws[0][:m], dws[1][:m]), ref):
        gated.assert_within(got, r, e, name)
    assert (dx[n:] == 7).all() and all((t[m:] == 7).all() for t in dws) and (ws[-256:] == 255).all()
    for i in range(3):  # each alone: the same bits for the weights', the same bounds for dx
        part = [None] * 3
        part[i] = torch.full_like((dx[:n], dws[0][:m], dws[1][:m])[i], 7.0)
        ops.glu_grad(*part, dout, x, wg, wu, act)
        gated.assert_within(part[i], *ref[i])
        assert i == 0 or torch.equal(part[i], dws[i - 1][:m])
    assert ops.read_error() == 0


def test_glu_grad_of_few_elements_past_the_range_of_fp16(ops):
    """An inner gradient that becomes infinite leaves no rest: dw is infinite, not NaN."""
    x, wg, wu, dout = gated.inputs(3, 64, 40, F16, 6)
    x[1], wg[7], wu[7], dout[1, 7] = 1.0, 0.25, 0.25, 4200.0  # 67200
    dw = torch.empty((40, 64), device=DEV)
    ops.glu_grad(None, dw, None, dout, x, wg, wu)
    assert (dw[7] == float("inf")).all() and dw[:7].isfinite().all() and dw[8:].isfinite().all()
