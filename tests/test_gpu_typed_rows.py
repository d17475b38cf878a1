"""The typed row operators (include/eg2_ops.h part 3) against their definitions
in 64 bits: embedding lookup and gradient, per-head norm with rotation and
gradient.

Tolerances are worst-case bounds, derived per element: u = 2^-24 per fp32
operation on the absolute values that enter it, half a unit of the output type
(finfo.eps / 2, relative) for the last rounding, and half the smallest
subnormal of that type where the result underflows.
"""
import importlib
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ops(eg2):
    return importlib.import_module("embeddinggemma2-amdkfd_b200.ops")


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(shape, g, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def half_unit(ref, dtype):
    """The last rounding's bound: half a unit, at least half the smallest subnormal."""
    fi = torch.finfo(dtype)
    return ref.abs() * (fi.eps / 2) * (1 + 1e-6) + fi.tiny * fi.eps / 2


def assert_within(got, ref, bound, what=""):
    err = (got.double() - ref).abs()
    bad = ~(err <= bound)
    assert not bad.any(), (what, int(bad.sum()), float(err[bad].max()), float(bound[bad].min()),
                           torch.nonzero(bad)[:3].tolist())


# ---------------------------------------------------------------- embed_rows
def embed_ref(table, ids, scale):
    v = table.shape[0]
    ok = (ids >= 0) & (ids < v)
    rows = table.double()[ids.clamp(0, max(v - 1, 0)).long()] * scale
    return torch.where(ok[:, None], rows, 0.0)


def make_ids(n, v, g, pad=0.1):
    ids = torch.randint(0, v, (n,), generator=g, device=DEV, dtype=torch.int32)
    r = torch.rand(n, generator=g, device=DEV)
    ids = torch.where(r < pad / 2, torch.full_like(ids, -1), ids)
    return torch.where(r > 1 - pad / 2, torch.full_like(ids, v), ids)  # one behind the table


@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (1, 37, 8), (7, 100, 512), (33, 50, 250), (300, 1000, 96),
                                   (17000, 777, 40), (16500, 300, 7), (5, 9, 2056)])
@pytest.mark.parametrize("ti,to", [(F32, F32), (BF16, BF16), (F16, F32), (F32, F16), (BF16, F16)])
def test_embed_rows(ops, n, v, d, ti, to):
    g = gen(n + v + d)
    table, ids = randn((v, d), g, ti), make_ids(n, v, g)
    out = torch.full((n + 2, d), 7.0, dtype=to, device=DEV)
    scale = math.sqrt(512)
    ops.embed_rows(out[:n], table, ids, scale)
    ref = embed_ref(table, ids, torch.tensor(scale, dtype=F32).item())
    assert_within(out[:n], ref, half_unit(ref, to) + ref.abs() * U)
    assert (out[n:] == 7.0).all()  # rows behind the last token stay


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("in_off,in_pad,out_off,out_pad", [(0, 8, 0, 16), (1, 7, 0, 0), (0, 0, 3, 5), (8, 16, 8, 1)])
def test_embed_rows_strides_and_alignment(ops, dtype, in_off, in_pad, out_off, out_pad):
    n, v, d, g = 70, 90, 128, gen(3)
    table = randn((v, d + in_off + in_pad), g, dtype)[:, in_off:in_off + d]
    whole = torch.full((n, d + out_off + out_pad), 7.0, dtype=dtype, device=DEV)
    out, ids = whole[:, out_off:out_off + d], make_ids(n, v, g)
    ops.embed_rows(out, table, ids, 0.5)
    ref = embed_ref(table, ids, 0.5)
    assert_within(out, ref, half_unit(ref, dtype) + ref.abs() * U)
    rest = torch.cat([whole[:, :out_off], whole[:, out_off + d:]], 1)
    assert (rest == 7.0).all()


def test_embed_rows_empty_and_nonfinite(ops):
    table = torch.tensor([[1.0, float("inf")], [float("nan"), -2.0]], device=DEV)
    ops.embed_rows(torch.empty((0, 2), device=DEV), table, torch.empty(0, dtype=torch.int32, device=DEV))
    out = torch.empty((3, 2), device=DEV)
    ops.embed_rows(out, table, torch.tensor([1, -1, 0], dtype=torch.int32, device=DEV), 2.0)
    assert out[0, 0].isnan() and out[0, 1] == -4.0 and (out[1] == 0).all() and out[2, 1] == float("inf")
    # A table without rows: every id is padding.
    ops.embed_rows(out, torch.empty((0, 2), device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV))
    assert (out == 0).all()


def test_embed_rows_offsets_past_32_bits(ops):
    """More than 2^31 elements (and 2^32 bytes) in the table and in its gradient."""
    v, d = 2_200_000, 1024
    table = torch.empty((v, d), dtype=F16, device=DEV)
    rows = [0, 2_097_151, 2_097_152, v - 1]
    for i, r in enumerate(rows):
        table[r] = float(i + 1)
    ids = torch.tensor(rows, dtype=torch.int32, device=DEV)
    out = torch.empty((4, d), dtype=F16, device=DEV)
    ops.embed_rows(out, table, ids)
    assert (out == torch.arange(1, 5, device=DEV)[:, None]).all()
    table.fill_(3.0)
    ops.embed_rows_grad(table, out, torch.tensor([rows[0], rows[3], rows[3], rows[2]], dtype=torch.int32, device=DEV))
    want = {rows[0]: 1.0, rows[3]: 5.0, rows[2]: 4.0}
    for r, x in want.items():
        assert (table[r] == x).all(), r
    assert int(torch.count_nonzero(table)) == 3 * d


# ---------------------------------------------------------------- embed_rows_grad
def embed_grad_ref(v, dout, ids):
    """(sums, sums of absolute values, counts) per table row."""
    ok = (ids >= 0) & (ids < v)
    idx, rows = ids[ok].long(), dout[ok].double()
    z = lambda: torch.zeros((v, dout.shape[1]), dtype=torch.float64, device=DEV)
    count = torch.zeros(v, dtype=torch.float64, device=DEV).index_add_(0, idx, torch.ones_like(idx, dtype=torch.float64))
    return z().index_add_(0, idx, rows), z().index_add_(0, idx, rows.abs()), count


def check_embed_grad(ops, v, dout, ids, dtype, scale=1.0, accumulate=False, dtable=None):
    d = dout.shape[1]
    if dtable is None:
        dtable = torch.full((v, d), 3.0, dtype=dtype, device=DEV)
    old = dtable.double()
    ops.embed_rows_grad(dtable, dout, ids, scale, accumulate)
    s, a, c = embed_grad_ref(v, dout, ids)
    ref = s * scale + (old if accumulate else 0.0)
    # c - 1 additions (any order), the scale, and the addition to what was there.
    bound = a * abs(scale) * (c[:, None] + 2) * U * 1.01 + half_unit(ref, dtype)
    if accumulate:
        bound = bound + (ref.abs() + old.abs()) * U
        bound[c == 0] = 0.0
    assert_within(dtable, ref, bound)
    return dtable


@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (1, 500, 512), (8, 3, 64), (9, 5000, 250), (700, 11, 264),
                                   (2048, 262144, 16), (2049, 1023, 40), (5000, 1024, 7), (40000, 3000, 72)])
@pytest.mark.parametrize("tg,tw", [(F32, F32), (BF16, BF16), (F16, F32), (F32, BF16)])
def test_embed_rows_grad(ops, n, v, d, tg, tw):
    g = gen(n * 3 + v + d)
    check_embed_grad(ops, v, randn((n, d), g, tg), make_ids(n, v, g), tw, 0.75)


@pytest.mark.parametrize("n,hot", [(300, 300), (33000, 33000), (33000, 20000), (4100, 2051)])
def test_embed_rows_grad_hot_token(ops, n, hot):
    """One id on most of the tokens: its run goes over many chunks."""
    g = gen(n + hot)
    ids = torch.randint(0, 50, (n,), generator=g, device=DEV, dtype=torch.int32)
    ids[torch.randperm(n, generator=g, device=DEV)[:hot]] = 17
    check_embed_grad(ops, 50, randn((n, 48), g, BF16), ids, F32)


def test_embed_rows_grad_all_padding_reads_nothing(ops):
    dout = torch.full((50, 16), float("nan"), device=DEV)
    ids = torch.full((50,), -1, dtype=torch.int32, device=DEV)
    dtable = torch.full((20, 16), 3.0, device=DEV)
    ops.embed_rows_grad(dtable, dout, ids)
    assert (dtable == 0).all()
    ids[7], dout[7] = 4, 2.0  # one live row among rows of NaN
    ops.embed_rows_grad(dtable, dout, ids, 0.5)
    assert (dtable[4] == 1).all() and int(torch.count_nonzero(dtable)) == 16


@pytest.mark.parametrize("v", [1023, 1024, 1 << 20, (1 << 20) + 5])
def test_embed_rows_grad_digit_borders(ops, v):
    """Vocabularies at the borders of one, two and three passes; the padding key is v."""
    g = gen(v)
    ids = make_ids(4000, v, g)
    ids[:6] = torch.tensor([0, v - 1, v - 1, 0, v, v // 2], dtype=torch.int32, device=DEV)
    check_embed_grad(ops, v, randn((4000, 8), g), ids, F32)


def test_embed_rows_grad_many_subtiles(ops):
    """More tokens than 128 tiles hold: a CTA sorts several stretches in order."""
    g, n = gen(8), 600_001
    check_embed_grad(ops, 30_000, randn((n, 8), g, BF16), make_ids(n, 30_000, g), F32)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_embed_rows_grad_accumulates(ops, dtype):
    g = gen(11)
    dtable = randn((400, 40), g, dtype)
    dtable[399] = float("nan")  # a row that does not occur is not touched
    ids = torch.randint(0, 399, (900,), generator=g, device=DEV, dtype=torch.int32)
    keep = dtable.clone()
    ops.embed_rows_grad(dtable, randn((900, 40), g), ids, accumulate=True)
    assert dtable[399].isnan().all()
    dtable[:399] = keep[:399]
    check_embed_grad(ops, 399, randn((900, 40), g), ids, dtype, 0.5, True, dtable[:399])


def test_embed_rows_grad_strides(ops):
    g = gen(12)
    for off, d in ((0, 64), (3, 30), (8, 128)):
        whole = torch.full((90, d + 24), 7.0, dtype=BF16, device=DEV)
        dout = randn((500, d + 16), g, BF16)[:, off:off + d]
        check_embed_grad(ops, 90, dout, make_ids(500, 90, g), BF16, 1.0, False, whole[:, off:off + d])
        assert (torch.cat([whole[:, :off], whole[:, off + d:]], 1) == 7.0).all()
    # A broadcast gradient: every token has the same row.
    row = randn((1, 64), g)
    check_embed_grad(ops, 90, row.expand(500, 64), make_ids(500, 90, g), F32)


def test_embed_rows_grad_empty(ops):
    ids, dout = torch.empty(0, dtype=torch.int32, device=DEV), torch.empty((0, 6), device=DEV)
    whole = torch.full((5, 9), 3.0, device=DEV)
    ops.embed_rows_grad(whole[:, :6], dout, ids, accumulate=True)
    assert (whole == 3).all()
    ops.embed_rows_grad(whole[:, :6], dout, ids)
    assert (whole[:, :6] == 0).all() and (whole[:, 6:] == 3).all()


def test_embed_rows_grad_same_bits_each_time(ops):
    g = gen(13)
    dout, ids = randn((30000, 136), g, BF16), make_ids(30000, 500, g)
    a, b = (torch.empty((500, 136), device=DEV) for _ in range(2))
    ops.embed_rows_grad(a, dout, ids)
    for _ in range(3):
        ops.embed_rows_grad(b, dout, ids)
        assert torch.equal(a, b)
    # Tokens of other ids in between do not change a row's bits.
    more = torch.randint(500, 900, (30000,), generator=g, device=DEV, dtype=torch.int32)
    both = torch.stack([ids, more], 1).flatten()
    both[both == 500] = 901  # the id behind the first table is padding there
    c = torch.empty((900, 136), device=DEV)
    ops.embed_rows_grad(c, dout.repeat_interleave(2, 0), both)
    s, ab, n = embed_grad_ref(500, dout, ids)
    assert_within(c[:500], s, ab * (n[:, None] + 2) * U * 1.01 + half_unit(s, F32))


# ---------------------------------------------------------------- qkv_norm_rope
EPS = 1e-6


def tables(d, positions):
    i = torch.arange(d // 2, dtype=torch.float64, device=DEV)
    a = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * 10000.0 ** (-2.0 * i / d)
    return torch.cos(a).float(), torch.sin(a).float()


def rotate(y, c, s):
    a, b = y.chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def unrotate(g, c, s):
    a, b = g.chunk(2, -1)
    return torch.cat([a * c + b * s, b * c - a * s], -1)


def qkv_ref(x, w, c, s):
    """Output in 64 bits and the magnitude that enters it (|y_i| + |y_pair|)."""
    x = x.double()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    if w is not None:
        y = y * w.double()
    if c is None:
        return y, y.abs()
    a, b = y.abs().chunk(2, -1)
    return rotate(y, c, s), torch.cat([a + b, a + b], -1)


def qkv_grad_ref(x, w, c, s, g):
    """dx, dw and the magnitudes of their terms, in 64 bits."""
    x, g = x.double(), g.double()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    mag = g.abs()
    if c is not None:
        g = unrotate(g, c, s)
        a, b = mag.chunk(2, -1)
        mag = torch.cat([a + b, a + b], -1)
    terms, term_mag = g * x * r, mag * x.abs() * r
    if w is not None:
        g, mag = g * w.double(), mag * w.double().abs()
    dx = r * (g - x * r * r * (g * x).mean(-1, keepdim=True))
    dx_mag = r * (mag + x.abs() * r * r * (mag * x.abs()).mean(-1, keepdim=True))
    return dx, dx_mag, terms, term_mag


def qkv_inputs(n, hq, hkv, d, dtype, wdtype, seed, pad=0.1, positions=64):
    g = gen(seed)
    x = randn((n, hq + 2 * hkv, d), g, dtype, 2.0)
    pos = torch.randint(0, positions, (n,), generator=g, device=DEV, dtype=torch.int32)
    r = torch.rand(n, generator=g, device=DEV)
    pos = torch.where(r < pad / 2, torch.full_like(pos, -1), pos)
    pos = torch.where(r > 1 - pad / 2, torch.full_like(pos, positions), pos)
    cos, sin = tables(d, positions)
    qw, kw = (randn((d,), g, F32, 0.2).add(1.0).to(wdtype) for _ in range(2))
    return x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], qw, kw, cos, sin, pos, g


def rope_rows(cos, sin, pos):
    keep = (pos >= 0) & (pos < cos.shape[0])
    p = torch.where(keep, pos, 0).long()
    return keep[:, None, None], cos.double()[p][:, None], sin.double()[p][:, None]


def check_forward(outs, ins, weights, cos, sin, pos, dtype):
    keep, c, s = rope_rows(cos, sin, pos)
    for kind, (o, x) in enumerate(zip(outs, ins)):
        if x is None:
            continue
        ref, mag = qkv_ref(x, weights[kind], c if kind < 2 else None, s)
        ref, mag = torch.where(keep, ref, 0.0), torch.where(keep, mag, 0.0)
        # The mean of d <= 512 squares: at most 16 in a lane, 5 shuffles; r, two products, the rotation.
        assert_within(o, ref, mag * 32 * U + half_unit(ref, dtype), f"kind {kind}")


SHAPES = [(1, 4, 2, 256), (1, 1, 1, 2), (3, 4, 1, 512), (33, 3, 3, 48), (70, 5, 1, 80), (129, 8, 2, 128),
          (65, 2, 1, 64), (40, 6, 2, 96), (31, 2, 2, 192), (50, 3, 1, 34), (2011, 4, 2, 256), (4099, 10, 2, 32)]


# Rows enough for the streaming form of the forward pass in every type: whole and
# partial halves, odd head counts, the widest rows, and more heads than groups of lanes.
LARGE = [(9001, 2, 1, 512), (12007, 8, 2, 128), (16001, 6, 2, 96), (30011, 3, 1, 48), (9001, 5, 1, 80),
         (21, 6000, 1, 256)]


@pytest.mark.parametrize("n,hq,hkv,d", SHAPES + LARGE)
@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (BF16, F32), (F16, F16), (BF16, BF16)])
def test_qkv_norm_rope(ops, n, hq, hkv, d, dtype, wdtype):
    q, k, v, qw, kw, cos, sin, pos, g = qkv_inputs(n, hq, hkv, d, dtype, wdtype, n + d)
    outs = [torch.full_like(t, 7.0, memory_format=torch.contiguous_format) for t in (q, k, v)]
    ops.qkv_norm_rope(*outs, q, k, v, qw, kw, cos, sin, pos, EPS)
    check_forward(outs, (q, k, v), (qw, kw, None), cos, sin, pos, dtype)


def test_qkv_norm_rope_parts_layouts_and_in_place(ops):
    n, hq, hkv, d = 77, 6, 2, 64
    q, k, v, qw, kw, cos, sin, pos, g = qkv_inputs(n, hq, hkv, d, BF16, F32, 5)
    # Queries only, without a weight; keys and values only.
    o = torch.empty((n, hq, d), dtype=BF16, device=DEV)
    ops.qkv_norm_rope(o, None, None, q, None, None, None, None, cos, sin, pos, EPS)
    check_forward((o, None, None), (q, None, None), (None, None, None), cos, sin, pos, BF16)
    ok, ov = (torch.empty((n, hkv, d), dtype=BF16, device=DEV) for _ in range(2))
    ops.qkv_norm_rope(None, ok, ov, None, k, v, None, kw, cos, sin, pos, EPS)
    check_forward((None, ok, ov), (None, k, v), (None, kw, None), cos, sin, pos, BF16)
    # Head-major outputs, rows not 16-byte aligned (odd strides and offset).
    oh = torch.full((hq, n, d), 7.0, dtype=BF16, device=DEV).transpose(0, 1)
    odd = torch.full((n, hkv, d + 3), 7.0, dtype=BF16, device=DEV)
    ops.qkv_norm_rope(oh, odd[..., 1:1 + d], None, q, k, None, qw, kw, cos, sin, pos, EPS)
    check_forward((oh, odd[..., 1:1 + d], None), (q, k, None), (qw, kw, None), cos, sin, pos, BF16)
    assert (odd[..., 0] == 7).all() and (odd[..., 1 + d:] == 7).all()
    # In place: the same values as out of place.
    fused = torch.cat([q, k, v], 1)
    ref = [torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v)]
    ops.qkv_norm_rope(*ref, q, k, v, qw, kw, cos, sin, pos, EPS)
    views = fused[:, :hq], fused[:, hq:hq + hkv], fused[:, hq + hkv:]
    ops.qkv_norm_rope(*views, *views, qw, kw, cos, sin, pos, EPS)
    for a, b in zip(views, ref):
        assert torch.equal(a, b)


def test_qkv_norm_rope_extremes(ops):
    """Rows of zeros, of large and tiny values; a row of NaN behind a padding position is not read."""
    d = 64
    x = torch.zeros((4, 1, d), device=DEV)
    x[1], x[2], x[3] = 1e18, 1e-18, float("nan")
    pos = torch.tensor([0, 1, 2, -1], dtype=torch.int32, device=DEV)
    cos, sin = tables(d, 4)
    o = torch.full_like(x, 7.0)
    ops.qkv_norm_rope(o, None, None, x, None, None, None, None, cos, sin, pos, EPS)
    check_forward((o, None, None), (torch.where(x.isnan(), 0.0, x), None, None), (None,) * 3, cos, sin, pos, F32)
    assert (o[0] == 0).all() and (o[3] == 0).all()
    dx, dw, g = torch.full_like(x, 7.0), torch.empty(d, device=DEV), torch.ones_like(x)
    w = torch.ones(d, device=DEV)
    g[3] = float("nan")
    ops.qkv_norm_rope_grad(dx, None, None, dw, None, g, None, None, x, None, None, w, None, cos, sin, pos, EPS)
    assert (dx[3] == 0).all() and dx.isfinite().all() and dw.isfinite().all()


@pytest.mark.parametrize("n,hq,hkv,d", SHAPES + LARGE)
@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (BF16, F32), (F16, F16), (BF16, BF16)])
def test_qkv_norm_rope_grad(ops, n, hq, hkv, d, dtype, wdtype):
    q, k, v, qw, kw, cos, sin, pos, g = qkv_inputs(n, hq, hkv, d, dtype, wdtype, 3 * n + d)
    gs = [randn(t.shape, g, dtype) for t in (q, k, v)]
    dx = [torch.full_like(t, 7.0) for t in gs]
    dws = [torch.full((d,), 7.0, dtype=wdtype, device=DEV) for _ in range(2)]
    ops.qkv_norm_rope_grad(*dx, *dws, *gs, q, k, v, qw, kw, cos, sin, pos, EPS)
    keep, c, s = rope_rows(cos, sin, pos)
    for kind, (x, w) in enumerate(((q, qw), (k, kw), (v, None))):
        ref, mag, terms, tmag = qkv_grad_ref(x, w, c if kind < 2 else None, s, gs[kind])
        ref, mag = torch.where(keep, ref, 0.0), torch.where(keep, mag, 0.0)
        # As forward, with a second mean of the same depth and six more operations.
        assert_within(dx[kind], ref, mag * 80 * U + half_unit(ref, dtype), f"dx {kind}")
        if kind < 2:
            total, bound = (torch.where(keep, t, 0.0).sum((0, 1)) for t in (terms, tmag))
            # Every addition of the rows, and 24 operations in a term.
            rows = n * x.shape[1]
            assert_within(dws[kind], total, bound * (rows + 24) * U + half_unit(total, wdtype), f"dw {kind}")


def test_qkv_norm_rope_grad_against_differences(ops):
    """<dx, e> and <dw, e> against central differences of the operator in 64 bits."""
    n, hq, hkv, d = 6, 2, 1, 32
    q, k, v, qw, kw, cos, sin, pos, g = qkv_inputs(n, hq, hkv, d, F32, F32, 21)
    gs = [randn(t.shape, g) for t in (q, k, v)]
    dx = [torch.empty_like(t) for t in gs]
    dws = [torch.empty(d, device=DEV) for _ in range(2)]
    ops.qkv_norm_rope_grad(*dx, *dws, *gs, q, k, v, qw, kw, cos, sin, pos, EPS)
    keep, c, s = rope_rows(cos, sin, pos)

    def loss(x, w, kind):
        y, _ = qkv_ref(x, w, c if kind < 2 else None, s)
        return (torch.where(keep, y, 0.0) * gs[kind].double()).sum()

    h = 1e-5
    for kind, (x, w) in enumerate(((q, qw), (k, kw), (v, None))):
        e = randn(x.shape, g).double()
        num = (loss(x.double() + h * e, w, kind) - loss(x.double() - h * e, w, kind)) / (2 * h)
        # Truncation h^2 |f'''| and cancellation 2^-53 |f| / h stay under 1e-7 of the terms' sum.
        scale = (dx[kind].double() * e).abs().sum()
        assert abs(num - (dx[kind].double() * e).sum()) <= scale * (1e-7 + 80 * U)
        if kind < 2:
            e = randn((d,), g).double()
            num = (loss(x, w.double() + h * e, kind) - loss(x, w.double() - h * e, kind)) / (2 * h)
            scale = (dws[kind].double() * e).abs().sum()
            assert abs(num - (dws[kind].double() * e).sum()) <= scale * (1e-7 + 200 * U)


def test_qkv_norm_rope_grad_options(ops):
    n, hq, hkv, d = 150, 4, 2, 64
    q, k, v, qw, kw, cos, sin, pos, g = qkv_inputs(n, hq, hkv, d, BF16, F32, 9)
    gs = [randn(t.shape, g, BF16) for t in (q, k, v)]
    dx = [torch.empty_like(t) for t in gs]
    dws = [torch.empty(d, device=DEV) for _ in range(2)]
    ops.qkv_norm_rope_grad(*dx, *dws, *gs, q, k, v, qw, kw, cos, sin, pos, EPS)
    # Again: the same bits.  Accumulated on top: twice the gradient exactly (a power of two).
    again = [w.clone() for w in dws]
    ops.qkv_norm_rope_grad(*dx, *again, *gs, q, k, v, qw, kw, cos, sin, pos, EPS, accumulate=True)
    for a, w in zip(again, dws):
        assert torch.equal(a, 2 * w)
    # Without weight gradients, and in place of the outputs' gradients.
    own = [t.clone() for t in gs]
    ops.qkv_norm_rope_grad(*own, None, None, *own, q, k, v, qw, kw, cos, sin, pos, EPS)
    for a, b in zip(own, dx):
        assert torch.equal(a, b)
    # Only the keys' weight; queries left out.
    one = torch.empty(d, device=DEV)
    ops.qkv_norm_rope_grad(None, dx[1], None, None, one, None, gs[1], None, None, k, None, None, kw, cos, sin, pos, EPS)
    # The rows are spread over other CTAs, so the sum's order differs: the bound of any order.
    assert (one - dws[1]).abs().max() <= 2 * (n * hkv + 24) * U * dws[1].abs().max() * n
    # No tokens: the weights' gradients are zero, or stay.
    e = lambda t: t[:0]
    ops.qkv_norm_rope_grad(e(dx[0]), None, None, one, None, e(gs[0]), None, None, e(q), None, None, qw, None, cos, sin,
                           e(pos), EPS)
    assert (one == 0).all()


# ---------------------------------------------------------------- as programs use them
def test_graph_replay_and_side_stream(ops):
    """Captured once, replayed on new inputs; and the same on a second stream."""
    g = gen(31)
    n, v, d, hq, hkv, hd = 200, 1000, 192, 2, 1, 64
    table, ids = randn((v, d), g, BF16), make_ids(n, v, g)
    x, dtable = torch.empty((n, d), dtype=BF16, device=DEV), torch.empty((v, d), device=DEV)
    cos, sin = tables(hd, 256)
    pos = torch.arange(n, device=DEV, dtype=torch.int32)
    w = torch.ones(hd, device=DEV)
    dqw, dkw = torch.empty(hd, device=DEV), torch.empty(hd, device=DEV)
    y, dx = torch.empty((n, 3, hd), dtype=BF16, device=DEV), torch.empty((n, 3, hd), dtype=BF16, device=DEV)

    def step():
        ops.embed_rows(x, table, ids, 2.0)
        heads = x.view(n, 3, hd)
        q, k = heads[:, :hq], heads[:, hq:]
        ops.qkv_norm_rope(y[:, :hq], y[:, hq:], None, q, k, None, w, w, cos, sin, pos)
        ops.qkv_norm_rope_grad(dx[:, :hq], dx[:, hq:], None, dqw, dkw, y[:, :hq], y[:, hq:], None, q, k, None, w, w,
                               cos, sin, pos)
        ops.embed_rows_grad(dtable, dx.view(n, d), ids, 2.0)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (1, 2):
        table.copy_(randn((v, d), gen(seed), BF16))
        ids.copy_(make_ids(n, v, gen(seed + 10)))
        graph.replay()
        got = [t.clone() for t in (x, y, dx, dqw, dkw, dtable)]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for t in (x, y, dx, dqw, dkw, dtable):
                t.zero_()
            step()
        torch.cuda.current_stream().wait_stream(s)
        for a, b in zip(got, (x, y, dx, dqw, dkw, dtable)):
            assert torch.equal(a, b)


def test_refusals_leave_outputs(ops):
    """Wrong tensors raise ValueError before anything runs."""
    n, v, d = 4, 6, 16
    table, out = torch.ones((v, d), device=DEV), torch.full((n, d), 7.0, device=DEV)
    ids = torch.zeros(n, dtype=torch.int32, device=DEV)
    for bad in (lambda: ops.embed_rows(out, table, ids.long()), lambda: ops.embed_rows(out, table, ids[:3]),
                lambda: ops.embed_rows(out[:, :8], table, ids), lambda: ops.embed_rows(out.double(), table, ids),
                lambda: ops.embed_rows(out.t().contiguous().t(), table, ids),
                lambda: ops.embed_rows(out, table, ids.cpu()), lambda: ops.embed_rows(out.cpu(), table, ids),
                lambda: ops.embed_rows_grad(table, out, ids, workspace=torch.empty(8, dtype=torch.uint8, device=DEV)),
                lambda: ops.embed_rows_grad(table, out[:, :1].expand(n, d), ids)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):  # output rows on top of one another
        ops.embed_rows(out[:1].expand(n, d), table, ids)
    assert (out == 7.0).all() and (table == 1.0).all()
    q = torch.ones((n, 2, 32), device=DEV)
    o = torch.full_like(q, 7.0)
    cos, sin = tables(32, 8)
    call = lambda q=q, o=o, w=None, cos=cos, sin=sin, pos=ids: ops.qkv_norm_rope(o, None, None, q, None, None, w, None,
                                                                                 cos, sin, pos)
    for bad in (lambda: call(q=q.half()), lambda: call(o=o[:, :1]), lambda: call(w=torch.ones(31, device=DEV)),
                lambda: call(w=torch.ones(32, device=DEV, dtype=BF16)), lambda: call(cos=cos[:, :8]),
                lambda: call(sin=sin[:4]), lambda: call(pos=ids.long()), lambda: call(q=None),
                lambda: call(q=torch.ones((n, 2, 514), device=DEV)), lambda: call(q=torch.ones((n, 2, 33), device=DEV))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        call(o=o[:, :1].expand(n, 2, 32))
    assert (o == 7.0).all()
