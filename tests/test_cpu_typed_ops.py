"""Refusals of the typed operators (include/eg2_ops.h part 3) without a GPU: the
C entry points return an error code for bad arguments before they launch
anything, and the Python entry points raise for tensors that are not theirs."""
import ctypes as C
import importlib

import pytest

torch = pytest.importorskip("torch")

INVALID = 1  # cudaErrorInvalidValue
A = 4096     # stands for an aligned device address; nothing below gets as far as using it


@pytest.fixture(scope="module")
def L(eg2):
    return eg2._lib


def call(L, name, struct):
    return getattr(L.load(), name)(C.byref(struct), None)


def embed(L, **kw):
    f = dict(out=A, table=A, ids=A, out_stride=16, table_stride=16, n=4, vocab=9, d=16, out_type=0, table_type=0,
             scale=1.0)
    f.update(kw)
    return call(L, "eg2_launch_embed_rows", L.EgEmbedRows(**f))


def embed_grad(L, **kw):
    f = dict(dtable=A, dout=A, ids=A, workspace=A, workspace_bytes=1 << 30, dtable_stride=16, dout_stride=16, n=4,
             vocab=9, d=16, dtable_type=0, dout_type=0, scale=1.0, accumulate=0)
    f.update(kw)
    return call(L, "eg2_launch_embed_rows_grad", L.EgEmbedRowsGrad(**f))


@pytest.mark.parametrize("kw", [dict(out=None), dict(table=None), dict(ids=None), dict(d=0), dict(d=1 << 21),
                                dict(n=1 << 31), dict(vocab=0xffffffff), dict(out_type=8), dict(table_type=2),
                                dict(out_stride=15), dict(out_stride=-16), dict(table_stride=8)])
def test_embed_rows_refuses(L, kw):
    assert embed(L, **kw) == INVALID


@pytest.mark.parametrize("kw", [dict(dtable=None), dict(dout=None), dict(ids=None), dict(workspace=None),
                                dict(workspace=A + 16), dict(workspace_bytes=100), dict(d=0), dict(n=1 << 31),
                                dict(vocab=0xffffffff), dict(dtable_type=8), dict(dout_type=2),
                                dict(dtable_stride=15), dict(dout_stride=-1)])
def test_embed_rows_grad_refuses(L, kw):
    assert embed_grad(L, **kw) == INVALID


def test_nothing_to_do_is_no_error(L):
    assert embed(L, n=0, out=None, ids=None) == 0
    assert embed_grad(L, vocab=0) == 0
    assert embed_grad(L, n=0, accumulate=1) == 0
    assert qkv(L, n=0) == 0
    assert qkv(L, q_heads=0, k_heads=0, v_heads=0) == 0
    assert qkv_grad(L, n=0, accumulate=1) == 0


def qkv_fields(L, names, **kw):
    s = [(4 * 64, 64)] * 3
    f = {k: L.P3(A, A, A) for k in names}
    f.update({k + "_stride": L.Strides3(*s) for k in names})
    f.update(weight=L.P2(A, A), rope_cos=A, rope_sin=A, pos=A, n=5, q_heads=4, k_heads=2, v_heads=2, d=64,
             positions=8, type=0, weight_type=0, eps=1e-6)
    f.update(kw)
    return f


def qkv(L, **kw):
    return call(L, "eg2_launch_qkv_norm_rope", L.EgQkvNormRope(**qkv_fields(L, ("out", "x"), **kw)))


def qkv_grad(L, **kw):
    f = dict(dweight=L.P2(A, A), workspace=A, workspace_bytes=1 << 30)
    f.update(kw)
    return call(L, "eg2_launch_qkv_norm_rope_grad",
                L.EgQkvNormRopeGrad(**qkv_fields(L, ("dx", "dout", "x"), **f)))


BAD_QKV = [dict(d=0), dict(d=63), dict(d=514), dict(type=8), dict(weight_type=1), dict(rope_cos=None),
           dict(rope_sin=None), dict(pos=None), dict(n=1 << 31), dict(positions=1 << 31), dict(q_heads=70000)]


@pytest.mark.parametrize("kw", BAD_QKV)
def test_qkv_norm_rope_refuses(L, kw):
    assert qkv(L, **kw) == INVALID
    assert qkv_grad(L, **kw) == INVALID


def test_qkv_norm_rope_refuses_pointers_and_strides(L):
    over = L.Strides3((4 * 64, 63), (256, 64), (256, 64))   # heads overlap
    tight = L.Strides3((255, 64), (256, 64), (256, 64))     # tokens overlap
    back = L.Strides3((256, -64), (256, 64), (256, 64))
    null = L.P3(A, None, A)
    for s in (over, tight, back):
        assert qkv(L, out_stride=s) == INVALID
        assert qkv_grad(L, dx_stride=s) == INVALID
    for kw in (dict(x=null), dict(x_stride=back)):
        assert qkv(L, **kw) == INVALID
        assert qkv_grad(L, **kw) == INVALID
    assert qkv(L, out=null) == INVALID
    for kw in (dict(dx=null), dict(dout=null), dict(dout_stride=back), dict(workspace=None), dict(workspace=A + 8),
               dict(workspace_bytes=64)):
        assert qkv_grad(L, **kw) == INVALID


def test_packed_parameters_have_the_struct_layout(eg2, L):
    """The Python entry points pack parameters as the C structs lay them out."""
    ops = importlib.import_module("embeddinggemma2-amdkfd_b200.ops")
    for op, cls in ((ops._embed_rows, L.EgEmbedRows), (ops._embed_rows_grad, L.EgEmbedRowsGrad),
                    (ops._qkv_norm_rope, L.EgQkvNormRope), (ops._qkv_norm_rope_grad, L.EgQkvNormRopeGrad),
                    (ops._glu, L.EgGlu), (ops._glu_grad, L.EgGluGrad)):
        flat, rows, i = [], {}, 1
        for name, t in cls._fields_:
            count = C.sizeof(t) // (4 if t in (C.c_uint, C.c_float) else 8)
            rows[name] = list(range(i, i + count))
            flat += rows[name]
            i += count
        params = op.pack(*flat)
        assert len(params) == C.sizeof(cls), op.name
        got = cls.from_buffer_copy(params)
        for name, t in cls._fields_:
            v = getattr(got, name)
            v = [x for y in v for x in (y if hasattr(y, "__len__") else [y])] if hasattr(v, "__len__") else [v]
            assert v == rows[name], (op.name, name)


def test_workspace_sizes(L):
    lib = L.load()
    for n in (1, 7, 2048, 32767, 32768, 262144, 262145, 1_000_000):
        for d in (1, 512):
            size = lib.eg2_embed_rows_grad_workspace(n, d)
            assert size >= 16 * n and size % 256 == 0
    assert lib.eg2_qkv_norm_rope_grad_workspace(1, 4, 2, 256) == 8 * 256 * 4
    assert lib.eg2_qkv_norm_rope_grad_workspace(100000, 4, 2, 256) == 1024 * 256 * 4


def test_python_entry_points_refuse_cpu_tensors(eg2):
    ops = importlib.import_module("embeddinggemma2-amdkfd_b200.ops")
    t, ids = torch.ones((4, 8)), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="expected a CUDA device"):
        ops.embed_rows(t, t, ids)
    with pytest.raises(ValueError, match="expected a CUDA device"):
        ops.embed_rows_grad(t, t, ids)
    x = torch.ones((4, 2, 8))
    with pytest.raises(ValueError, match="expected a CUDA device"):
        ops.qkv_norm_rope(x, None, None, x, None, None, None, None, t[:, :4], t[:, :4], ids)


def glu_fields(names, **kw):
    f = {k: A for k in names}
    width = {k: 128 if k in ("out", "dout") else 64 for k in names}
    f.update({k + "_stride": width[k] for k in names})
    f.update(n=20, k=64, m=128, type=30, act=0)
    f.update(kw)
    return f


def glu(L, **kw):
    return call(L, "eg2_launch_glu", L.EgGlu(**glu_fields(("out", "x", "w_gate", "w_up"), **kw)))


def glu_grad(L, **kw):
    f = dict(workspace=A, workspace_bytes=1 << 30, dw_type=30, accumulate=0)
    f.update(kw)
    names = ("dx", "dw_gate", "dw_up", "dout", "x", "w_gate", "w_up")
    return call(L, "eg2_launch_glu_grad", L.EgGluGrad(**glu_fields(names, **f)))


@pytest.mark.parametrize("kw", [dict(k=0), dict(m=0), dict(k=60), dict(m=124), dict(type=0), dict(type=8),
                                dict(act=2), dict(n=1 << 31), dict(k=1 << 25), dict(x=None), dict(w_gate=None),
                                dict(w_up=None), dict(x=A + 2), dict(w_up=A + 8), dict(x_stride=63),
                                dict(x_stride=68), dict(w_gate_stride=-64), dict(w_up_stride=66)])
def test_glu_refuses(L, kw):
    assert glu(L, **kw) == INVALID
    assert glu_grad(L, **kw) == INVALID


@pytest.mark.parametrize("kw", [dict(dout=None), dict(dout_stride=120), dict(dout=A + 8), dict(dx_stride=32),
                                dict(dx=A + 4), dict(dw_gate_stride=68), dict(dw_up=A + 2), dict(dw_type=1),
                                dict(accumulate=1), dict(workspace=None), dict(workspace=A + 16),
                                dict(workspace_bytes=2 * 20 * 128 * 2 - 1)])
def test_glu_grad_refuses(L, kw):
    assert glu_grad(L, **kw) == INVALID


def test_glu_nothing_to_do(L):
    assert glu(L, n=0, x=None, out=None) == 0
    assert glu(L, out=None) == INVALID
    assert glu_grad(L, n=0, dx=None, dw_gate=None, dw_up=None) == 0
    assert glu_grad(L, n=0, dw_type=0, accumulate=1) == 0
    assert glu_grad(L, dx=None, dw_gate=None, dw_up=None) == 0
