"""Operator ABI calls (include/eg2_ops.h) on torch CUDA tensors.

Each function fills the parameter struct with device pointers and enqueues the
operator on the current torch stream; a non-zero return code raises.  torch is
only the allocator and stream provider here.
"""
from __future__ import annotations

import ctypes as C

from . import _lib


def _p(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _stream():
    import torch
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _call(name, struct, *extra):
    fn = getattr(_lib.load(), name)
    rc = fn(C.byref(struct), *extra, _stream())
    if rc:
        raise RuntimeError(f"{name} failed with CUDA error {rc}")


# ---- kernels/abi.h operators (reference semantics) ----
def gather(out, weight, ids, n):
    _call("eg2_launch_gather", _lib.EgGather(_p(out), _p(weight), _p(ids), n))


def mm(out, x, weight, n, k, m, type_):
    _call("eg2_launch_mm", _lib.EgMM(_p(out), _p(x), _p(weight), n, k, m, type_))


def norm(out, x, weight, rows, d, scale=1.0):
    _call("eg2_launch_norm", _lib.EgNorm(_p(out), _p(x), _p(weight), rows, d, scale))


def rope(x, table, n, heads, d):
    _call("eg2_launch_rope", _lib.EgRope(_p(x), _p(table), n, heads, d))


def attention(out, q, k, v, bounds, n, window, d):
    _call("eg2_launch_attention", _lib.EgAttention(_p(out), _p(q), _p(k), _p(v), _p(bounds), n, window), C.c_uint(d))


def element(out, x, other, n, mode, layer=0, scale=1.0):
    _call("eg2_launch_element", _lib.EgElement(_p(out), _p(x), _p(other), n, mode, layer, scale))


def pool(out, x, offsets, batch):
    _call("eg2_launch_pool", _lib.EgPool(_p(out), _p(x), _p(offsets), batch))


def norm_residual(out, x, weight, rows, d, scale):
    _call("eg2_launch_norm_residual", _lib.EgNormResidual(_p(out), _p(x), _p(weight), rows, d, scale))


def norm_rope(x, weight, table, rows, d, heads):
    _call("eg2_launch_norm_rope", _lib.EgNormRope(_p(x), _p(weight), _p(table), rows, d, heads))


# ---- fused executor operators ----
def embed(x, x_hi, x_lo, token_embd, ids, n):
    _call("eg2_launch_embed", _lib.EgEmbed(_p(x), _p(x_hi), _p(x_lo), _p(token_embd), _p(ids), n))


def ple_proj(ple, x_hi, x_lo, weight, norm_w, n):
    _call("eg2_launch_ple_proj", _lib.EgPleProj(_p(ple), _p(x_hi), _p(x_lo), _p(weight), _p(norm_w), n))


def norm_quant(q, scale, scale_stride, x, weight, rows, width, y=None, tier=0):
    _call("eg2_launch_norm_quant", _lib.EgNormQuant(_p(q), _p(scale), scale_stride, _p(y), _p(x), _p(weight),
                                                    rows, width, tier))


def q8_mm(out, xq, xs, xs_stride, wq, ws, n, k, m, exact=False):
    _call("eg2_launch_q8_mm", _lib.EgQ8MM(_p(out), _p(xq), _p(xs), xs_stride, _p(wq), _p(ws), n, k, m, int(exact)))


def q8_geglu(q, scale, scale_stride, xq, xs, xs_stride, wq, ws, n, k, m, exact=False, tier=0):
    _call("eg2_launch_q8_geglu", _lib.EgQ8GeGLU(_p(q), _p(scale), scale_stride, _p(xq), _p(xs), xs_stride, _p(wq),
                                                _p(ws), n, k, m, int(exact), tier))


def qkv_post(q, k, v, qkv, q_norm, k_norm, rope_cos, rope_sin, pos, n, d):
    _call("eg2_launch_qkv_post", _lib.EgQkvPost(_p(q), _p(k), _p(v), _p(qkv), _p(q_norm), _p(k_norm),
                                                _p(rope_cos), _p(rope_sin), _p(pos), n, d))


def attention_exact(out, q, k, v, bounds, n, d, window):
    """fp32 attention in the reference CPU graph's scalar order (parity mode)."""
    _call("eg2_launch_attention_exact", _lib.EgAttention(_p(out), _p(q), _p(k), _p(v), _p(bounds), n, window), d)


def attention_f16(out, q, k, v, bounds, n, d, window):
    _call("eg2_launch_attention_f16", _lib.EgAttentionF16(_p(out), _p(q), _p(k), _p(v), _p(bounds), n, d, window))


def attention_tc(out, q, k, v, bounds, n, window, d=256):
    """attention_f16 on the tcgen05 tensor cores (d = 256 or 512, n <= 8192)."""
    _call("eg2_launch_attention_tc", _lib.EgAttentionF16(_p(out), _p(q), _p(k), _p(v), _p(bounds), n, d, window))


def attention_tc_q8(q, qscale, scale_stride, qh, k, v, bounds, n, window, tier=0, d=256):
    """attention_tc with its output rows quantized to Q8_0 in the epilogue."""
    _call("eg2_launch_attention_tc_q8", _lib.EgAttentionQ8(_p(q), _p(qscale), scale_stride, _p(qh), _p(k), _p(v),
                                                           _p(bounds), n, window, tier, d))


def post_add(x, h, weight, scale, q, qscale, scale_stride, next_weight, rows, tier=0):
    _call("eg2_launch_post_add", _lib.EgPostAdd(_p(x), _p(h), _p(weight), _p(scale), _p(q), _p(qscale),
                                                scale_stride, _p(next_weight), rows, tier))


def gate_quant(q, scale, scale_stride, x, other, rows, width, other_stride, other_offset, tier=0):
    _call("eg2_launch_gate_quant", _lib.EgGateQuant(_p(q), _p(scale), scale_stride, _p(x), _p(other), rows, width,
                                                    other_stride, other_offset, tier))


def gelu_mul(g, u, n, tier=0):
    """g[:n] = gelu_tanh(g[:n]) * u[:n] in place (u None: gelu only)."""
    _call("eg2_launch_gelu_mul", _lib.EgGeluMul(_p(g), _p(u), n, tier))


def pool_l2(out, y, offsets, batch, width):
    _call("eg2_launch_pool_l2", _lib.EgPoolL2(_p(out), _p(y), _p(offsets), batch, width))


# ---- typed operators and their gradients (fp32, fp16, bf16) ----
# These check their tensors (ValueError before anything is enqueued) and run on
# the current stream of their tensors' device, whichever device is current.
_TYPES = {"torch.float32": 0, "torch.float16": 1, "torch.bfloat16": 30}


def _type(t, name):
    code = _TYPES.get(str(t.dtype))
    if code is None:
        raise ValueError(f"{name} is {t.dtype}: expected float32, float16 or bfloat16")
    return code


def _check(t, name, shape, device=None, dtype=None, contiguous=False):
    """A CUDA tensor of `shape` (None: any size) whose last dimension is contiguous."""
    if not t.is_cuda or (device is not None and t.device != device):
        raise ValueError(f"{name} is on {t.device}: expected {device or 'a CUDA device'}")
    if t.dim() != len(shape) or any(s is not None and s != g for s, g in zip(shape, t.shape)):
        raise ValueError(f"{name} has shape {tuple(t.shape)}: expected {tuple('any' if s is None else s for s in shape)}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} is {t.dtype}: expected {dtype}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} is not contiguous")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}'s rows are not contiguous (last stride {t.stride(-1)})")


def _check_ids(t, name, n, device):
    import torch
    _check(t, name, (n,), device, torch.int32, contiguous=True)


def _workspace(workspace, need, device):
    """The caller's workspace, or a fresh one on the current stream."""
    import torch
    if workspace is None:
        return torch.empty(need, dtype=torch.uint8, device=device)
    if workspace.device != device or not workspace.is_contiguous():
        raise ValueError(f"workspace must be contiguous and on {device}")
    size = workspace.numel() * workspace.element_size()
    if size < need:
        raise ValueError(f"workspace has {size} bytes: {need} needed")
    if size and workspace.data_ptr() % 256:
        raise ValueError("workspace must be 256-byte aligned")
    return workspace


def _call_on(device, name, struct):
    """_call on `device`, on that device's current stream."""
    import torch
    if device.index == torch.cuda.current_device():
        return _call(name, struct)
    with torch.cuda.device(device):
        _call(name, struct)


def embed_rows(out, table, ids, scale=1.0):
    """out[t] = scale * table[ids[t]]; an id outside the table is padding (zeros).

    out [n][d] and table [vocab][d] are float32, float16 or bfloat16 (each its
    own), ids int32 [n]."""
    dev = table.device
    _check(table, "table", (None, None))
    vocab, d = table.shape
    _check(out, "out", (None, d), dev)
    n = out.shape[0]
    _check_ids(ids, "ids", n, dev)
    _call_on(dev, "eg2_launch_embed_rows", _lib.EgEmbedRows(
        _p(out), _p(table), _p(ids), out.stride(0), table.stride(0), n, vocab, d, _type(out, "out"),
        _type(table, "table"), scale))


def embed_rows_grad_workspace(n, d) -> int:
    """Bytes of workspace for embed_rows_grad."""
    return int(_lib.load().eg2_embed_rows_grad_workspace(n, d))


def embed_rows_grad(dtable, dout, ids, scale=1.0, accumulate=False, workspace=None):
    """dtable[v] = scale * sum of dout[t] over ids[t] = v, or added to dtable (accumulate)."""
    dev = dtable.device
    _check(dtable, "dtable", (None, None))
    vocab, d = dtable.shape
    _check(dout, "dout", (None, d), dev)
    n = dout.shape[0]
    _check_ids(ids, "ids", n, dev)
    tw, tg = _type(dtable, "dtable"), _type(dout, "dout")
    ws = _workspace(workspace, embed_rows_grad_workspace(n, d), dev)
    _call_on(dev, "eg2_launch_embed_rows_grad", _lib.EgEmbedRowsGrad(
        _p(dtable), _p(dout), _p(ids), _p(ws), ws.numel() * ws.element_size(), dtable.stride(0), dout.stride(0),
        n, vocab, d, tw, tg, scale, int(accumulate)))


def _heads(name, t, n, d, device, dtype):
    """(pointer, strides, heads) of a [n][heads][d] tensor, or of None."""
    if t is None:
        return None, (0, 0), 0
    _check(t, name, (n, None, d), device, dtype)
    return _p(t), (t.stride(0), t.stride(1)), t.shape[1]


def _qkv_args(x, weights, rope_cos, rope_sin, pos):
    """The first given of queries, keys and values sets n, d, device and type."""
    import torch
    lead = next((t for t in x if t is not None), None)
    if lead is None:
        raise ValueError("queries, keys and values are all None")
    _check(lead, "x", (None, None, None))
    (n, _, d), dev = lead.shape, lead.device
    code = _type(lead, "x")
    if d % 2 or not 0 < d <= 512:
        raise ValueError(f"head width {d}: expected an even number up to 512")
    _check_ids(pos, "pos", n, dev)
    wtypes = {w.dtype for w in weights if w is not None} or {torch.float32}
    if len(wtypes) > 1 or not wtypes <= {torch.float32, lead.dtype}:
        raise ValueError(f"weights are {wtypes}: expected one of float32 and {lead.dtype} for both")
    for name, w in zip(("q_weight", "k_weight"), weights):
        if w is not None:
            _check(w, name, (d,), dev)
    _check(rope_cos, "rope_cos", (None, d // 2), dev, torch.float32, contiguous=True)
    _check(rope_sin, "rope_sin", tuple(rope_cos.shape), dev, torch.float32, contiguous=True)
    wtype = 0 if wtypes == {torch.float32} else code
    return n, d, dev, lead.dtype, code, wtype, rope_cos.shape[0]


def qkv_norm_rope(q_out, k_out, v_out, q, k, v, q_weight, k_weight, rope_cos, rope_sin, pos, eps=1e-6):
    """Per-head RMS norm of q, k [n][heads][d] with weights [d] and NEOX rotation by
    row pos[t] of rope_cos, rope_sin [positions][d / 2]; v gets the norm alone.

    Any of the three may be None with its output; a weight None is 1.  A position
    outside the tables is padding (zeros).  An output may be its input."""
    n, d, dev, dtype, code, wtype, positions = _qkv_args((q, k, v), (q_weight, k_weight), rope_cos, rope_sin, pos)
    x = [_heads(name, t, n, d, dev, dtype) for name, t in (("q", q), ("k", k), ("v", v))]
    out = [_heads(name, t, n, d, dev, dtype) for name, t in (("q_out", q_out), ("k_out", k_out), ("v_out", v_out))]
    heads = [a[2] for a in x]
    if heads != [a[2] for a in out]:
        raise ValueError(f"outputs have {[a[2] for a in out]} heads, inputs {heads}")
    L = _lib
    _call_on(dev, "eg2_launch_qkv_norm_rope", L.EgQkvNormRope(
        L.P3(*[a[0] for a in out]), L.P3(*[a[0] for a in x]), L.P2(_p(q_weight), _p(k_weight)), _p(rope_cos),
        _p(rope_sin), _p(pos), L.Strides3(*[a[1] for a in out]), L.Strides3(*[a[1] for a in x]), n, *heads, d,
        positions, code, wtype, eps))


def qkv_norm_rope_grad_workspace(n, q_heads, kv_heads, d) -> int:
    """Bytes of workspace for qkv_norm_rope_grad."""
    return int(_lib.load().eg2_qkv_norm_rope_grad_workspace(n, q_heads, kv_heads, d))


def qkv_norm_rope_grad(dq, dk, dv, dq_weight, dk_weight, dq_out, dk_out, dv_out, q, k, v, q_weight, k_weight,
                       rope_cos, rope_sin, pos, eps=1e-6, accumulate=False, workspace=None):
    """The gradient of qkv_norm_rope: dq, dk, dv from the outputs' gradients, and the
    weights' gradients (None: not wanted), added to what they hold with accumulate."""
    n, d, dev, dtype, code, wtype, positions = _qkv_args((q, k, v), (q_weight, k_weight), rope_cos, rope_sin, pos)
    x = [_heads(name, t, n, d, dev, dtype) for name, t in (("q", q), ("k", k), ("v", v))]
    dx = [_heads(name, t, n, d, dev, dtype) for name, t in (("dq", dq), ("dk", dk), ("dv", dv))]
    g = [_heads(name, t, n, d, dev, dtype) for name, t in (("dq_out", dq_out), ("dk_out", dk_out), ("dv_out", dv_out))]
    heads = [a[2] for a in x]
    if heads != [a[2] for a in dx] or heads != [a[2] for a in g]:
        raise ValueError(f"gradients have {[a[2] for a in dx]} and {[a[2] for a in g]} heads, inputs {heads}")
    need = 0
    for name, w, given in (("dq_weight", dq_weight, q_weight), ("dk_weight", dk_weight, k_weight)):
        if w is not None:
            if given is None:
                raise ValueError(f"{name} is wanted of a weight that is None")
            _check(w, name, (d,), dev, given.dtype)
            need = qkv_norm_rope_grad_workspace(n, heads[0], max(heads[1:]), d)
    ws = _workspace(workspace, need, dev)
    L = _lib
    _call_on(dev, "eg2_launch_qkv_norm_rope_grad", L.EgQkvNormRopeGrad(
        L.P3(*[a[0] for a in dx]), L.P2(_p(dq_weight), _p(dk_weight)), L.P3(*[a[0] for a in g]),
        L.P3(*[a[0] for a in x]), L.P2(_p(q_weight), _p(k_weight)), _p(rope_cos), _p(rope_sin), _p(pos), _p(ws),
        ws.numel() * ws.element_size(), L.Strides3(*[a[1] for a in dx]), L.Strides3(*[a[1] for a in g]),
        L.Strides3(*[a[1] for a in x]), n, *heads, d, positions, code, wtype, eps, int(accumulate)))


_ACTS = {"gelu_tanh": 0, "silu": 1}


def _glu_args(x, w_gate, w_up, act):
    if act not in _ACTS:
        raise ValueError(f"act {act!r}: expected one of {sorted(_ACTS)}")
    dev = x.device
    _check(x, "x", (None, None))
    n, k = x.shape
    code = _type(x, "x")
    if code == 0:
        raise ValueError("x is torch.float32: expected float16 or bfloat16")
    _check(w_gate, "w_gate", (None, k), dev, x.dtype)
    m = w_gate.shape[0]
    _check(w_up, "w_up", (m, k), dev, x.dtype)
    if k % 8 or m % 8 or not k or not m:
        raise ValueError(f"k = {k}, m = {m}: expected multiples of 8")
    return n, k, m, dev, code


def glu(out, x, w_gate, w_up, act="gelu_tanh"):
    """out = act(x w_gate^T) * (x w_up^T): x [n][k], weights [m][k], out [n][m], float16 or bfloat16.

    act is "gelu_tanh" or "silu"; k and m are multiples of 8, rows 16-byte aligned."""
    n, k, m, dev, code = _glu_args(x, w_gate, w_up, act)
    _check(out, "out", (n, m), dev, x.dtype)
    _call_on(dev, "eg2_launch_glu", _lib.EgGlu(
        _p(out), _p(x), _p(w_gate), _p(w_up), out.stride(0), x.stride(0), w_gate.stride(0), w_up.stride(0), n, k, m,
        code, _ACTS[act]))


def glu_grad_workspace(n, k, m) -> int:
    """Bytes of workspace for glu_grad."""
    return int(_lib.load().eg2_glu_grad_workspace(n, k, m))


def glu_grad(dx, dw_gate, dw_up, dout, x, w_gate, w_up, act="gelu_tanh", accumulate=False, workspace=None):
    """The gradient of glu from dout [n][m] (None among dx, dw_gate, dw_up: not wanted).

    The weights' gradients are of x's type or float32; with accumulate they are
    float32 and added to.  Nothing is kept from the forward pass: the
    projections are computed again."""
    n, k, m, dev, code = _glu_args(x, w_gate, w_up, act)
    _check(dout, "dout", (n, m), dev, x.dtype)
    if dx is not None:
        _check(dx, "dx", (n, k), dev, x.dtype)
    dw_code = code
    for name, w in (("dw_gate", dw_gate), ("dw_up", dw_up)):
        if w is not None:
            _check(w, name, (m, k), dev)
            dw_code = _type(w, name)
    if dw_gate is not None and dw_up is not None and dw_gate.dtype != dw_up.dtype:
        raise ValueError(f"dw_gate is {dw_gate.dtype}, dw_up {dw_up.dtype}: expected one type")
    if dw_code not in (0, code) or (accumulate and dw_code != 0 and not (dw_gate is None and dw_up is None)):
        raise ValueError("weight gradients are float32 or x's type, float32 with accumulate")
    ws = _workspace(workspace, glu_grad_workspace(n, k, m), dev)
    st = lambda t: 0 if t is None else t.stride(0)
    _call_on(dev, "eg2_launch_glu_grad", _lib.EgGluGrad(
        _p(dx), _p(dw_gate), _p(dw_up), _p(dout), _p(x), _p(w_gate), _p(w_up), _p(ws), ws.numel() * ws.element_size(),
        st(dx), st(dw_gate), st(dw_up), dout.stride(0), x.stride(0), w_gate.stride(0), w_up.stride(0), n, k, m, code,
        _ACTS[act], dw_code, int(accumulate and dw_code == 0)))


def repack_q8(blocks, rows, k, codes, scales):
    rc = _lib.load().eg2_repack_q8(_p(blocks), rows, k, _p(codes), _p(scales), _stream())
    if rc:
        raise RuntimeError(f"eg2_repack_q8 failed with CUDA error {rc}")


def read_error() -> int:
    return int(_lib.load().eg2_read_error())


def clear_error():
    _lib.load().eg2_clear_error()


def selftest_wait_timeout(stream=None):
    """Enqueue a kernel whose bounded wait runs out (sets the error word)."""
    rc = _lib.load().eg2_selftest_wait_timeout(C.c_void_p(stream) if stream is not None else _stream())
    if rc:
        raise RuntimeError(f"eg2_selftest_wait_timeout failed with CUDA error {rc}")
