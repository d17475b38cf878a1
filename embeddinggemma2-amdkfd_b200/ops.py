"""Operator ABI calls (include/eg2_ops.h) on torch CUDA tensors.

Each function fills the parameter struct with device pointers and enqueues the
operator on the current torch stream; a non-zero return code raises.  torch is
only the allocator and stream provider here.
"""
from __future__ import annotations

import ctypes as C
import struct

import torch

from . import _lib


def _p(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _call(name, params, *extra):
    fn = getattr(_lib.load(), name)
    rc = fn(C.byref(params), *extra, _stream())
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
# These check their tensors' shapes, types, devices and rows (ValueError) and leave
# alignment, overlapping rows and limits to the C entry point (RuntimeError); both
# before anything is enqueued.  They run on the current stream of their tensors'
# device, whichever device is current, and record nothing for autograd.  A
# call of a small operator is mostly host time, so a check that passes is a few
# comparisons, and the parameters are packed straight into the C struct's bytes.
class _Typed:
    """One C entry point; arrays of its parameter struct are passed flat."""

    CODES = {C.c_void_p: "P", C.c_int64: "q", C.c_uint64: "Q", C.c_uint: "I", C.c_float: "f"}

    def __init__(self, name, cls):
        self.name, self.fn = name, None
        fmt = "@"
        for _, t in cls._fields_:
            count = 1
            while hasattr(t, "_length_"):
                count, t = count * t._length_, t._type_
            fmt += f"{count}{self.CODES[t]}"
        self.pack = struct.Struct(fmt + "0P").pack  # 0P: the struct's trailing alignment

    def __call__(self, device, *values):
        if self.fn is None:
            self.fn = getattr(_lib.load(), self.name)
        params, index = self.pack(*values), device.index
        if index == torch._C._cuda_getDevice():
            rc = self.fn(params, torch._C._cuda_getCurrentRawStream(index))
        else:
            with torch.cuda.device(index):
                rc = self.fn(params, torch._C._cuda_getCurrentRawStream(index))
        if rc == 1:  # cudaErrorInvalidValue, before anything is enqueued
            raise RuntimeError(f"{self.name} refused its arguments (CUDA error 1): rows that overlap or are not "
                               "aligned as it needs, or sizes past its limits")
        if rc:
            raise RuntimeError(f"{self.name} failed with CUDA error {rc}")


_embed_rows = _Typed("eg2_launch_embed_rows", _lib.EgEmbedRows)
_embed_rows_grad = _Typed("eg2_launch_embed_rows_grad", _lib.EgEmbedRowsGrad)
_qkv_norm_rope = _Typed("eg2_launch_qkv_norm_rope", _lib.EgQkvNormRope)
_qkv_norm_rope_grad = _Typed("eg2_launch_qkv_norm_rope_grad", _lib.EgQkvNormRopeGrad)
_glu = _Typed("eg2_launch_glu", _lib.EgGlu)
_glu_grad = _Typed("eg2_launch_glu_grad", _lib.EgGluGrad)
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
_ACTS = {"gelu_tanh": 0, "silu": 1}


def _type(t, name):
    code = _TYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} is {t.dtype}: expected float32, float16 or bfloat16")
    return code


def _lead(t, name, dims):
    """Shape, device and strides of the tensor that sets the call's sizes."""
    shape, stride = t.shape, t.stride()
    if not t.is_cuda:
        raise ValueError(f"{name} is on {t.device}: expected a CUDA device")
    if len(shape) != dims:
        raise ValueError(f"{name} has shape {tuple(shape)}: expected {dims} dimensions")
    if stride[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"{name}'s rows are not contiguous (last stride {stride[-1]})")
    return shape, t.device, stride


def _check(t, name, shape, device, dtype):
    """The strides of a tensor of that shape, device and type whose last dimension is contiguous."""
    stride = t.stride()
    if t.dtype is dtype and t.shape == shape and t.device == device and (stride[-1] == 1 or shape[-1] < 2):
        return stride
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}: expected {tuple(shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}: expected {device}")
    if t.dtype != dtype:
        raise ValueError(f"{name} is {t.dtype}: expected {dtype}")
    raise ValueError(f"{name}'s rows are not contiguous (last stride {stride[-1]})")


def _rows(t, name, width, device):
    """Rows and row stride of a tensor of shape [any][width]."""
    shape = t.shape
    if len(shape) != 2 or shape[1] != width:
        raise ValueError(f"{name} has shape {tuple(shape)}: expected (any, {width})")
    return shape[0], _check(t, name, shape, device, t.dtype)[0]


def _workspace(workspace, need, device):
    """(address, bytes, tensor) of the caller's workspace, or of a fresh one on the current stream."""
    if workspace is None:
        with torch.cuda.device(device):
            workspace = torch.empty(need, dtype=torch.uint8, device=device)
        return workspace.data_ptr(), need, workspace
    size, ptr = workspace.numel() * workspace.element_size(), workspace.data_ptr()
    if workspace.device != device or not workspace.is_contiguous():
        raise ValueError(f"workspace must be contiguous and on {device}")
    if size < need:
        raise ValueError(f"workspace has {size} bytes: {need} needed")
    if need and ptr % 256:
        raise ValueError("workspace must be 256-byte aligned")
    return ptr, size, workspace


def _apart(a, b, names):
    """Two gradients written by one call are two tensors: one given twice would lose a part of each."""
    if a is not None and b is not None and a.data_ptr() == b.data_ptr() and a.numel():
        raise ValueError(f"{names} are the same memory: each needs its own")


def embed_rows(out, table, ids, scale=1.0):
    """out[t] = scale * table[ids[t]]; an id outside the table is padding (zeros).

    out [n][d] and table [vocab][d] are float32, float16 or bfloat16 (each its
    own), ids int32 [n]."""
    (vocab, d), dev, stride = _lead(table, "table", 2)
    n, out_stride = _rows(out, "out", d, dev)
    _check(ids, "ids", (n,), dev, torch.int32)
    _embed_rows(dev, out.data_ptr(), table.data_ptr(), ids.data_ptr(), out_stride, stride[0], n, vocab, d,
                _type(out, "out"), _type(table, "table"), scale)


def embed_rows_grad_workspace(n, d) -> int:
    """Bytes of workspace for embed_rows_grad."""
    return int(_lib.load().eg2_embed_rows_grad_workspace(n, d))


def embed_rows_grad(dtable, dout, ids, scale=1.0, accumulate=False, workspace=None):
    """dtable[v] = scale * sum of dout[t] over ids[t] = v, or added to dtable (accumulate).

    dtable [vocab][d] and dout [n][d] are float32, float16 or bfloat16 (each its
    own), ids int32 [n]; the sums are in fp32 and the same inputs give the same
    bits.  dout may be broadcast over tokens (row stride 0)."""
    (vocab, d), dev, stride = _lead(dtable, "dtable", 2)
    n, dout_stride = _rows(dout, "dout", d, dev)
    _check(ids, "ids", (n,), dev, torch.int32)
    types = _type(dtable, "dtable"), _type(dout, "dout")
    ws = _workspace(workspace, embed_rows_grad_workspace(n, d), dev)
    _embed_rows_grad(dev, dtable.data_ptr(), dout.data_ptr(), ids.data_ptr(), ws[0], ws[1], stride[0],
                     dout_stride, n, vocab, d, *types, scale, bool(accumulate))


def _qkv_args(x, q_weight, k_weight, rope_cos, rope_sin, pos):
    """Sizes and types; the first given of queries, keys and values sets n, d, device and type."""
    q, k, v = x
    lead = q if q is not None else k if k is not None else v
    if lead is None:
        raise ValueError("queries, keys and values are all None")
    (n, _, d), dev, _ = _lead(lead, "x", 3)
    dtype = lead.dtype
    code = wtype = _type(lead, "x")
    if d % 2 or not 0 < d <= 512:
        raise ValueError(f"head width {d}: expected an even number up to 512")
    _check(pos, "pos", (n,), dev, torch.int32)
    wdtype = q_weight.dtype if q_weight is not None else k_weight.dtype if k_weight is not None else dtype
    if wdtype == torch.float32:
        wtype = 0
    elif wdtype != dtype:
        raise ValueError(f"weights are {wdtype}: expected float32 or {dtype}")
    if q_weight is not None:
        _check(q_weight, "q_weight", (d,), dev, wdtype)
    if k_weight is not None:
        _check(k_weight, "k_weight", (d,), dev, wdtype)
    half = d // 2
    table = rope_cos.shape
    if len(table) != 2 or table[1] != half:
        raise ValueError(f"rope_cos has shape {tuple(table)}: expected (any, {half})")
    cos_stride = _check(rope_cos, "rope_cos", table, dev, torch.float32)[0]
    sin_stride = _check(rope_sin, "rope_sin", table, dev, torch.float32)[0]
    if table[0] > 1 and not cos_stride == sin_stride == half:
        raise ValueError("rope_cos and rope_sin must be contiguous")
    heads = [0 if t is None else t.shape[1] if t.dim() == 3 else -1 for t in x]
    return (n, *heads, d, table[0], code, wtype), dev, dtype


def _qkv_tensors(names, tensors, sizes, dev, dtype):
    """Addresses and (token, head) strides of three [n][heads][d] tensors."""
    n, d, ptrs, strides = sizes[0], sizes[4], [], []
    for i in (0, 1, 2):
        t, heads = tensors[i], sizes[i + 1]
        if t is None:
            if heads:
                raise ValueError(f"{names[i]} is None: expected {heads} heads")
            ptrs.append(0)
            strides += (0, 0)
            continue
        stride = t.stride()
        if t.dtype is not dtype or t.shape != (n, heads, d) or t.device != dev or stride[2] != 1:
            _check(t, names[i], (n, heads, d), dev, dtype)  # raises, saying what is wrong
        ptrs.append(t.data_ptr())
        strides += stride[:2]
    return ptrs, strides


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def qkv_norm_rope(q_out, k_out, v_out, q, k, v, q_weight, k_weight, rope_cos, rope_sin, pos, eps=1e-6):
    """Per-head RMS norm of q, k [n][heads][d] with weights [d] and NEOX rotation by
    row pos[t] of rope_cos, rope_sin [positions][d / 2]; v gets the norm alone.

    Any of the three may be None with its output; a weight None is 1.  A position
    outside the tables is padding (zeros), so they are given for values alone
    too.  An output may be its input."""
    sizes, dev, dtype = _qkv_args((q, k, v), q_weight, k_weight, rope_cos, rope_sin, pos)
    x, xs = _qkv_tensors(("q", "k", "v"), (q, k, v), sizes, dev, dtype)
    out, outs = _qkv_tensors(("q_out", "k_out", "v_out"), (q_out, k_out, v_out), sizes, dev, dtype)
    _qkv_norm_rope(dev, *out, *x, _ptr(q_weight), _ptr(k_weight), rope_cos.data_ptr(), rope_sin.data_ptr(),
                   pos.data_ptr(), *outs, *xs, *sizes, eps)


def qkv_norm_rope_grad_workspace(n, q_heads, kv_heads, d) -> int:
    """Bytes of workspace for qkv_norm_rope_grad."""
    return int(_lib.load().eg2_qkv_norm_rope_grad_workspace(n, q_heads, kv_heads, d))


def qkv_norm_rope_grad(dq, dk, dv, dq_weight, dk_weight, dq_out, dk_out, dv_out, q, k, v, q_weight, k_weight,
                       rope_cos, rope_sin, pos, eps=1e-6, accumulate=False, workspace=None):
    """The gradient of qkv_norm_rope: dq, dk, dv from the outputs' gradients, and the
    weights' gradients (None: not wanted), added to what they hold with accumulate."""
    sizes, dev, dtype = _qkv_args((q, k, v), q_weight, k_weight, rope_cos, rope_sin, pos)
    x, xs = _qkv_tensors(("q", "k", "v"), (q, k, v), sizes, dev, dtype)
    dx, dxs = _qkv_tensors(("dq", "dk", "dv"), (dq, dk, dv), sizes, dev, dtype)
    g, gs = _qkv_tensors(("dq_out", "dk_out", "dv_out"), (dq_out, dk_out, dv_out), sizes, dev, dtype)
    n, hq, hk, hv, d = sizes[:5]
    need = 0
    for name, w, given in (("dq_weight", dq_weight, q_weight), ("dk_weight", dk_weight, k_weight)):
        if w is not None:
            if given is None:
                raise ValueError(f"{name} is wanted of a weight that is None")
            _check(w, name, (d,), dev, given.dtype)
            need = qkv_norm_rope_grad_workspace(n, hq, max(hk, hv), d)
    _apart(dq_weight, dk_weight, "dq_weight and dk_weight")
    ws = _workspace(workspace, need, dev) if need else (0, 0, None)
    _qkv_norm_rope_grad(dev, *dx, _ptr(dq_weight), _ptr(dk_weight), *g, *x, _ptr(q_weight), _ptr(k_weight),
                        rope_cos.data_ptr(), rope_sin.data_ptr(), pos.data_ptr(), ws[0], ws[1], *dxs, *gs, *xs,
                        *sizes, eps, bool(accumulate))


def _glu_args(x, w_gate, w_up, act):
    if act not in _ACTS:
        raise ValueError(f"act {act!r}: expected one of {sorted(_ACTS)}")
    (n, k), dev, xs = _lead(x, "x", 2)
    dtype = x.dtype
    code = _type(x, "x")
    if code == 0:
        raise ValueError("x is torch.float32: expected float16 or bfloat16")
    m = w_gate.shape[0]
    gs = _check(w_gate, "w_gate", (m, k), dev, dtype)
    us = _check(w_up, "w_up", (m, k), dev, dtype)
    if k % 8 or m % 8 or not k or not m:
        raise ValueError(f"k = {k}, m = {m}: expected multiples of 8")
    return n, k, m, dev, dtype, code, (xs[0], gs[0], us[0])


def glu(out, x, w_gate, w_up, act="gelu_tanh"):
    """out = act(x w_gate^T) * (x w_up^T): x [n][k], weights [m][k], out [n][m], float16 or bfloat16.

    act is "gelu_tanh" or "silu"; k and m are multiples of 8, rows 16-byte aligned."""
    n, k, m, dev, dtype, code, strides = _glu_args(x, w_gate, w_up, act)
    out_stride = _check(out, "out", (n, m), dev, dtype)[0]
    _glu(dev, out.data_ptr(), x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), out_stride, *strides, n, k, m, code,
         _ACTS[act])


def glu_grad_workspace(n, k, m) -> int:
    """Bytes of workspace for glu_grad."""
    return int(_lib.load().eg2_glu_grad_workspace(n, k, m))


def glu_grad(dx, dw_gate, dw_up, dout, x, w_gate, w_up, act="gelu_tanh", accumulate=False, workspace=None):
    """The gradient of glu from dout [n][m] (None among dx, dw_gate, dw_up: not wanted).

    dout may be broadcast over tokens (row stride 0).
    The weights' gradients are of x's type or float32; with accumulate they are
    float32 and added to.  Nothing is kept from the forward pass: the
    projections are computed again, and their gradients are rounded to x's type
    (in float16 one above 65504 is infinite, and so are the rows it enters)."""
    n, k, m, dev, dtype, code, strides = _glu_args(x, w_gate, w_up, act)
    dout_stride = _check(dout, "dout", (n, m), dev, dtype)[0]
    # Where neither is wanted there is nothing to add to, and accumulate says nothing.
    dw_type = dw_gate.dtype if dw_gate is not None else dw_up.dtype if dw_up is not None else torch.float32
    if dw_type not in (torch.float32, dtype) or (accumulate and dw_type != torch.float32):
        raise ValueError(f"weight gradients are {dw_type}: expected float32" + ("" if accumulate else f" or {dtype}"))
    dx_stride = 0 if dx is None else _check(dx, "dx", (n, k), dev, dtype)[0]
    dg_stride = 0 if dw_gate is None else _check(dw_gate, "dw_gate", (m, k), dev, dw_type)[0]
    du_stride = 0 if dw_up is None else _check(dw_up, "dw_up", (m, k), dev, dw_type)[0]
    _apart(dw_gate, dw_up, "dw_gate and dw_up")
    ws = _workspace(workspace, glu_grad_workspace(n, k, m), dev)
    _glu_grad(dev, _ptr(dx), _ptr(dw_gate), _ptr(dw_up), dout.data_ptr(), x.data_ptr(), w_gate.data_ptr(),
              w_up.data_ptr(), ws[0], ws[1], dx_stride, dg_stride, du_stride, dout_stride, *strides, n, k, m, code,
              _ACTS[act], _TYPES[dw_type], bool(accumulate))


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
