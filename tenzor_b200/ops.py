"""Op-level entry points on device tensors (torch CUDA tensors are used only as device memory;
every computation runs in libtenzor_cuda.so).  Names follow the reference kernels they replace:

  layer_norm_last_dim   layernorm.zig:26-116          softmax_last_axis   softmax.zig:20-155
  linear (f32)          arctic.zig:599-620 / matmul.zig:54-77 (tcgen05 kind::tf32)
  linear_w8a32          matmul_w8a32.zig:14-58        linear_w8a8         (W8A8, no counterpart)
  gemm_i8_i32           exact int32 accumulators      quantize_weight_rows  quantize_arctic_xs.zig:94-115
  matmul_epilogue       codegen.zig:78-147            ew_add_mul_exp      executor.zig:114-197
  ew_unary_chain        codegen.zig:15-74             reduce              codegen.zig:151-205
  gather_rows           gather.zig:15-57
Gated feed-forward block (no counterpart in the reference): gated_linear, gated_linear_backward.
Microscaled 4-bit floating point (no counterpart): quantize_mxfp4, dequantize_mxfp4, linear_mxfp4,
pack_gated_mxfp4, gated_linear_mxfp4.
N-D forms (executor.zig / onnx/executor.zig): batched_matmul, matmul_f32x3, reduce_axis, softmax_axis,
permute, cast, concat.
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _lib as L
from .runtime import Context


def _p(t):
    return None if t is None else t.data_ptr()


CUDA_STREAM_LEGACY = 0x1  # cudaStreamLegacy: the handle torch's default stream (0) stands for


def _stream(s=None):
    """The stream to launch on: torch's current stream.  Its default stream has handle 0, which the C
    ABI reads as 'the context's own stream', so it is passed as cudaStreamLegacy instead."""
    h = torch._C._cuda_getCurrentRawStream(torch.cuda.current_device()) if s is None else s
    return h if h else CUDA_STREAM_LEGACY


def _dev(t, dtype):
    assert t.is_cuda and t.is_contiguous() and t.dtype == dtype, (t.device, t.dtype, t.is_contiguous())
    return t


def layer_norm_last_dim(ctx: Context, x, gamma, beta, eps: float, out=None):
    _dev(x, torch.float32)
    out = torch.empty_like(x) if out is None else out
    cols = x.shape[-1]
    L.check(L.lib().tz_layernorm_last_dim(ctx.handle, _p(x), _p(gamma), _p(beta), _p(out), x.numel() // cols,
                                          cols, eps, _stream()))
    return out


def softmax_last_axis(ctx: Context, x, mask=None, out=None):
    _dev(x, torch.float32)
    out = torch.empty_like(x) if out is None else out
    cols = x.shape[-1]
    L.check(L.lib().tz_softmax_last_axis(ctx.handle, _p(x), _p(mask), _p(out), x.numel() // cols, cols, _stream()))
    return out


def softmax_keylen(ctx: Context, x, key_len, out=None):
    """x [G, R, C]; group g keeps its first key_len[g] columns."""
    _dev(x, torch.float32)
    out = torch.empty_like(x) if out is None else out
    G, R, Cc = x.shape
    L.check(L.lib().tz_softmax_keylen(ctx.handle, _p(x), _p(key_len), _p(out), G, R, Cc, _stream()))
    return out


def attention(ctx: Context, qkv, cu_seqlens, max_len: int, out=None):
    """selfAttention (arctic.zig:639-747) over packed sequences: qkv [T, 1152] float16 or bfloat16
    (Q | K | V, 12 heads of 32), cu_seqlens int32 [B + 1] on the device; returns [T, 384] of qkv's type."""
    if qkv.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("attention: qkv must be float16 or bfloat16")
    _dev(qkv, qkv.dtype)
    _dev(cu_seqlens, torch.int32)
    T = qkv.shape[0]
    if qkv.shape != (T, 1152):
        raise ValueError(f"attention: qkv must be [T, 1152], got {tuple(qkv.shape)}")
    out = torch.empty((T, 384), device=qkv.device, dtype=qkv.dtype) if out is None else out
    L.check(L.lib().tz_attention(ctx.handle, _p(qkv), T, _p(cu_seqlens), cu_seqlens.numel() - 1, int(max_len), _p(out),
                                 int(qkv.dtype == torch.bfloat16), _stream()))
    return out


def linear(ctx: Context, x, w, bias=None, residual=None, out=None):
    m, k = x.shape
    n = w.shape[0]
    out = torch.empty((m, n), device=x.device, dtype=torch.float32) if out is None else out
    L.check(L.lib().tz_linear_f32(ctx.handle, _p(x), _p(w), _p(bias), _p(residual), _p(out), m, k, n, _stream()))
    return out


def linear_w8a32(ctx: Context, x, wq, scale_f16, bias, out=None):
    m, k = x.shape
    n = wq.shape[0]
    out = torch.empty((m, n), device=x.device, dtype=torch.float32) if out is None else out
    L.check(L.lib().tz_linear_w8a32(ctx.handle, _p(x), _p(wq), _p(scale_f16), _p(bias), _p(out), m, k, n, _stream()))
    return out


def linear_w8a8(ctx: Context, x, wq, scale_f16, bias, out=None):
    m, k = x.shape
    n = wq.shape[0]
    out = torch.empty((m, n), device=x.device, dtype=torch.float32) if out is None else out
    L.check(L.lib().tz_linear_w8a8(ctx.handle, _p(x), _p(wq), _p(scale_f16), _p(bias), _p(out), m, k, n, _stream()))
    return out


def gemm_i8_i32(ctx: Context, a, w, out=None):
    m, k = a.shape
    n = w.shape[0]
    out = torch.empty((m, n), device=a.device, dtype=torch.int32) if out is None else out
    L.check(L.lib().tz_gemm_i8_i32(ctx.handle, _p(a), _p(w), _p(out), m, k, n, _stream()))
    return out


def quantize_weight_rows(ctx: Context, w):
    rows, cols = w.shape
    q = torch.empty((rows, cols), device=w.device, dtype=torch.int8)
    s = torch.empty(rows, device=w.device, dtype=torch.int16)  # IEEE half bits
    L.check(L.lib().tz_quantize_weight_rows(ctx.handle, _p(w), _p(q), _p(s), rows, cols, _stream()))
    return q, s


def quantize_act_rows(ctx: Context, x):
    rows, cols = x.shape
    q = torch.empty((rows, cols), device=x.device, dtype=torch.int8)
    s = torch.empty(rows, device=x.device, dtype=torch.float32)
    L.check(L.lib().tz_quantize_act_rows(ctx.handle, _p(x), _p(q), _p(s), rows, cols, _stream()))
    return q, s


def matmul_epilogue(ctx: Context, a, b, bias, ops, trans_b=False, out=None):
    m, k = a.shape
    n = b.shape[0] if trans_b else b.shape[1]
    out = torch.empty((m, n), device=a.device, dtype=torch.float32) if out is None else out
    codes = (C.c_int * max(1, len(ops)))(*[L.OP[o] if isinstance(o, str) else int(o) for o in ops])
    L.check(L.lib().tz_matmul_epilogue(ctx.handle, _p(a), _p(b), int(trans_b), _p(bias), C.addressof(codes),
                                       len(ops), _p(out), m, k, n, _stream()))
    return out


def ew_add_mul_exp(ctx: Context, a, b_row, c, out=None):
    out = torch.empty_like(a) if out is None else out
    cols = b_row.numel()
    L.check(L.lib().tz_ew_add_mul_exp(ctx.handle, _p(a), _p(b_row), _p(c), _p(out), a.numel() // cols, cols,
                                      _stream()))
    return out


def ew_unary_chain(ctx: Context, x, ops, out=None):
    out = torch.empty_like(x) if out is None else out
    codes = (C.c_int * max(1, len(ops)))(*[L.OP[o] for o in ops])
    L.check(L.lib().tz_ew_unary_chain(ctx.handle, _p(x), _p(out), x.numel(), C.addressof(codes), len(ops),
                                      _stream()))
    return out


def reduce(ctx: Context, op: str, pre_ops, x):
    out = torch.empty(1, device=x.device, dtype=torch.float32)
    codes = (C.c_int * max(1, len(pre_ops)))(*[L.OP[o] for o in pre_ops])
    L.check(L.lib().tz_reduce(ctx.handle, L.RED[op], C.addressof(codes), len(pre_ops), _p(x), x.numel(), _p(out),
                              _stream()))
    return out


def gather_rows(ctx: Context, table, ids, out=None):
    rows, cols = table.shape
    out = torch.empty((ids.numel(), cols), device=table.device, dtype=torch.float32) if out is None else out
    L.check(L.lib().tz_gather_rows(ctx.handle, _p(table), rows, _p(ids), ids.numel(), cols, _p(out), _stream()))
    return out


# ---- N-D ops -------------------------------------------------------------------------------------
_TORCH_DT = {torch.float32: "f32", torch.float16: "f16", torch.int8: "i8", torch.int32: "i32",
             torch.int64: "i64", torch.uint8: "u8", torch.bool: "u8"}


def matmul_f32x3(ctx: Context, a, b, bias, ops, trans_b=False, out=None):
    """matmul_epilogue with f32-accurate products (split tf32 on the tensor cores)."""
    m, k = a.shape
    n = b.shape[0] if trans_b else b.shape[1]
    out = torch.empty((m, n), device=a.device, dtype=torch.float32) if out is None else out
    codes = (C.c_int * max(1, len(ops)))(*[L.OP[o] if isinstance(o, str) else int(o) for o in ops])
    L.check(L.lib().tz_matmul_f32x3(ctx.handle, _p(a), _p(b), int(trans_b), _p(bias), C.addressof(codes),
                                    len(ops), _p(out), m, k, n, _stream()))
    return out


def batched_matmul(ctx: Context, a, b, out_shape, batch_shape, a_bstride, b_bstride, m, k, n,
                   a_rs, a_cs, b_rs, b_cs, out=None, c_view=None):
    """Batched matmul on element strides (tz_batched_matmul).  The output is a new contiguous
    tensor of out_shape unless `out` is given with `c_view` = (c_bstride, c_rs, c_cs)."""
    if out is None:
        out = torch.empty(out_shape, device=a.device, dtype=torch.float32)
    lay = L.BmmLayout()
    lay.batch_ndim = len(batch_shape)
    if c_view is None:
        cb, acc = [], m * n
        for d in reversed(batch_shape):
            cb.append(acc)
            acc *= d
        c_view = (list(reversed(cb)), n, 1)
    for d, e in enumerate(batch_shape):
        lay.batch_shape[d] = e
        lay.a_bstride[d] = a_bstride[d]
        lay.b_bstride[d] = b_bstride[d]
        lay.c_bstride[d] = c_view[0][d]
    lay.a_rs, lay.a_cs, lay.b_rs, lay.b_cs = a_rs, a_cs, b_rs, b_cs
    lay.c_rs, lay.c_cs = c_view[1], c_view[2]
    lay.m, lay.k, lay.n = m, k, n
    L.check(L.lib().tz_batched_matmul(ctx.handle, _p(a), _p(b), _p(out), C.byref(lay), _stream()))
    return out


def _split_axis(shape, axis):
    axis = axis % len(shape) if shape else 0
    outer = 1
    for d in shape[:axis]:
        outer *= d
    inner = 1
    for d in shape[axis + 1:]:
        inner *= d
    return axis, outer, shape[axis], inner


def reduce_axis(ctx: Context, op: str, x, axis: int, keepdims=False):
    """reduceAxis (reduce.zig:52-95): one axis of a contiguous f32 tensor."""
    shape = list(x.shape)
    axis, outer, ln, inner = _split_axis(shape, axis)
    oshape = shape[:axis] + ([1] if keepdims else []) + shape[axis + 1:]
    out = torch.empty(oshape, device=x.device, dtype=torch.float32)
    L.check(L.lib().tz_reduce_axis(ctx.handle, L.RED[op], _p(x), outer, ln, inner, _p(out), _stream()))
    return out


def softmax_axis(ctx: Context, x, axis: int = -1, out=None):
    """softmaxAxis (softmax.zig:157-220)."""
    shape = list(x.shape)
    axis, outer, ln, inner = _split_axis(shape, axis)
    out = torch.empty_like(x) if out is None else out
    L.check(L.lib().tz_softmax_axis(ctx.handle, _p(x), _p(out), outer, ln, inner, _stream()))
    return out


def permute(ctx: Context, x, perm):
    """Transpose (onnx/executor.zig:2296): a contiguous copy of x.permute(perm)."""
    shape = list(x.shape)
    out = torch.empty([shape[p] for p in perm], device=x.device, dtype=x.dtype)
    sh = (C.c_int64 * max(1, len(shape)))(*shape)
    pm = (C.c_int * max(1, len(perm)))(*perm)
    L.check(L.lib().tz_permute(ctx.handle, _p(x), _p(out), x.element_size(), len(shape), C.addressof(sh),
                               C.addressof(pm), _stream()))
    return out


def cast(ctx: Context, x, dtype):
    """Cast (onnx/executor.zig:2852) on the device."""
    out = torch.empty(x.shape, device=x.device, dtype=dtype)
    L.check(L.lib().tz_cast(ctx.handle, _p(x), L.DT[_TORCH_DT[x.dtype]], _p(out), L.DT[_TORCH_DT[dtype]], x.numel(),
                            _stream()))
    return out


def concat(ctx: Context, xs, axis: int):
    """Concat (onnx/executor.zig:2112) of contiguous tensors of one dtype along `axis`."""
    shape = list(xs[0].shape)
    axis = axis % len(shape)
    outer = 1
    for d in shape[:axis]:
        outer *= d
    inner = 1
    for d in shape[axis + 1:]:
        inner *= d
    lens = [int(t.shape[axis]) for t in xs]
    oshape = shape[:axis] + [sum(lens)] + shape[axis + 1:]
    out = torch.empty(oshape, device=xs[0].device, dtype=xs[0].dtype)
    ptrs = (C.c_void_p * len(xs))(*[t.data_ptr() for t in xs])
    ln = (C.c_int64 * len(xs))(*lens)
    L.check(L.lib().tz_concat(ctx.handle, C.addressof(ptrs), C.addressof(ln), len(xs), outer, inner,
                              xs[0].element_size(), _p(out), _stream()))
    return out


# ---- gated feed-forward block ----------------------------------------------------------------------
GATED_ACTS = ("silu", "gelu", "gelu_erf", "relu", "sigmoid")
_ACT_CODE = {a: L.OP[a] for a in GATED_ACTS}
_DT16 = {torch.float16: 0, torch.bfloat16: 1}  # tz_gemm_prec


def _dtype16(fn, dtype):
    d = _DT16.get(dtype)
    if d is None:
        raise TypeError(f"{fn}: float16 or bfloat16 tensors, got {dtype}")
    return d


def _act_code(fn, act):
    c = _ACT_CODE.get(act)
    if c is None:
        raise ValueError(f"{fn}: activation {act!r} is not one of {GATED_ACTS}")
    return c


def _on(fn, ctx):
    """The stream to launch on: the current one of the context's device, which has to be the current device."""
    d = torch.cuda.current_device()
    if d != ctx.device:
        raise ValueError(f"{fn}: the context is on device {ctx.device}, the current device is {d}")
    return torch._C._cuda_getCurrentRawStream(d) or CUDA_STREAM_LEGACY


def _rows(fn, name, ctx, t, rows, cols, dtype):
    """Row stride of a matrix [rows, cols] on the context's device whose rows are contiguous."""
    if t.dtype is not dtype or t.shape != (rows, cols) or t.get_device() != ctx.device or (cols > 1 and t.stride(1) != 1):
        raise ValueError(f"{fn}: {name} must be a {dtype} tensor of shape {(rows, cols)} on device {ctx.device} with "
                         f"contiguous rows, got {t.dtype} {tuple(t.shape)} stride {t.stride()} on {t.device}")
    return t.stride(0) if rows > 1 else cols


def _full(fn, name, ctx, t, shape, dtype):
    if t.dtype is not dtype or t.shape != shape or t.get_device() != ctx.device or not t.is_contiguous():
        raise ValueError(f"{fn}: {name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on device {ctx.device}, "
                         f"got {t.dtype} {tuple(t.shape)} stride {t.stride()} on {t.device}")


def _two(fn, x, w):
    if x.dim() != 2 or w.dim() != 2:
        raise ValueError(f"{fn}: x [T, D] and weights [F, D], got {tuple(x.shape)} and {tuple(w.shape)}")


def gated_linear(ctx: Context, x, w_gate, w_up, act: str = "silu", out=None):
    """act(x @ w_gate.T) * (x @ w_up.T) in one kernel: x [T, D] (rows may be strided), w_gate and w_up [F, D],
    all float16 or all bfloat16, D and F multiples of 8; returns [T, F].  act: one of GATED_ACTS.  `out` shares no
    memory with the inputs."""
    dtype = x.dtype
    dt = _dtype16("gated_linear", dtype)
    code = _act_code("gated_linear", act)
    _two("gated_linear", x, w_gate)
    T, D = x.shape
    F = w_gate.shape[0]
    ldx = _rows("gated_linear", "x", ctx, x, T, D, dtype)
    _full("gated_linear", "w_gate", ctx, w_gate, (F, D), dtype)
    _full("gated_linear", "w_up", ctx, w_up, (F, D), dtype)
    if out is None:
        out = x.new_empty(T, F)
    else:
        _full("gated_linear", "out", ctx, out, (T, F), dtype)
    rc = L.lib().tz_gated_linear(ctx.ptr, x.data_ptr(), ldx, w_gate.data_ptr(), w_up.data_ptr(), out.data_ptr(), T, D, F,
                                 code, dt, _on("gated_linear", ctx))
    if rc:
        L.check(rc)
    return out


@functools.lru_cache(maxsize=4096)
def _gated_workspace(sms, t, d, f):
    need = C.c_size_t()
    L.check(L.lib().tz_gated_linear_backward_workspace(sms, t, d, f, C.byref(need)))
    return need.value


def gated_linear_backward(ctx: Context, x, w_gate, w_up, dh, act: str = "silu"):
    """(dx, dw_gate, dw_up) of gated_linear for the output's gradient dh [T, F] (rows may be strided)."""
    fn = "gated_linear_backward"
    dtype = x.dtype
    dt = _dtype16(fn, dtype)
    code = _act_code(fn, act)
    _two(fn, x, w_gate)
    T, D = x.shape
    F = w_gate.shape[0]
    ldx = _rows(fn, "x", ctx, x, T, D, dtype)
    lddh = _rows(fn, "dh", ctx, dh, T, F, dtype)
    _full(fn, "w_gate", ctx, w_gate, (F, D), dtype)
    _full(fn, "w_up", ctx, w_up, (F, D), dtype)
    stream = _on(fn, ctx)
    size = _gated_workspace(ctx.sm_count - ctx.sm_reserve, T, D, F)
    ws = x.new_empty(size, dtype=torch.uint8)
    dx, dwg, dwu = torch.empty_like(x, memory_format=torch.contiguous_format), torch.empty_like(w_gate), torch.empty_like(w_up)
    rc = L.lib().tz_gated_linear_backward(ctx.ptr, x.data_ptr(), ldx, w_gate.data_ptr(), w_up.data_ptr(), dh.data_ptr(), lddh,
                                          dx.data_ptr(), dwg.data_ptr(), dwu.data_ptr(), ws.data_ptr(), size, T, D, F, code, dt,
                                          stream)
    if rc:
        L.check(rc)
    return dx, dwg, dwu


# ---- microscaled 4-bit floating point --------------------------------------------------------------
_DTF = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # TZ_DT_*


class Mxfp4:
    """A matrix [rows, cols] in MXFP4 on the device: `codes` [rows, cols / 2] and the tiled `scales` (layout in
    tenzor_cuda.h), one allocation.  With `gated` the rows are two weight matrices interleaved by
    pack_gated_mxfp4."""

    __slots__ = ("buf", "rows", "cols", "gated", "index", "codes_ptr", "scales_ptr")

    def __init__(self, rows, cols, like, gated=False):
        self.rows, self.cols, self.gated = rows, cols, gated
        off, size = _mx_layout(rows, cols)
        self.buf = like.new_empty(size, dtype=torch.uint8)
        self.index = like.get_device()
        self.codes_ptr = self.buf.data_ptr()
        self.scales_ptr = self.codes_ptr + off

    @property
    def shape(self):
        return (self.rows, self.cols)

    @property
    def device(self):
        return self.buf.device

    @property
    def codes(self):
        return self.buf[:self.rows * (self.cols // 2)].view(self.rows, self.cols // 2)

    @property
    def scales(self):
        return self.buf[_mx_layout(self.rows, self.cols)[0]:]


def _mx_layout(rows, cols):
    """Byte offset of the scales behind the codes (256-byte aligned), and the bytes of both."""
    off = (rows * (cols // 2) + 255) // 256 * 256
    return off, off + (rows + 127) // 128 * ((cols + 127) // 128) * 512


def _dtype_f(fn, dtype):
    d = _DTF.get(dtype)
    if d is None:
        raise TypeError(f"{fn}: float32, float16 or bfloat16, got {dtype}")
    return d


def _mx_cols(fn, cols):
    if cols < 32 or cols % 32:
        raise ValueError(f"{fn}: the row length must be a positive multiple of 32, got {cols}")


def _mx(fn, name, ctx, q):
    if not isinstance(q, Mxfp4) or q.index != ctx.device:
        raise ValueError(f"{fn}: {name} must be an Mxfp4 on device {ctx.device}")


def quantize_mxfp4(ctx: Context, x) -> Mxfp4:
    """x [rows, cols] (float32, float16 or bfloat16; rows may be strided) in MXFP4, cols a multiple of 32."""
    dt = _dtype_f("quantize_mxfp4", x.dtype)
    if x.dim() != 2:
        raise ValueError(f"quantize_mxfp4: a matrix, got {tuple(x.shape)}")
    rows, cols = x.shape
    _mx_cols("quantize_mxfp4", cols)
    ldx = _rows("quantize_mxfp4", "x", ctx, x, rows, cols, x.dtype)
    stream = _on("quantize_mxfp4", ctx)
    q = Mxfp4(rows, cols, x)
    rc = L.lib().tz_quantize_mxfp4(ctx.ptr, x.data_ptr(), ldx, dt, q.codes_ptr, q.scales_ptr, rows, cols, stream)
    if rc:
        L.check(rc)
    return q


def dequantize_mxfp4(ctx: Context, q: Mxfp4, dtype=torch.float32):
    """The values q stands for, as [rows, cols] of `dtype`."""
    dt = _dtype_f("dequantize_mxfp4", dtype)
    _mx("dequantize_mxfp4", "q", ctx, q)
    if q.gated:
        raise ValueError("dequantize_mxfp4: a gated pair's rows are interleaved; quantise the matrices one by one")
    stream = _on("dequantize_mxfp4", ctx)
    out = q.buf.new_empty(q.rows, q.cols, dtype=dtype)
    rc = L.lib().tz_dequantize_mxfp4(ctx.ptr, q.codes_ptr, q.scales_ptr, out.data_ptr(), dt, q.rows, q.cols, stream)
    if rc:
        L.check(rc)
    return out


def pack_gated_mxfp4(ctx: Context, w_gate, w_up) -> Mxfp4:
    """w_gate and w_up [F, D] (F a multiple of 16, D of 32) as the weights of gated_linear_mxfp4."""
    fn = "pack_gated_mxfp4"
    dt = _dtype_f(fn, w_gate.dtype)
    if w_gate.dim() != 2 or w_gate.shape[0] % 16 or w_gate.shape[0] == 0:
        raise ValueError(f"{fn}: [F, D] with F a positive multiple of 16, got {tuple(w_gate.shape)}")
    F, D = w_gate.shape
    _mx_cols(fn, D)
    _full(fn, "w_gate", ctx, w_gate, (F, D), w_gate.dtype)
    _full(fn, "w_up", ctx, w_up, (F, D), w_gate.dtype)
    stream = _on(fn, ctx)
    q = Mxfp4(2 * F, D, w_gate, gated=True)
    L.check(L.lib().tz_pack_gated_mxfp4(ctx.ptr, w_gate.data_ptr(), w_up.data_ptr(), dt, q.codes_ptr, q.scales_ptr, F, D, stream))
    return q


@functools.lru_cache(maxsize=4096)
def _mx_workspace(m, k, n):
    need = C.c_size_t()
    L.check(L.lib().tz_linear_mxfp4_workspace(m, k, n, C.byref(need)))
    return need.value


def linear_mxfp4(ctx: Context, x, w: Mxfp4, bias=None, out_dtype=None, out=None):
    """q(x) @ w.T (+ bias f32 [N]): x [M, K] (float32, float16 or bfloat16, quantised in the call) or an Mxfp4;
    returns [M, N] of `out_dtype` (x's type; float32 for an Mxfp4).  N is a multiple of 8.  `out` shares no memory with
    the inputs."""
    fn = "linear_mxfp4"
    _mx(fn, "w", ctx, w)
    given = isinstance(x, Mxfp4)
    if w.gated or (given and x.gated):
        raise ValueError(f"{fn}: a gated pair of weights goes to gated_linear_mxfp4")
    if len(x.shape) != 2 or x.shape[1] != w.cols:
        raise ValueError(f"{fn}: x [M, {w.cols}], got {tuple(x.shape)}")
    M, K = x.shape
    N = w.rows
    if out_dtype is None:
        out_dtype = torch.float32 if given else x.dtype
    ydt = _dtype_f(fn, out_dtype)
    if bias is not None:
        _full(fn, "bias", ctx, bias, (N,), torch.float32)
        bias = bias.data_ptr()
    stream = _on(fn, ctx)
    if out is None:
        out = w.buf.new_empty(M, N, dtype=out_dtype) if given or x.dtype is not out_dtype else x.new_empty(M, N)
    else:
        _full(fn, "out", ctx, out, (M, N), out_dtype)
    if given:
        _mx(fn, "x", ctx, x)
        rc = L.lib().tz_gemm_mxfp4(ctx.ptr, x.codes_ptr, x.scales_ptr, w.codes_ptr, w.scales_ptr, bias, out.data_ptr(), ydt,
                                   M, K, N, stream)
    else:
        ldx = _rows(fn, "x", ctx, x, M, K, x.dtype)
        size = _mx_workspace(M, K, N)
        ws = x.new_empty(size, dtype=torch.uint8) if size else None
        rc = L.lib().tz_linear_mxfp4(ctx.ptr, x.data_ptr(), ldx, _dtype_f(fn, x.dtype), w.codes_ptr, w.scales_ptr, bias,
                                     out.data_ptr(), ydt, ws.data_ptr() if size else None, size, M, K, N, stream)
    if rc:
        L.check(rc)
    return out


def gated_linear_mxfp4(ctx: Context, x, w: Mxfp4, act: str = "silu", out=None):
    """act(q(x) @ wg.T) * (q(x) @ wu.T) with the weights of pack_gated_mxfp4: x [T, D] float16 or bfloat16;
    returns [T, F].  `out` shares no memory with the inputs."""
    fn = "gated_linear_mxfp4"
    dtype = x.dtype
    _dtype16(fn, dtype)
    code = _act_code(fn, act)
    _mx(fn, "w", ctx, w)
    if not w.gated:
        raise ValueError(f"{fn}: weights come from pack_gated_mxfp4")
    if x.dim() != 2 or x.shape[1] != w.cols:
        raise ValueError(f"{fn}: x [T, {w.cols}], got {tuple(x.shape)}")
    T, D = x.shape
    F = w.rows // 2
    ldx = _rows(fn, "x", ctx, x, T, D, dtype)
    stream = _on(fn, ctx)
    if out is None:
        out = x.new_empty(T, F)
    else:
        _full(fn, "out", ctx, out, (T, F), dtype)
    size = _mx_workspace(T, D, 2 * F)
    ws = x.new_empty(size, dtype=torch.uint8) if size else None
    rc = L.lib().tz_gated_linear_mxfp4(ctx.ptr, x.data_ptr(), ldx, _DTF[dtype], w.codes_ptr, w.scales_ptr, out.data_ptr(), code,
                                       ws.data_ptr() if size else None, size, T, D, F, stream)
    if rc:
        L.check(rc)
    return out
