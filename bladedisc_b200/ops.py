"""Operators of the quantized path on torch CUDA tensors.

Every function launches hand-written sm_100a kernels through the C ABI of
libdisc_b200_ral.so on torch's current stream.  torch is used for device
memory and streams only.  Nothing here computes on the CPU and nothing falls
back to torch operators.
"""
import ctypes
import math
from typing import NamedTuple, Optional, Tuple

import torch

from . import lib as _lib

_ACT = {None: _lib.ACT_NONE, "none": _lib.ACT_NONE, "gelu": _lib.ACT_GELU, "silu": _lib.ACT_SILU}
_OUT = {torch.int8: _lib.OUT_I8, torch.float16: _lib.OUT_F16, torch.float32: _lib.OUT_F32,
        torch.int32: _lib.OUT_I32}
_PATH = {None: _lib.PATH_AUTO, "auto": _lib.PATH_AUTO, "tiled": _lib.PATH_TILED,
         "small_m": _lib.PATH_SMALL_M, "simt": _lib.PATH_SIMT, "pair": _lib.PATH_PAIR,
         "gemv": _lib.PATH_GEMV, "skinny": _lib.PATH_SKINNY}
_scratch = {}


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _cuda(t: torch.Tensor, name: str, dtype=None) -> torch.Tensor:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor: the quantized path has no CPU implementation")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    return t.contiguous()


def _etype(t: torch.Tensor) -> int:
    if t.dtype == torch.float32:
        return _lib.F32
    if t.dtype == torch.float16:
        return _lib.F16
    raise TypeError(f"float32 or float16 expected, got {t.dtype}")


def qgemm_scratch(device: torch.device, nbytes: int) -> torch.Tensor:
    """Zero-initialised scratch of the small-M path, one per (device, stream)."""
    key = (device.index, _stream())
    buf = _scratch.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.zeros(max(nbytes, 8 << 20), dtype=torch.uint8, device=device)
        _scratch[key] = buf
    return buf


def _scale_kind(s: Optional[torch.Tensor], rows: int, cols: int, what: str, x_per_col: bool) -> int:
    if s is None:
        return _lib.SCALE_NONE
    if s.numel() == 1:
        return _lib.SCALE_SCALAR
    if what == "x" and not x_per_col:
        if s.numel() != rows:
            raise ValueError(f"x_scale has {s.numel()} entries; expected 1 or one per row ({rows})")
        return _lib.SCALE_PER_ROW
    if s.numel() != cols:
        raise ValueError(f"{what}_scale has {s.numel()} entries; expected 1 or one per channel ({cols})")
    return _lib.SCALE_PER_COL


def qgemm(a: torch.Tensor, w: torch.Tensor, *, x_scale: Optional[torch.Tensor] = None,
          w_scale: Optional[torch.Tensor] = None, out_scale: Optional[torch.Tensor] = None,
          bias: Optional[torch.Tensor] = None, act: Optional[str] = None,
          out_dtype: torch.dtype = torch.int8, fold_out_scale: bool = False,
          x_scale_per_col: bool = False, path: Optional[str] = None, split_k: int = 0,
          out: Optional[torch.Tensor] = None, a_gathered: bool = False,
          weights_static: bool = False, exact_division: bool = False) -> torch.Tensor:
    """out = epilogue(a[..., K] @ w[N, K]^T) with int8 operands and int32 accumulation.

    ``fold_out_scale=True`` is the reference custom call ``ral_pdll_qgemm``:
    ``sat_s8(rne(acc * (x_scale * w_scale / out_scale) + bias))``.  Otherwise
    ``v = act(acc * x_scale * w_scale + bias)`` and int8 output divides ``v`` by
    ``out_scale`` before rounding: as a product with the correctly rounded
    reciprocal (at most one int8 level from the quotient, at rounding ties only),
    or, with ``exact_division=True``, as the IEEE quotient the reference's
    quantize computes, bit for bit.  Scales and bias are device tensors.

    ``a_gathered=True``: ``a`` is ``[g, M, K / g]``, the buffer an all-gather of
    column-parallel outputs leaves (slab ``r`` holds columns ``r * K / g ...``);
    it is consumed in place, the result is ``[M, N]``.

    ``weights_static=True`` promises that ``w`` was final before the previous
    kernel on the stream was launched (inference weights): the few-row paths
    then fetch it while that kernel still runs.
    """
    if a_gathered:
        # a block of rows of a gathered buffer ([:, m0:m1, :]) is accepted as it is
        if not a.is_cuda or a.dtype != torch.int8:
            raise TypeError("a must be a CUDA int8 tensor")
        if a.dim() == 3 and (a.stride(2) != 1 or a.stride(1) != a.shape[2]):
            a = a.contiguous()
    else:
        a = _cuda(a, "a", torch.int8)
    w = _cuda(w, "w", torch.int8)
    if a_gathered:
        if a.dim() != 3 or w.dim() != 2 or a.shape[0] * a.shape[2] != w.shape[1]:
            raise ValueError(f"shape mismatch: gathered a {tuple(a.shape)} w {tuple(w.shape)}")
    elif w.dim() != 2 or a.shape[-1] != w.shape[1]:
        raise ValueError(f"shape mismatch: a {tuple(a.shape)} w {tuple(w.shape)}")
    K = w.shape[1]
    N = w.shape[0]
    M = a.numel() // K if K else 0
    out_shape = ((a.shape[1],) if a_gathered else tuple(a.shape[:-1])) + (N,)
    if out is None:
        out = torch.empty(out_shape, dtype=out_dtype, device=a.device)
    elif out.dtype != out_dtype or not out.is_contiguous() or out.numel() != M * N:
        raise ValueError("out must be a contiguous tensor of the result's dtype and size")
    if M == 0 or N == 0:
        return out
    args = _lib.QGemmArgs()
    args.a, args.w, args.out = a.data_ptr(), w.data_ptr(), out.data_ptr()
    args.M, args.N, args.K = M, N, K
    args.lda, args.ldw, args.ldo = K, K, N
    if a_gathered:
        args.a_slabs, args.a_slab_cols, args.a_slab_stride = a.shape[0], a.shape[2], a.stride(0)
        args.lda = a.shape[2]
    args.weights_static = 1 if weights_static else 0
    keep = []
    for name, t in (("x", x_scale), ("w", w_scale), ("out", out_scale)):
        if t is not None:
            t = _cuda(t, f"{name}_scale", torch.float32)
            keep.append(t)
        kind = _scale_kind(t, M, N, name, x_scale_per_col)
        setattr(args, f"{name}_scale", _p(t))
        setattr(args, f"{name}_scale_kind", kind)
    if bias is not None:
        bias = _cuda(bias, "bias")
        if bias.dtype == torch.float32:
            args.bias_kind = _lib.BIAS_F32
        elif bias.dtype == torch.int8:
            args.bias_kind = _lib.BIAS_I8
        else:
            raise TypeError("bias must be float32 or int8")
        if bias.numel() != N:
            raise ValueError("bias must have one entry per output channel")
        args.bias = bias.data_ptr()
    args.fold_out_scale = 1 if fold_out_scale else 0
    args.div_out_scale = 1 if (out_dtype == torch.int8 and out_scale is not None and not fold_out_scale) else 0
    args.div_exact = 1 if exact_division else 0
    args.act = _ACT[act]
    args.out_dtype = _OUT[out_dtype]
    args.path = _PATH[path]
    args.split_k = split_k
    L = _lib.load()
    if M <= 128:
        need = L.disc_b200_qgemm_scratch_bytes(M, N, K)
        ws = qgemm_scratch(a.device, need)
        args.splitk_ws = ws.data_ptr()
        args.splitk_ws_bytes = ws.numel()
    _lib.check(L.disc_b200_qgemm(ctypes.byref(args), _stream()))
    return out


def qgemm_path(M: int, N: int, K: int) -> str:
    """Which kernel path an aligned (M, N, K) problem takes."""
    args = _lib.QGemmArgs()
    args.a, args.w, args.out = 16, 16, 16
    args.M, args.N, args.K, args.lda, args.ldw, args.ldo = M, N, K, K, K, N
    code = _lib.load().disc_b200_qgemm_path(ctypes.byref(args))
    return {1: "tiled", 2: "small_m", 3: "simt", 4: "pair", 5: "gemv", 6: "skinny"}[code]


def quantize(x: torch.Tensor, scale: torch.Tensor, zero_point: Optional[torch.Tensor] = None,
             axis: Optional[int] = None, qmin: int = -128, qmax: int = 127) -> torch.Tensor:
    """q = clamp(rne(x / scale + zero_point), qmin, qmax) as int8 (static scales)."""
    x = _cuda(x, "x")
    scale = _cuda(scale, "scale", torch.float32)
    if zero_point is not None:
        zero_point = _cuda(zero_point, "zero_point", torch.int32)
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    channels, inner = 1, 1
    if axis is not None and scale.numel() > 1:
        axis = axis % x.dim()
        channels = x.shape[axis]
        inner = 1
        for d in x.shape[axis + 1:]:
            inner *= d
        if scale.numel() != channels:
            raise ValueError("scale must have one entry per slice along axis")
    _lib.check(_lib.load().disc_b200_quantize(x.data_ptr(), _etype(x), q.data_ptr(), x.numel(),
                                              scale.data_ptr(), _p(zero_point), channels, inner,
                                              qmin, qmax, _stream()))
    return q


def dequantize(q: torch.Tensor, scale: torch.Tensor, zero_point: Optional[torch.Tensor] = None,
               axis: Optional[int] = None, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """y = (q - zero_point) * scale."""
    q = _cuda(q, "q", torch.int8)
    scale = _cuda(scale, "scale", torch.float32)
    if zero_point is not None:
        zero_point = _cuda(zero_point, "zero_point", torch.int32)
    y = torch.empty(q.shape, dtype=dtype, device=q.device)
    channels, inner = 1, 1
    if axis is not None and scale.numel() > 1:
        axis = axis % q.dim()
        channels = q.shape[axis]
        for d in q.shape[axis + 1:]:
            inner *= d
    _lib.check(_lib.load().disc_b200_dequantize(q.data_ptr(), y.data_ptr(), _etype(y), q.numel(),
                                                scale.data_ptr(), _p(zero_point), channels, inner,
                                                _stream()))
    return y


def dynamic_quantize(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Per-row symmetric int8: returns (q, row_scale) with row_scale = max|row| / 127."""
    x = _cuda(x, "x")
    cols = x.shape[-1]
    rows = x.numel() // cols if cols else 0
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    s = torch.empty(rows, dtype=torch.float32, device=x.device)
    _lib.check(_lib.load().disc_b200_dynamic_quantize(x.data_ptr(), _etype(x), q.data_ptr(),
                                                      s.data_ptr(), rows, cols, _stream()))
    return q, s


def _norm(x, residual, gamma, beta, eps, rms, q_scale, want_y, want_sum, want_q, dynamic_q,
          x_gathered=False):
    x = _cuda(x, "x")
    gamma = _cuda(gamma, "gamma", x.dtype)
    a = _lib.NormArgs()
    if x_gathered:  # [g, rows, cols / g] column slabs
        if x.dim() != 3:
            raise ValueError("a gathered x is [g, rows, cols / g]")
        rows, cols = x.shape[1], x.shape[0] * x.shape[2]
        a.x_slab_cols, a.x_slab_stride = x.shape[2], x.shape[1] * x.shape[2]
        shape = (rows, cols)
    else:
        cols = x.shape[-1]
        rows = x.numel() // cols if cols else 0
        shape = tuple(x.shape)
    a.x = x.data_ptr()
    a.gamma = gamma.data_ptr()
    keep = [x, gamma]
    if residual is not None:
        residual = _cuda(residual, "residual", x.dtype)
        if tuple(residual.shape) != shape:
            raise ValueError("residual must have the shape of x")
        a.residual = residual.data_ptr()
        keep.append(residual)
    if beta is not None:
        beta = _cuda(beta, "beta", x.dtype)
        a.beta = beta.data_ptr()
        keep.append(beta)
    y = s = q = rs = None
    if want_y:
        y = torch.empty(shape, dtype=x.dtype, device=x.device)
        a.y = y.data_ptr()
    if want_sum:
        s = torch.empty(shape, dtype=x.dtype, device=x.device)
        a.sum_out = s.data_ptr()
    if want_q:
        q = torch.empty(shape, dtype=torch.int8, device=x.device)
        a.q_out = q.data_ptr()
        if dynamic_q:
            rs = torch.empty(rows, dtype=torch.float32, device=x.device)
            a.q_row_scale = rs.data_ptr()
        else:
            q_scale = _cuda(q_scale, "q_scale", torch.float32)
            a.q_scale = q_scale.data_ptr()
            keep.append(q_scale)
    a.rows, a.cols, a.eps, a.type, a.rms = rows, cols, eps, _etype(x), 1 if rms else 0
    _lib.check(_lib.load().disc_b200_norm(ctypes.byref(a), _stream()))
    return y, s, q, rs


def layernorm(x, gamma, beta, eps: float = 1e-5, residual=None) -> torch.Tensor:
    """LayerNorm(x [+ residual]) over the last axis."""
    return _norm(x, residual, gamma, beta, eps, False, None, True, False, False, False)[0]


def layernorm_quant(x, gamma, beta, q_scale, eps: float = 1e-5, residual=None):
    """LayerNorm(x [+ residual]) and its int8 copy at a static scale: (y, q)."""
    y, _, q, _ = _norm(x, residual, gamma, beta, eps, False, q_scale, True, False, True, False)
    return y, q


def rmsnorm(x, gamma, eps: float = 1e-6, residual=None, return_sum: bool = False, x_gathered: bool = False):
    """RMSNorm(x [+ residual]); with return_sum also x + residual."""
    y, s, _, _ = _norm(x, residual, gamma, None, eps, True, None, True, return_sum, False, False,
                       x_gathered=x_gathered)
    return (y, s) if return_sum else y


def rmsnorm_dynamic_quant(x, gamma, eps: float = 1e-6, residual=None, x_gathered: bool = False):
    """RMSNorm(x [+ residual]) quantized per row: (q, row_scale, x + residual or None).

    ``x_gathered``: x is ``[g, rows, cols / g]``, the buffer an all-gather of
    column-parallel outputs leaves; it is read in place."""
    _, s, q, rs = _norm(x, residual, gamma, None, eps, True, None, False, residual is not None, True, True,
                        x_gathered=x_gathered)
    return q, rs, s


def _gated(gate, up, q, row_scale, pass_):
    gate = _cuda_strided(gate, "gate")
    a = _lib.GatedQuantArgs()
    a.gate, a.ld = gate.data_ptr(), gate.stride(0)
    a.rows, a.cols, a.type, a.pass_ = gate.shape[0], gate.shape[1], _etype(gate), pass_
    if up is not None:
        up = _cuda_strided(up, "up")
        if up.shape != gate.shape or up.stride(0) != gate.stride(0) or up.dtype != gate.dtype:
            raise ValueError("up must match gate in shape, row stride and dtype")
        a.up = up.data_ptr()
    a.row_scale = row_scale.data_ptr()
    if q is not None:
        a.q, a.ldq = q.data_ptr(), q.stride(0)
    _lib.check(_lib.load().disc_b200_gated_quantize(ctypes.byref(a), _stream()))


def _cuda_strided(t: torch.Tensor, name: str) -> torch.Tensor:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor: this library has no CPU path")
    if t.dim() != 2 or t.stride(1) != 1:
        raise ValueError(f"{name} must be 2-D with unit column stride")
    return t


def quantize_rows_whole(gate: torch.Tensor, up: Optional[torch.Tensor] = None,
                        out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Both passes in one kernel for rows that are whole on this GPU: ``(q, row_scale)``."""
    s = torch.empty(gate.shape[0], dtype=torch.float32, device=gate.device)
    if out is None:
        out = torch.empty(gate.shape, dtype=torch.int8, device=gate.device)
    elif out.dtype != torch.int8 or tuple(out.shape) != tuple(gate.shape) or out.stride(1) != 1:
        raise ValueError("out must be int8 of gate's shape with unit column stride")
    _gated(gate, up, out, s, 2)
    return out, s


def row_scale_local(gate: torch.Tensor, up: Optional[torch.Tensor] = None) -> torch.Tensor:
    """First pass of the two-pass per-row quantization of ``h = silu(gate) * up``
    (``h = gate`` without ``up``): ``max(max|h[r, :]| / 127, eps)`` over the
    columns this GPU holds.  Rows may be strided views (column halves of one buffer)."""
    s = torch.empty(gate.shape[0], dtype=torch.float32, device=gate.device)
    _gated(gate, up, None, s, 0)
    return s


def quantize_rows(gate: torch.Tensor, row_scale: torch.Tensor, up: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Second pass: ``sat(rne(h / row_scale[r]))`` into ``out`` (int8, may be a strided view)."""
    row_scale = _cuda(row_scale, "row_scale", torch.float32)
    if out is None:
        out = torch.empty(gate.shape, dtype=torch.int8, device=gate.device)
    elif out.dtype != torch.int8 or tuple(out.shape) != tuple(gate.shape) or out.stride(1) != 1:
        raise ValueError("out must be int8 of gate's shape with unit column stride")
    _gated(gate, up, out, row_scale, 1)
    return out


def weight_only_qgemm(x: torch.Tensor, w: torch.Tensor, scale: torch.Tensor, zero_point: Optional[torch.Tensor] = None,
                      bias: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                      path: Optional[str] = None) -> torch.Tensor:
    """``x @ ((w - zero_point) * scale) + bias`` with ``w`` uint8 ``[K, N]`` (the transposed
    weight the reference's pattern hands to ``ral_pdll_weight_only_qgemm``), ``scale`` /
    ``bias`` of ``x``'s dtype (float16 or float32) ``[N]``, ``zero_point`` int32 ``[N]``.
    Dequantization happens in the kernel; sums are fp32.  ``path``: None (by shape),
    "stream" or "tensor" (fp16, 16-byte aligned operands, N a multiple of 16)."""
    x = _cuda(x, "x")
    w = _cuda(w, "w", torch.uint8)
    if w.dim() != 2 or x.shape[-1] != w.shape[0]:
        raise ValueError("w must be [K, N] with K = x.shape[-1]")
    K, N = w.shape
    M = math.prod(x.shape[:-1])
    scale = _cuda(scale, "scale", x.dtype)
    if scale.numel() != N:
        raise ValueError("one scale per output column expected")
    if zero_point is not None:
        zero_point = _cuda(zero_point, "zero_point", torch.int32)
        if zero_point.numel() != N:
            raise ValueError("one zero point per output column expected")
    if bias is not None:
        bias = _cuda(bias, "bias", x.dtype)
        if bias.numel() != N:
            raise ValueError("one bias per output column expected")
    if out is None:
        out = torch.empty(x.shape[:-1] + (N,), dtype=x.dtype, device=x.device)
    elif out.dtype != x.dtype or not out.is_contiguous() or out.numel() != M * N:
        raise ValueError("out must be contiguous, of x's dtype and [..., N]")
    L = _lib.load()
    a = _lib.WeightOnlyQGemmArgs()
    a.x, a.w, a.scale, a.zero_point, a.bias, a.out = x.data_ptr(), w.data_ptr(), scale.data_ptr(), _p(zero_point), \
        _p(bias), out.data_ptr()
    a.m, a.n, a.k, a.ldx, a.ldw, a.ldo = M, N, K, K, N, N
    a.type = _etype(x)
    a.path = {None: 0, "stream": 1, "tensor": 2}[path]
    _lib.check(L.disc_b200_weight_only_qgemm(ctypes.byref(a), _stream()))
    return out


def qconv2d_plan(data_format: str, input_shape, weight_shape, strides=(1,), dilations=(1,), padding="VALID",
                 explicit_paddings=(), weight_is_const: bool = True):
    """(padding (top, bottom, left, right), result shape, metadata) of a quantized convolution from the
    attributes of ``ral_pdll_qconv2d``; host only."""
    L = _lib.load()
    arr = lambda v: (ctypes.c_int64 * max(len(v), 1))(*[int(i) for i in v])
    pad = (ctypes.c_int32 * 4)()
    res = (ctypes.c_int64 * 4)()
    meta = (ctypes.c_int32 * 17)()
    _lib.check(L.disc_b200_qconv2d_plan(data_format.encode(), arr(strides), len(strides), arr(dilations),
                                        len(dilations), padding.encode(), arr(explicit_paddings),
                                        len(explicit_paddings), 1 if weight_is_const else 0, arr(input_shape),
                                        arr(weight_shape), pad, res, meta))
    return tuple(pad), tuple(res), tuple(meta)


def qconv2d(x: torch.Tensor, w: torch.Tensor, x_scale: torch.Tensor, w_scale: torch.Tensor, out_scale: torch.Tensor,
            data_format: str = "NHWC", strides=(1,), dilations=(1,), padding="VALID",
            explicit_paddings=()) -> torch.Tensor:
    """int8 convolution ``sat(rne(conv(x, w) * (x_scale * w_scale / out_scale)))``: ``x`` int8 in ``data_format``,
    ``w`` int8 ``[out, y, x, in]``, scales float32 CUDA tensors (``w_scale``: one value or one per output
    channel); ``padding`` "SAME" | "VALID" | "EXPLICIT" with the reference's rules."""
    x = _cuda(x, "x", torch.int8)
    w = _cuda(w, "w", torch.int8)
    if x.dim() != 4 or w.dim() != 4:
        raise ValueError("rank-4 input and kernel expected")
    x_scale, w_scale, out_scale = (_cuda(t, n, torch.float32) for t, n in
                                   ((x_scale, "x_scale"), (w_scale, "w_scale"), (out_scale, "out_scale")))
    pad, res, meta = qconv2d_plan(data_format, x.shape, w.shape, strides, dilations, padding, explicit_paddings)
    out = torch.empty(res, dtype=torch.int8, device=x.device)
    if out.numel() == 0 or x.numel() == 0:
        return out
    if w_scale.numel() not in (1, w.shape[0]):
        raise ValueError("w_scale must hold one value or one per output channel")
    L = _lib.load()
    a = _lib.QConv2dArgs()
    a.x, a.w, a.out = x.data_ptr(), w.data_ptr(), out.data_ptr()
    a.input_sizes[:] = list(x.shape)
    a.kernel_sizes[:] = list(w.shape)
    a.output_sizes[:] = list(res)
    a.padding[:] = list(pad)
    a.metadata[:] = list(meta[:16])
    a.x_scale, a.w_scale, a.out_scale = x_scale.data_ptr(), w_scale.data_ptr(), out_scale.data_ptr()
    a.w_scale_per_channel = 1 if w_scale.numel() > 1 else 0
    need = L.disc_b200_qconv2d_workspace_bytes(ctypes.byref(a))
    if need < 0:
        raise ValueError("shapes, padding and metadata do not describe a convolution (one group only)")
    work = torch.empty(need, dtype=torch.uint8, device=x.device)
    rows = out.numel() // w.shape[0]
    kp = (w.shape[1] * w.shape[2] * w.shape[3] + 15) // 16 * 16
    ws = qgemm_scratch(x.device, L.disc_b200_qgemm_scratch_bytes(rows, w.shape[0], kp))
    a.workspace, a.workspace_bytes = work.data_ptr(), need
    a.splitk_ws, a.splitk_ws_bytes = ws.data_ptr(), ws.numel()
    _lib.check(L.disc_b200_qconv2d(ctypes.byref(a), _stream()))
    return out


def softmax(x: torch.Tensor, scale: float = 1.0, lens: Optional[torch.Tensor] = None,
            mask: Optional[torch.Tensor] = None, log: bool = False) -> torch.Tensor:
    """softmax(x * scale + mask) over the last axis.

    ``lens`` (int32, one per index of the leading axis) zeroes the columns at
    and beyond the length; ``mask`` ([leading, cols], dtype of x) is added.
    """
    x = _cuda(x, "x")
    cols = x.shape[-1]
    rows = x.numel() // cols if cols else 0
    y = torch.empty_like(x)
    rpb = rows
    if lens is not None:
        lens = _cuda(lens, "lens", torch.int32)
        if lens.numel() != x.shape[0]:
            raise ValueError("one length per index of the leading axis expected")
        rpb = rows // x.shape[0]
    if mask is not None:
        mask = _cuda(mask, "mask", x.dtype)
        if mask.numel() != x.shape[0] * cols:
            raise ValueError("mask must be [leading axis, cols]")
        rpb = rows // x.shape[0]
    _lib.check(_lib.load().disc_b200_softmax(x.data_ptr(), y.data_ptr(), _etype(x), rows, cols, rpb,
                                             _p(lens), _p(mask), float(scale), 1 if log else 0,
                                             _stream()))
    return y


def attention_blocks(lens, heads: int = 12, group: int = 1) -> torch.Tensor:
    """Work list of `attention` for sequences packed one after the other (host tensor, int32 [n, 4]): one row
    {first token of the sequence, length, first query row of the item, query blocks of the item} per item.
    An item is `group` (or, at the end of a sequence, fewer) consecutive blocks of 128 query rows of a
    sequence; its thread block fetches the sequence's keys and values once.  Which size is fastest depends on
    the batch: with many more items than SMs whole-sequence items win (34 vs 43 us on 32 sequences of up to
    512 tokens), on a few sequences one block per item does (9 vs 28 us on 4 sequences).  Longer items come
    first; the kernel starts all heads of an item before the next item."""
    lens = [int(v) for v in lens]
    for n in lens:
        if n < 1 or n > 512:
            raise ValueError(f"sequence length {n} outside 1..512")
    group = max(1, min(4, int(group)))
    rows = []
    tok0 = 0
    for n in lens:
        nblk = (n + 127) // 128
        for b0 in range(0, nblk, group):
            rows.append((tok0, n, b0 * 128, min(group, nblk - b0)))
        tok0 += n
    rows.sort(key=lambda r: -(r[1] * r[3]))
    return torch.tensor(rows, dtype=torch.int32).reshape(-1, 4)


def attention(qkv: torch.Tensor, blocks: torch.Tensor, heads: int, scale: float,
              out_scale: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(q k^T * scale) v per head over packed sequences, in one kernel.

    ``qkv``: f16 [tokens, 3 * heads * 64]; ``blocks``: device copy of ``attention_blocks(lens)``.
    Returns [tokens, heads * 64]: int8 quantized at ``out_scale`` (a device scalar), f16 without it."""
    qkv = _cuda(qkv, "qkv", torch.float16)
    if qkv.dim() != 2 or qkv.shape[1] != 3 * heads * 64:
        raise ValueError(f"qkv must be [tokens, {3 * heads * 64}], got {tuple(qkv.shape)}")
    if not blocks.is_cuda or blocks.dtype != torch.int32 or blocks.dim() != 2 or blocks.shape[1] != 4:
        raise ValueError("blocks must be a CUDA int32 [n, 4] tensor (see attention_blocks)")
    tokens = qkv.shape[0]
    hidden = heads * 64
    dtype = torch.int8 if out_scale is not None else torch.float16
    if out is None:
        out = torch.empty((tokens, hidden), dtype=dtype, device=qkv.device)
    elif out.dtype != dtype or tuple(out.shape) != (tokens, hidden) or not out.is_contiguous():
        raise ValueError("out must be a contiguous [tokens, hidden] tensor of the result's dtype")
    args = _lib.AttentionArgs()
    args.qkv, args.tokens, args.ld_qkv, args.heads = qkv.data_ptr(), tokens, qkv.shape[1], heads
    blocks = blocks.contiguous()
    args.blocks, args.num_blocks, args.scale = blocks.data_ptr(), blocks.shape[0], float(scale)
    args.out, args.ld_out = out.data_ptr(), hidden
    if out_scale is not None:
        out_scale = _cuda(out_scale, "out_scale", torch.float32)
        args.out_scale = out_scale.data_ptr()
    _lib.check(_lib.load().disc_b200_attention(ctypes.byref(args), _stream()))
    return out


def rope_kv_append(qkv: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, cos: torch.Tensor,
                   sin: torch.Tensor, batch: int, seq: int, pos0: int) -> None:
    """Rotates q and k inside ``qkv`` (fp16 ``[batch * seq, 3 * heads * dim]``, q in place) and
    appends the rotated k and v to the caches ``[batch, heads, cache_len, dim]`` at ``pos0``."""
    for t, n in ((qkv, "qkv"), (k_cache, "k_cache"), (v_cache, "v_cache")):
        if not t.is_cuda or t.dtype != torch.float16 or not t.is_contiguous():
            raise ValueError(f"{n} must be a contiguous CUDA fp16 tensor")
    heads, cache_len, dim = k_cache.shape[1], k_cache.shape[2], k_cache.shape[3]
    if qkv.numel() != batch * seq * 3 * heads * dim or k_cache.shape[0] != batch or v_cache.shape != k_cache.shape:
        raise ValueError("qkv / cache shapes disagree")
    cos, sin = _cuda(cos, "cos", torch.float32), _cuda(sin, "sin", torch.float32)
    if cos.shape[0] < pos0 + seq or cos.shape[1] != dim // 2 or sin.shape != cos.shape:
        raise ValueError("cos / sin tables must be [>= pos0 + seq, dim / 2]")
    _lib.check(_lib.load().disc_b200_rope_kv_append(qkv.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                                                    cos.data_ptr(), sin.data_ptr(), batch, seq, heads, dim, pos0,
                                                    cache_len, _stream()))


# ---------------------------------------------------------------- paged key / value cache in 8 bits
class KvPlan(NamedTuple):
    """What `kv_blocks_extend` says about one batch of new tokens (int32 CUDA tensors)."""
    slots: torch.Tensor      # [max_tokens] slot of each token row, -1 = none
    positions: torch.Tensor  # [max_tokens] position in its request, -1 = none
    q_start: torch.Tensor    # [requests + 1] first token row of each request
    q_lens: torch.Tensor     # [requests] tokens that found room (all that were asked for, or 0)
    kv_lens: torch.Tensor    # [requests] cached tokens with the new ones


def _one_device(*tensors) -> int:
    """Ordinal of the CUDA device that all of them (None aside) are on."""
    dev = tensors[0].get_device()
    if dev < 0:
        raise ValueError("the paged cache lives on CUDA tensors: there is no CPU implementation")
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"a tensor is on {t.device}, not on cuda:{dev} like the others")
    return dev


def _call(dev: int, fn, args) -> None:
    """Launches on the current stream of device `dev`, whichever device is current."""
    stream = torch._C._cuda_getCurrentRawStream(dev)
    if torch._C._cuda_getDevice() == dev:
        code = fn(args, stream)
    else:
        with torch.cuda.device(dev):
            code = fn(args, stream)
    if code:
        _lib.check(code)


def _is(t: torch.Tensor, dtype: torch.dtype, dims: int) -> bool:
    return t.dtype is dtype and t.dim() == dims and t.is_contiguous()


def _dense(name: str, t: torch.Tensor, dtype: torch.dtype, dims: int) -> None:
    if not _is(t, dtype, dims):
        raise ValueError(f"{name} must be a contiguous {dtype} tensor with {dims} dimension(s), got {t.dtype} "
                         f"{tuple(t.shape)} with strides {t.stride()}")


def _kv_blocks_args(tokens, lens, table, free_list, free_count, block_size):
    dev = _one_device(lens, tokens, table, free_list, free_count)
    i32 = torch.int32
    if not (_is(tokens, i32, 1) and _is(lens, i32, 1) and _is(table, i32, 2) and _is(free_list, i32, 1)):
        for name, t, dims in (("tokens", tokens, 1), ("lens", lens, 1), ("table", table, 2),
                              ("free_list", free_list, 1)):
            _dense(name, t, i32, dims)
    if free_count.dtype != torch.int32 or free_count.numel() != 1:
        raise ValueError("free_count must be one int32 value")
    n = lens.numel()
    rows, width = table.shape
    if not 0 < block_size < 1 << 31:
        raise ValueError("block_size must be positive")
    if tokens.numel() != n or rows != n:
        raise ValueError("tokens, lens and table must have one entry (row) per request")
    a = _lib.KvBlocksArgs(tokens.data_ptr(), lens.data_ptr(), table.data_ptr(), free_list.data_ptr(),
                          free_count.data_ptr(), n, width, free_list.numel(), block_size)
    return dev, a


def kv_blocks_extend(tokens: torch.Tensor, lens: torch.Tensor, table: torch.Tensor, free_list: torch.Tensor,
                     free_count: torch.Tensor, block_size: int, max_tokens: int) -> KvPlan:
    """Makes room for ``tokens[r]`` new tokens of each request: pops blocks off the stack
    ``free_list[:free_count]``, enters them into ``table [requests, width]`` and grows ``lens`` (all int32, updated
    in place), and returns where every token of the batch goes.  The batch holds the tokens of the requests one
    after the other; ``max_tokens`` is the number of rows it has room for.

    A request is refused as a whole (``q_lens`` 0, slots -1, nothing else changed) when the blocks for it and for
    all requests before it are not there, its table row is too short, or its rows end behind ``max_tokens``."""
    dev, a = _kv_blocks_args(tokens, lens, table, free_list, free_count, block_size)
    n, cap = lens.numel(), int(max_tokens)
    if not 0 <= cap < 1 << 31:
        raise ValueError("max_tokens must not be negative, nor pass 32 bits")
    buf = lens.new_empty(2 * cap + 3 * n + 1)
    out = KvPlan(*torch.unsafe_split_with_sizes(buf, (cap, cap, n + 1, n, n)))
    at = buf.data_ptr()
    a.max_tokens = cap
    a.slots, a.positions, a.q_start = at, at + 4 * cap, at + 8 * cap
    a.q_lens, a.kv_lens = at + 4 * (2 * cap + n + 1), at + 4 * (2 * cap + 2 * n + 1)
    _call(dev, _lib.load().disc_b200_kv_blocks_extend, a)
    return out


def kv_blocks_trim(keep: torch.Tensor, lens: torch.Tensor, table: torch.Tensor, free_list: torch.Tensor,
                   free_count: torch.Tensor, block_size: int) -> None:
    """Keeps the first ``keep[r]`` cached tokens of each request (0 releases it) and gives the blocks behind them
    back to the stack, in place.  Trimming to the lengths before a `kv_blocks_extend` undoes it exactly; scales and levels
    that a `kv8_append` changed in a block that keeps tokens stay as they are."""
    dev, a = _kv_blocks_args(keep, lens, table, free_list, free_count, block_size)
    _call(dev, _lib.load().disc_b200_kv_blocks_trim, a)


_KV_TYPE = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def _kv8_cache(k, v, k_scale, v_scale) -> "_lib.Kv8Cache":
    i8, f32 = torch.int8, torch.float32
    if not (_is(k, i8, 4) and _is(v, i8, 4) and _is(k_scale, f32, 2) and _is(v_scale, f32, 2)):
        for name, t, dtype, dims in (("k", k, i8, 4), ("v", v, i8, 4), ("k_scale", k_scale, f32, 2),
                                     ("v_scale", v_scale, f32, 2)):
            _dense(name, t, dtype, dims)
    blocks, heads, size, dim = shape = k.shape
    if v.shape != shape or k_scale.shape != shape[:2] or v_scale.shape != shape[:2]:
        raise ValueError("k and v must be [blocks, kv heads, block size, head size], their scales [blocks, kv heads]")
    return _lib.Kv8Cache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), blocks, heads, size, dim)


def _kv_type(name: str, dtype: torch.dtype) -> int:
    if dtype not in _KV_TYPE:
        raise TypeError(f"{name} must be float16 or bfloat16, got {dtype}")
    return _KV_TYPE[dtype]


def kv8_append(qkv: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
               slots: torch.Tensor, positions: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None,
               sin: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Quantizes the new keys and values of ``qkv [tokens, (q heads + 2 kv heads) * head size]`` (float16 or
    bfloat16, rows may be strided) into one layer of the cache, in place, after rotating q and k by ``cos`` / ``sin``
    (float32 ``[positions, head size / 2]``) when those are given.  Returns q ``[tokens, q heads, head size]``,
    rotated (a view of ``qkv`` without ``cos``), or None if there are no query heads.

    The cache is ``k``, ``v`` int8 ``[blocks, kv heads, block size, head size]`` with ``k_scale``, ``v_scale`` float32
    ``[blocks, kv heads]``: a block and a head share the scale ``max|x| / 127`` of the tokens stored since its first one,
    tokens that a trim took back among them; tokens that the block held before are moved to the new scale when it grows,
    and a value that is not finite makes them NaN until the block is begun anew.  ``slots`` and ``positions`` are those of
    `kv_blocks_extend` (the first ``tokens`` entries are read; slot -1 = not stored)."""
    dev = _one_device(k, qkv, v, k_scale, v_scale, slots, positions, cos, sin)
    cache = _kv8_cache(k, v, k_scale, v_scale)
    kind = _kv_type("qkv", qkv.dtype)
    if qkv.dim() != 2 or (qkv.shape[0] > 1 and qkv.stride(0) < qkv.shape[1]) or (qkv.numel() and qkv.stride(1) != 1):
        raise ValueError("qkv must be [tokens, columns] with unit column stride and rows that do not overlap")
    tokens, cols = qkv.shape
    dim, kv_heads = cache.dim, cache.kv_heads
    if cols % dim or cols < 2 * kv_heads * dim:
        raise ValueError(f"qkv rows of {cols} values do not hold whole heads of {dim} beside {kv_heads} + {kv_heads}")
    q_heads = cols // dim - 2 * kv_heads
    _dense("slots", slots, torch.int32, 1)
    if slots.numel() < tokens:
        raise ValueError("one slot per token expected")
    ld = qkv.stride(0) if tokens > 1 else cols
    a = _lib.Kv8AppendArgs(qkv.data_ptr(), tokens, ld, q_heads, kind, None, slots.data_ptr())
    a.cache = cache
    q = None
    if cos is not None or sin is not None:
        if cos is None or sin is None or positions is None:
            raise ValueError("a rotation needs cos, sin and positions")
        _dense("cos", cos, torch.float32, 2)
        _dense("sin", sin, torch.float32, 2)
        _dense("positions", positions, torch.int32, 1)
        if cos.shape[1] != dim // 2 or cos.shape != sin.shape or cos.shape[0] < 1 or positions.numel() < tokens:
            raise ValueError("cos / sin must be [positions, head size / 2], positions one per token")
        a.positions, a.cos_table, a.sin_table = positions.data_ptr(), cos.data_ptr(), sin.data_ptr()
        a.table_rows = cos.shape[0]
        if q_heads:
            q = qkv.new_empty(tokens, q_heads, dim)
            a.q_out = q.data_ptr()
    elif q_heads:
        q = qkv[:, :q_heads * dim].unflatten(1, (q_heads, dim))
    _call(dev, _lib.load().disc_b200_kv8_append, a)
    return q


def kv8_read(k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, blocks: torch.Tensor,
             dtype: torch.dtype = torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The given blocks (int32 ids) of one layer as the values they stand for: keys and values of ``dtype``
    ``[len(blocks), kv heads, block size, head size]``; zeros for an id outside the cache."""
    dev = _one_device(k, v, k_scale, v_scale, blocks)
    a = _lib.Kv8ReadArgs(_kv8_cache(k, v, k_scale, v_scale))
    _dense("blocks", blocks, torch.int32, 1)
    a.type = _kv_type("dtype", dtype)
    a.blocks, a.count = blocks.data_ptr(), blocks.numel()
    _, heads, size, dim = k.shape
    ko = k.new_empty(blocks.numel(), heads, size, dim, dtype=dtype)
    vo = torch.empty_like(ko)
    a.k_out, a.v_out = ko.data_ptr(), vo.data_ptr()
    _call(dev, _lib.load().disc_b200_kv8_read, a)
    return ko, vo


def kv8_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                  table: torch.Tensor, q_start: torch.Tensor, q_lens: torch.Tensor, kv_lens: torch.Tensor, *,
                  max_q: int, scale: Optional[float] = None, max_kv: Optional[int] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of ``q [tokens, q heads, head size]`` over one layer of the 8-bit cache.

    Request ``r`` has the rows ``q_start[r] ... q_start[r] + q_lens[r] - 1`` of ``q``, its last tokens; they see its
    ``kv_lens[r]`` cached tokens (their own included: append first) up to their own position.  Requests may not share
    rows; rows of a request behind the end of ``q`` are not there.  The index tensors
    are int32 and stay on the device; ``max_q`` bounds ``q_lens`` and shapes the launch (rows behind it are not
    computed), ``max_kv`` bounds ``kv_lens`` and only steers how the work is split (default: the table's width).
    Query heads are a multiple of the kv heads.  ``scale`` defaults to ``head size ** -0.5``.  Rows that belong to
    no request are left as ``out`` had them; a row that sees no key gives zeros.  ``out`` may not overlap ``q``."""
    dev = _one_device(q, k, v, k_scale, v_scale, table, q_start, q_lens, kv_lens, out)
    cache = _kv8_cache(k, v, k_scale, v_scale)
    kind = _kv_type("q", q.dtype)
    dim = cache.dim
    if q.dim() != 3 or q.shape[2] != dim or q.shape[1] < 1 or q.shape[1] % cache.kv_heads:
        raise ValueError(f"q must be [tokens, heads, {dim}] with a multiple of {cache.kv_heads} heads, got "
                         f"{tuple(q.shape)}")
    tokens, heads, _ = q.shape
    if not q.is_contiguous() and q.numel() and (q.stride(2) != 1 or (heads > 1 and q.stride(1) != dim) or
                      (tokens > 1 and q.stride(0) < heads * dim)):
        raise ValueError("the heads of a row of q must lie one after the other, and rows may not overlap")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.dtype != q.dtype or out.shape != q.shape or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor of q's shape and dtype")
    i32 = torch.int32
    if not (_is(table, i32, 2) and _is(q_start, i32, 1) and _is(q_lens, i32, 1) and _is(kv_lens, i32, 1)):
        for name, t, dims in (("table", table, 2), ("q_start", q_start, 1), ("q_lens", q_lens, 1),
                              ("kv_lens", kv_lens, 1)):
            _dense(name, t, i32, dims)
    n = q_lens.numel()
    rows, width = table.shape
    if kv_lens.numel() != n or rows != n or q_start.numel() < n:
        raise ValueError("q_start, q_lens, kv_lens and table must have one entry (row) per request")
    room = width * cache.block_size
    if max_kv is None or max_kv > room:
        max_kv = room
    if max_q < 0 or max_kv < 0:
        raise ValueError("max_q and max_kv must not be negative")
    if max_q > tokens:  # no request has more rows than there are
        max_q = tokens
    a = _lib.Kv8AttentionArgs(q.data_ptr(), out.data_ptr(), tokens, q.stride(0) if tokens > 1 else heads * dim,
                              heads * dim, heads, kind, cache, table.data_ptr(), q_start.data_ptr(),
                              q_lens.data_ptr(), kv_lens.data_ptr(), n, width, max_q, max_kv,
                              dim ** -0.5 if scale is None else scale)
    lib = _lib.load()
    if max_kv > _lib.KV8_DIRECT_KEYS:
        if torch._C._cuda_getDevice() == dev:
            need = lib.disc_b200_kv8_attention_workspace_bytes(a)
        else:
            with torch.cuda.device(dev):
                need = lib.disc_b200_kv8_attention_workspace_bytes(a)
        if need:  # from torch's allocator: ordered with this stream, a captured graph keeps its own
            work = k.new_empty(need)
            a.workspace, a.workspace_bytes = work.data_ptr(), need
    _call(dev, lib.disc_b200_kv8_attention, a)
    return out


def kernel_status() -> int:
    """0 unless a kernel's bounded wait ran out since the last query (synchronises)."""
    return _lib.load().disc_b200_kernel_status()
