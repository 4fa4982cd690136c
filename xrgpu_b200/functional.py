"""Zero-copy PyTorch entry points over the C ABI (``xrgpu_mmnb_forward``, ``xrgpu_mxfp4_*``, ``xrgpu_kv8_*``, ...).

Tensors stay on the device; the kernels run on the current torch CUDA stream. torch
supplies device memory and streams only: every numerical step runs in this package's
CUDA kernels.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _native
from ._native import check

_PATHS = {"auto": _native.PATH_AUTO, "generic": _native.PATH_GENERIC, "gemv": _native.PATH_GEMV,
          "gemm": _native.PATH_GEMM}


def _dtype_code(t: torch.dtype) -> int:
    if t == torch.float32:
        return _native.FLOAT32
    if t == torch.float16:
        return _native.FLOAT16
    raise ValueError(f"MatMulNBits T1 must be float32 or float16, got {t}")


def _zp_code(zp: Optional[torch.Tensor]) -> int:
    if zp is None:
        return _native.UNSPECIFIED
    if zp.dtype == torch.uint8:
        return _native.UINT8
    if zp.dtype == torch.float32:
        return _native.FLOAT32
    if zp.dtype == torch.float16:
        return _native.FLOAT16
    raise ValueError("zero_points must be float32/float16 (contract) or packed uint8")


def _ptr(t: Optional[torch.Tensor]):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def _problem(a, b, scales, zero_points, bias, y, *, K, N, bits, block_size, path, ldy=0, dtype=None):
    p = _native.Problem_()
    p.dtype = _dtype_code(dtype if dtype is not None else a.dtype)
    p.zero_point_dtype = _zp_code(zero_points)
    p.path = _PATHS[path]
    p.M = 0 if a is None else a.numel() // K
    p.K, p.N, p.block_size, p.bits = int(K), int(N), int(block_size), int(bits)
    p.a, p.b, p.scales = _ptr(a), _ptr(b), _ptr(scales)
    p.zero_points, p.bias, p.y = _ptr(zero_points), _ptr(bias), _ptr(y)
    p.ldy = int(ldy)
    return p


def _require(t: Optional[torch.Tensor], name: str, device):
    if t is None:
        return
    if not t.is_cuda or t.device != device:
        raise ValueError(f"{name} must be a CUDA tensor on {device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def matmul_nbits(a: torch.Tensor, b: torch.Tensor, scales: torch.Tensor, zero_points: Optional[torch.Tensor] = None,
                 bias: Optional[torch.Tensor] = None, *, K: Optional[int] = None, N: Optional[int] = None,
                 bits: int = 4, block_size: int = 32, out: Optional[torch.Tensor] = None, path: str = "auto",
                 workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Y = A . dequant(B)^T (+ bias) for com.microsoft.MatMulNBits on the current CUDA stream.

    Shapes: a [..., K] (T1), b uint8 [N, ceil(K/bs), ceil(bs*bits/8)], scales [N, ceil(K/bs)] (T1),
    zero_points float [N, ceil(K/bs)] or packed uint8 [N, ceil(ceil(K/bs)*bits/8)], bias [N] (T1).
    ``out`` may be a [..., >=N] view whose last-dim stride is 1 (rows may be strided).
    """
    K = int(a.shape[-1]) if K is None else int(K)
    N = int(b.shape[0]) if N is None else int(N)
    dev = a.device
    for t, name in ((a, "a"), (b, "b"), (scales, "scales"), (zero_points, "zero_points"), (bias, "bias")):
        _require(t, name, dev)
    if out is None:
        out = torch.empty(tuple(a.shape[:-1]) + (N,), dtype=a.dtype, device=dev)
        ldy = N
    else:
        if out.dtype != a.dtype or out.device != dev or out.stride(-1) != 1 or out.shape[-1] != N:
            raise ValueError("out must match a's dtype/device, end with N columns and have unit column stride")
        ldy = out.stride(-2) if out.dim() >= 2 else N
    p = _problem(a, b, scales, zero_points, bias, out, K=K, N=N, bits=bits, block_size=block_size, path=path, ldy=ldy)
    lib = _native.load()
    stream = torch.cuda.current_stream(dev).cuda_stream
    ws_ptr, ws_bytes = None, 0
    if workspace is not None:
        ws_ptr, ws_bytes = ctypes.c_void_p(workspace.data_ptr()), workspace.numel() * workspace.element_size()
    if torch.cuda.current_device() == dev.index:
        check(lib.xrgpu_mmnb_forward(ctypes.byref(p), ws_ptr, ws_bytes, ctypes.c_void_p(stream)))
    else:
        with torch.cuda.device(dev):
            check(lib.xrgpu_mmnb_forward(ctypes.byref(p), ws_ptr, ws_bytes, ctypes.c_void_p(stream)))
    return out


def workspace_size(a_rows: int, *, K: int, N: int, bits: int = 4, block_size: int = 32, dtype=torch.float16,
                   zero_points_dtype=None, path: str = "auto") -> int:
    """Device scratch bytes ``matmul_nbits`` needs for this shape (0 when none)."""
    p = _native.Problem_()
    p.dtype = _dtype_code(dtype)
    p.zero_point_dtype = {None: _native.UNSPECIFIED, torch.uint8: _native.UINT8, torch.float32: _native.FLOAT32,
                          torch.float16: _native.FLOAT16}[zero_points_dtype]
    p.path = _PATHS[path]
    p.M, p.K, p.N, p.block_size, p.bits = int(a_rows), int(K), int(N), int(block_size), int(bits)
    p.a = p.b = p.scales = p.y = ctypes.c_void_p(256)
    if zero_points_dtype is not None:
        p.zero_points = ctypes.c_void_p(256)
    need = ctypes.c_uint64(0)
    check(_native.load().xrgpu_mmnb_workspace_size(ctypes.byref(p), ctypes.byref(need)))
    return int(need.value)


def select_path(a: torch.Tensor, b, scales, zero_points=None, *, K=None, N=None, bits=4, block_size=32,
                path: str = "auto") -> str:
    K = int(a.shape[-1]) if K is None else int(K)
    N = int(b.shape[0]) if N is None else int(N)
    p = _problem(a, b, scales, zero_points, None, None, K=K, N=N, bits=bits, block_size=block_size, path=path)
    buf = ctypes.create_string_buffer(32)
    check(_native.load().xrgpu_mmnb_select_path(ctypes.byref(p), buf, len(buf)))
    return buf.value.decode()


def dequantize(b: torch.Tensor, scales: torch.Tensor, zero_points: Optional[torch.Tensor] = None, *, K: int,
               bits: int = 4, block_size: int = 32) -> torch.Tensor:
    """Exact float32 W[N, K] = (float(q) - z) * s on the device (nbitWeight)."""
    N = int(b.shape[0])
    dev = b.device
    for t, name in ((b, "b"), (scales, "scales"), (zero_points, "zero_points")):
        _require(t, name, dev)
    w = torch.empty((N, K), dtype=torch.float32, device=dev)
    p = _problem(None, b, scales, zero_points, None, None, K=K, N=N, bits=bits, block_size=block_size, path="auto",
                 dtype=scales.dtype)
    stream = torch.cuda.current_stream(dev).cuda_stream
    with torch.cuda.device(dev):
        check(_native.load().xrgpu_mmnb_dequantize(ctypes.byref(p), ctypes.c_void_p(w.data_ptr()),
                                                    ctypes.c_void_p(stream)))
    return w


def device_error(device: int = 0, clear: bool = True) -> int:
    code = ctypes.c_uint32(0)
    check(_native.load().xrgpu_device_error(int(device), ctypes.byref(code), int(clear)))
    return int(code.value)


# ---------------------------------------------------------------------------------------------
# Operators around MatMulNBits (zero-copy, current CUDA stream).
_ACTIVATIONS = {"none": 0, "identity": 0, "relu": 1, "silu": 2, "swish": 2, "gelu": 3, "tanh": 4, "sigmoid": 5,
                "swiglu": 6}


def _act_code(activation) -> int:
    if isinstance(activation, int):
        return activation
    if activation not in _ACTIVATIONS:
        raise ValueError(f"Unknown fused activation: {activation}")
    return _ACTIVATIONS[activation]


def _workspace(nbytes: int, device) -> Optional[torch.Tensor]:
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=device) if nbytes else None


def _call(fn, prob, ws, device):
    stream = torch.cuda.current_stream(device).cuda_stream
    args = [ctypes.byref(prob)]
    if ws is not False:
        args += [ctypes.c_void_p(ws.data_ptr()) if ws is not None else None,
                 (ws.numel() if ws is not None else 0)]
    args.append(ctypes.c_void_p(stream))
    with torch.cuda.device(device):
        check(fn(*args))


def matmul_nbits_mlp(a, gate_b, gate_scales, up_b, up_scales, *, skip=None, norm_scale=None, gate_bias=None,
                     up_bias=None, K: Optional[int] = None, N: Optional[int] = None, bits: int = 4, block_size: int = 32,
                     activation="silu", epsilon: float = 1e-5, want_residual: bool = False):
    """com.microsoft.MatMulNBitsMlp: y = fused(x.gate^T + gate_bias) * (x.up^T + up_bias), x = a + skip,
    RMS-normalised by norm_scale when given. Returns y, or (y, residual) with want_residual."""
    K = int(a.shape[-1]) if K is None else int(K)
    N = int(gate_b.shape[0]) if N is None else int(N)
    dev = a.device
    for t, n in ((a, "a"), (gate_b, "gate_b"), (gate_scales, "gate_scales"), (up_b, "up_b"), (up_scales, "up_scales"),
                 (skip, "skip"), (norm_scale, "norm_scale"), (gate_bias, "gate_bias"), (up_bias, "up_bias")):
        _require(t, n, dev)
    y = torch.empty(tuple(a.shape[:-1]) + (N,), dtype=a.dtype, device=dev)
    res = torch.empty_like(a) if want_residual else None
    p = _native.MlpProblem_()
    p.dtype = _dtype_code(a.dtype)
    p.activation = _act_code(activation)
    p.M, p.K, p.N, p.block_size, p.bits = a.numel() // K, K, N, int(block_size), int(bits)
    p.epsilon = float(epsilon)
    p.a, p.skip, p.norm_scale = _ptr(a), _ptr(skip), _ptr(norm_scale)
    p.gate_b, p.gate_scales, p.gate_bias = _ptr(gate_b), _ptr(gate_scales), _ptr(gate_bias)
    p.up_b, p.up_scales, p.up_bias = _ptr(up_b), _ptr(up_scales), _ptr(up_bias)
    p.y, p.residual = _ptr(y), _ptr(res)
    lib = _native.load()
    need = ctypes.c_uint64(0)
    check(lib.xrgpu_mlp_workspace_size(ctypes.byref(p), ctypes.byref(need)))
    _call(lib.xrgpu_mlp_forward, p, _workspace(need.value, dev), dev)
    return (y, res) if want_residual else y


def matmul_nbits_qkv(a, norm_scale, q_b, q_scales, k_b, k_scales, v_b, v_scales, *, skip=None, K: Optional[int] = None,
                     Nq: Optional[int] = None, Nkv: Optional[int] = None, bits: int = 4, block_size: int = 32,
                     epsilon: float = 1e-6, want_residual: bool = False):
    """com.microsoft.MatMulNBitsQkv: q, k, v = x.W^T with x = RMSNorm(a + skip) * norm_scale.
    Returns (q, k, v) or (q, k, v, residual)."""
    K = int(a.shape[-1]) if K is None else int(K)
    Nq = int(q_b.shape[0]) if Nq is None else int(Nq)
    Nkv = int(k_b.shape[0]) if Nkv is None else int(Nkv)
    dev = a.device
    for t, n in ((a, "a"), (norm_scale, "norm_scale"), (skip, "skip"), (q_b, "q_b"), (q_scales, "q_scales"),
                 (k_b, "k_b"), (k_scales, "k_scales"), (v_b, "v_b"), (v_scales, "v_scales")):
        _require(t, n, dev)
    lead = tuple(a.shape[:-1])
    q = torch.empty(lead + (Nq,), dtype=a.dtype, device=dev)
    k = torch.empty(lead + (Nkv,), dtype=a.dtype, device=dev)
    v = torch.empty(lead + (Nkv,), dtype=a.dtype, device=dev)
    res = torch.empty_like(a) if want_residual else None
    p = _native.QkvProblem_()
    p.dtype = _dtype_code(a.dtype)
    p.M, p.K, p.Nq, p.Nkv, p.block_size, p.bits = a.numel() // K, K, Nq, Nkv, int(block_size), int(bits)
    p.epsilon = float(epsilon)
    p.a, p.skip, p.norm_scale = _ptr(a), _ptr(skip), _ptr(norm_scale)
    p.q_b, p.q_scales, p.k_b, p.k_scales, p.v_b, p.v_scales = (_ptr(q_b), _ptr(q_scales), _ptr(k_b), _ptr(k_scales),
                                                               _ptr(v_b), _ptr(v_scales))
    p.q, p.k, p.v, p.residual = _ptr(q), _ptr(k), _ptr(v), _ptr(res)
    lib = _native.load()
    need = ctypes.c_uint64(0)
    check(lib.xrgpu_qkv_workspace_size(ctypes.byref(p), ctypes.byref(need)))
    _call(lib.xrgpu_qkv_forward, p, _workspace(need.value, dev), dev)
    return (q, k, v, res) if want_residual else (q, k, v)


def matmul_bnb4(a, b, absmax, *, K: int, N: int, block_size: int, quant_type: int = 1):
    """com.microsoft.MatMulBnb4 (transB = 1): NF4 (quant_type 1) or FP4 (0) codebook weights."""
    dev = a.device
    for t, n in ((a, "a"), (b, "b"), (absmax, "absmax")):
        _require(t, n, dev)
    y = torch.empty(tuple(a.shape[:-1]) + (int(N),), dtype=a.dtype, device=dev)
    p = _native.Bnb4Problem_()
    p.dtype = _dtype_code(a.dtype)
    p.quant_type = int(quant_type)
    p.M, p.K, p.N, p.block_size = a.numel() // int(K), int(K), int(N), int(block_size)
    p.a, p.b, p.absmax, p.y = _ptr(a), _ptr(b), _ptr(absmax), _ptr(y)
    _call(_native.load().xrgpu_bnb4_forward, p, False, dev)
    return y


def gather_block_quantized(data, indices, scales, zero_points=None, *, bits: int = 4, block_size: int = 128):
    """com.microsoft.GatherBlockQuantized (gather_axis 0, quantize_axis 1): float32 rows
    (q - z) * scale of the selected rows. Out-of-range indices leave zeros and device error 55."""
    dev = data.device
    for t, n in ((data, "data"), (indices, "indices"), (scales, "scales"), (zero_points, "zero_points")):
        _require(t, n, dev)
    if indices.dtype not in (torch.int64, torch.int32):
        raise ValueError("indices must be int64 or int32")
    width = data.shape[1] * (8 // int(bits))
    out = torch.empty((indices.numel(), width), dtype=torch.float32, device=dev)
    p = _native.GatherProblem_()
    p.bits = int(bits)
    p.index_dtype = _native.INT64 if indices.dtype == torch.int64 else _native.INT32
    p.rows, p.row_bytes, p.count, p.block_size = data.shape[0], data.shape[1], indices.numel(), int(block_size)
    p.data, p.indices, p.scales, p.zero_points, p.out = _ptr(data), _ptr(indices), _ptr(scales), _ptr(zero_points), _ptr(out)
    _call(_native.load().xrgpu_gather_block_quantized_forward, p, False, dev)
    return out


def qmoe(x, router, fc1, fc1_scales, fc2, fc2_scales, *, k: int = 1, bits: int = 4, block_size: int = 0,
         activation="relu", swiglu_fusion: int = 0, activation_alpha: float = 1.0, activation_beta: float = 0.0,
         swiglu_limit: Optional[float] = None):
    """com.microsoft.QMoE (float32): top-k routing, symmetric int4/int8 expert weights, relu or swiglu."""
    dev = x.device
    for t, n in ((x, "x"), (router, "router"), (fc1, "fc1"), (fc1_scales, "fc1_scales"), (fc2, "fc2"),
                 (fc2_scales, "fc2_scales")):
        _require(t, n, dev)
    hidden = int(x.shape[-1])
    out = torch.empty_like(x)
    p = _native.QmoeProblem_()
    p.bits, p.activation, p.swiglu_fusion = int(bits), _act_code(activation), int(swiglu_fusion)
    p.has_swiglu_limit = int(swiglu_limit is not None)
    p.tokens, p.hidden, p.experts, p.k = x.numel() // hidden, hidden, int(router.shape[1]), int(k)
    p.fc1_rows, p.block_size = int(fc1.shape[1]), int(block_size)
    p.activation_alpha, p.activation_beta = float(activation_alpha), float(activation_beta)
    p.swiglu_limit = float(swiglu_limit or 0.0)
    p.input, p.router, p.fc1, p.fc1_scales = _ptr(x), _ptr(router), _ptr(fc1), _ptr(fc1_scales)
    p.fc2, p.fc2_scales, p.output = _ptr(fc2), _ptr(fc2_scales), _ptr(out)
    lib = _native.load()
    need = ctypes.c_uint64(0)
    check(lib.xrgpu_qmoe_workspace_size(ctypes.byref(p), ctypes.byref(need)))
    _call(lib.xrgpu_qmoe_forward, p, _workspace(need.value, dev), dev)
    return out


# ---------------------------------------------------------------------------------------------
# Block-scaled serving operators: microscaled 4-bit floating point, and the paged key/value cache of
# 8-bit codes with its attention (zero-copy, current CUDA stream of the tensors' device).
_FLOATS = {torch.float32: _native.FLOAT32, torch.float16: _native.FLOAT16}
_CACHES = {torch.int8: _native.INT8, torch.float8_e4m3fn: _native.FLOAT8_E4M3}


# Handle of a device's current stream, without the Stream object around it (these calls are launch-bound).
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _launch(index: int, fn, *args):
    """fn(*args, stream) on the current stream of device `index`, with that device current."""
    if torch.cuda.current_device() == index:
        check(fn(*args, _current_stream(index)))
    else:
        with torch.cuda.device(index):
            check(fn(*args, _current_stream(index)))


def _workspace_bytes(index: int, size, p) -> int:
    """What `size` asks for the call p on device `index` (it may depend on the current device's number of SMs)."""
    need = ctypes.c_uint64(0)
    if torch.cuda.current_device() == index:
        check(size(ctypes.byref(p), ctypes.byref(need)))
    else:
        with torch.cuda.device(index):
            check(size(ctypes.byref(p), ctypes.byref(need)))
    return need.value


def _device_of(t: torch.Tensor, name: str) -> int:
    index = t.get_device()
    if index < 0:
        raise ValueError(f"{name} must be a CUDA tensor")
    return index


def _on(t: torch.Tensor, name: str, dtype, index: int):
    if t.get_device() != index:
        raise ValueError(f"{name} must be a CUDA tensor on cuda:{index}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _float_code(dtype) -> int:
    if dtype not in _FLOATS:
        raise ValueError(f"T1 must be float32 or float16, got {dtype}")
    return _FLOATS[dtype]


def _row_stride(t: torch.Tensor, name: str) -> int:
    """Elements from one row of [..., K] to the next; the rows must lie at one stride, values side by side."""
    if t.is_contiguous():
        return t.shape[-1]
    if t.stride(-1) != 1:
        raise ValueError(f"{name} must have unit stride in its last dimension")
    step = want = 0
    for d in range(t.dim() - 2, -1, -1):
        if t.shape[d] == 1:
            continue
        if step == 0:
            step = want = t.stride(d)
        if t.stride(d) != want or step < t.shape[-1]:
            raise ValueError(f"{name} must have its rows at one stride")
        want *= t.shape[d]
    return step or t.shape[-1]


def _scale_shape(rows: int, kb: int):
    return (-(-rows // 128), -(-kb // 4), 32, 4, 4)


def _require_mxfp4(codes, scales, rows: int, kb: int, name: str, index: int):
    _on(codes, name, torch.uint8, index)
    _on(scales, name + "_scales", torch.uint8, index)
    if codes.dim() < 2 or tuple(codes.shape[-2:]) != (kb, 16) or codes.numel() != rows * kb * 16:
        raise ValueError(f"{name} must be [..., {kb}, 16] codes")
    if scales.shape != _scale_shape(rows, kb):
        raise ValueError(f"{name}_scales must be tiled scales of shape {list(_scale_shape(rows, kb))}")


def mxfp4_quantize(x: torch.Tensor):
    """Microscaled 4-bit form of x [..., K] (float32 or float16; rows may be strided): (codes, scales).

    codes uint8 [..., kb, 16], kb = ceil(K / 32): 32 four-bit floating-point codes a block, low nibble first, the
    last block padded with zeros. scales uint8 [ceil(rows/128), ceil(kb/4), 32, 4, 4]: one power of two a block, in
    the order the tensor cores take them (``mxfp4_tile_scales``). A block that holds a NaN or an infinity reads as NaN.
    """
    dtype = _float_code(x.dtype)
    index = _device_of(x, "x")
    K = x.shape[-1] if x.dim() else 0
    if K < 1:
        raise ValueError("x must be [..., K] with K >= 1")
    rows, kb, ldx = x.numel() // K, -(-K // 32), _row_stride(x, "x")
    codes = x.new_empty((*x.shape[:-1], kb, 16), dtype=torch.uint8)
    scales = x.new_empty(_scale_shape(rows, kb), dtype=torch.uint8)
    t = _native.Mxfp4Tensor_(dtype, 0, rows, K, codes.data_ptr(), scales.data_ptr())
    _launch(index, _native.load().xrgpu_mxfp4_quantize, ctypes.byref(t), x.data_ptr(), ldx)
    return codes, scales


def mxfp4_dequantize(codes: torch.Tensor, scales: torch.Tensor, *, K: Optional[int] = None, dtype=torch.float32) -> torch.Tensor:
    """The values [..., K] that microscaled codes and tiled scales hold (K defaults to 32 kb)."""
    if codes.dim() < 2:
        raise ValueError("codes must be [..., kb, 16]")
    kb = int(codes.shape[-2])
    K = kb * 32 if K is None else int(K)
    if K < 1 or -(-K // 32) != kb:
        raise ValueError("K does not match the codes")
    rows = codes.numel() // (kb * 16) if kb else 0
    code, index = _float_code(dtype), _device_of(codes, "codes")
    _require_mxfp4(codes, scales, rows, kb, "codes", index)
    out = codes.new_empty((*codes.shape[:-2], K), dtype=dtype)
    t = _native.Mxfp4Tensor_(code, 0, rows, K, codes.data_ptr(), scales.data_ptr())
    _launch(index, _native.load().xrgpu_mxfp4_dequantize, ctypes.byref(t), out.data_ptr())
    return out


def mxfp4_tile_scales(scales: torch.Tensor) -> torch.Tensor:
    """Scale bytes [rows, kb] (as checkpoints hold them) in the tiled order of ``matmul_mxfp4``."""
    if scales.dim() != 2 or scales.dtype != torch.uint8 or scales.shape[1] < 1:
        raise ValueError("scales must be uint8 [rows, kb]")
    index = _device_of(scales, "scales")
    _on(scales, "scales", torch.uint8, index)
    rows, kb = scales.shape
    tiled = scales.new_empty(_scale_shape(rows, kb))
    _launch(index, _native.load().xrgpu_mxfp4_tile_scales, rows, kb, scales.data_ptr(), tiled.data_ptr())
    return tiled


def matmul_mxfp4(a: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                 a_scales: Optional[torch.Tensor] = None, K: Optional[int] = None, dtype=None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Y = A . B^T (+ bias) with both operands in microscaled 4-bit form, float32 sums.

    b [N, kb, 16] codes and b_scales (tiled), a either codes [..., kb, 16] with a_scales, or float32 / float16
    [..., K], which the call quantises first. Y [..., N] in `dtype` (default a's, float16 for codes); bias [N] in it.
    ``out`` may be a [..., N] view with unit column stride and rows at one stride.
    """
    index = _device_of(a, "a")
    held = a_scales is not None
    if b.dim() != 3:
        raise ValueError("b must be [N, kb, 16] codes")
    N, kb = b.shape[0], b.shape[1]
    lda = ldy = nbytes = 0
    bias_ptr = scales_ptr = ws = None
    if held:
        if a.dim() < 2 or a.shape[-1] != 16:
            raise ValueError("a must be [..., kb, 16] codes")
        if a.shape[-2] != kb:
            raise ValueError("a and b differ in K")
        lead = a.shape[:-2]
        M = a.numel() // (kb * 16) if kb else 0
        K = kb * 32 if K is None else int(K)
        _require_mxfp4(a, a_scales, M, kb, "a", index)
        a_code, scales_ptr = _native.UINT8, a_scales.data_ptr()
        dtype = torch.float16 if dtype is None else dtype
    else:
        a_code = _float_code(a.dtype)
        lead = a.shape[:-1]
        if K is not None and K != a.shape[-1]:
            raise ValueError("K does not match a")
        K = a.shape[-1]
        M = a.numel() // K if K else 0
        lda = _row_stride(a, "a")
        dtype = a.dtype if dtype is None else dtype
    if K < 1 or -(-K // 32) != kb:
        raise ValueError("a and b differ in K")
    _require_mxfp4(b, b_scales, N, kb, "b", index)
    code = _float_code(dtype)
    if bias is not None:
        _on(bias, "bias", dtype, index)
        if bias.shape != (N,):
            raise ValueError("bias must be [N] in the output dtype")
        bias_ptr = bias.data_ptr()
    if out is None:
        out = a.new_empty((*lead, N), dtype=dtype)
    else:
        if out.dtype != dtype or out.get_device() != index or out.shape != (*lead, N):
            raise ValueError("out must be [..., N] in the output dtype on a's device")
        ldy = _row_stride(out, "out")
    p = _native.Mxfp4Problem_(code, a_code, M, K, N, a.data_ptr(), scales_ptr, lda, b.data_ptr(), b_scales.data_ptr(), bias_ptr,
                              out.data_ptr(), ldy)
    if not held and M:
        nbytes = -(-M * kb * 16 // 256) * 256 + -(-M // 128) * -(-kb // 4) * 512
        scratch = a.new_empty(nbytes, dtype=torch.uint8)
        ws = scratch.data_ptr()
    _launch(index, _native.load().xrgpu_mxfp4_forward, ctypes.byref(p), ws, nbytes)
    return out


def _kv8_problem(k_cache, v_cache, k_scale, v_scale, page_table, cu_seqlens, kv_len, dtype):
    """The cache's part of a call, checked, and its device."""
    code = k_cache.dtype
    if code not in _CACHES:
        raise ValueError("k_cache and v_cache must both be int8 or float8_e4m3fn")
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError("k_cache and v_cache must be [pages, heads, page, head_dim]")
    index = _device_of(k_cache, "k_cache")
    P, H, page, D = k_cache.shape
    _on(k_cache, "k_cache", code, index)
    _on(v_cache, "v_cache", code, index)
    _on(k_scale, "k_scale", torch.float32, index)
    _on(v_scale, "v_scale", torch.float32, index)
    _on(page_table, "page_table", torch.int32, index)
    _on(kv_len, "kv_len", torch.int32, index)
    if k_scale.shape != (P, H) or v_scale.shape != (P, H):
        raise ValueError("k_scale and v_scale must be [pages, heads]")
    if kv_len.dim() != 1 or page_table.dim() != 2 or page_table.shape[0] != kv_len.shape[0]:
        raise ValueError("page_table must be [sequences, max_pages] and kv_len [sequences]")
    B, cu = kv_len.shape[0], None
    if cu_seqlens is not None:
        _on(cu_seqlens, "cu_seqlens", torch.int32, index)
        if cu_seqlens.shape != (B + 1,):
            raise ValueError("cu_seqlens must be [sequences + 1]")
        cu = cu_seqlens.data_ptr()
    p = _native.Kv8Problem_(_float_code(dtype), _CACHES[code], 0, 0.0, 0, 0, 0, B, 0, H, D, page, P, page_table.shape[1], 0, 0, 0, 0, 0,
                            None, None, None, None, k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
                            v_scale.data_ptr(), page_table.data_ptr(), cu, kv_len.data_ptr())
    return p, index, H, D


def _head_rows(t, name: str, heads: Optional[int], D: int, index: int) -> int:
    """Row stride of [rows, heads, D] whose rows may be strided, heads and values side by side."""
    if t.get_device() != index:
        raise ValueError(f"{name} must be a CUDA tensor on cuda:{index}")
    if t.dim() != 3 or t.shape[2] != D or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must be [rows, heads, head_dim]")
    H = t.shape[1]
    if t.is_contiguous() or t.shape[0] == 0:
        return H * D
    if t.stride(2) != 1 or (H > 1 and t.stride(1) != D) or (t.shape[0] > 1 and t.stride(0) < H * D):
        raise ValueError(f"{name} must have its heads and values side by side")
    return t.stride(0) if t.shape[0] > 1 else H * D


def kv8_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
               v_scale: torch.Tensor, page_table: torch.Tensor, cu_seqlens: Optional[torch.Tensor],
               kv_len: torch.Tensor) -> None:
    """Writes new keys and values [rows, heads, head_dim] (float32 or float16; rows may be strided) into the cache.

    k_cache, v_cache [pages, heads, page, head_dim] int8 or float8_e4m3fn and k_scale, v_scale float32 [pages, heads]
    are updated in place; page_table int32 [sequences, max_pages], cu_seqlens int32 [sequences + 1] (None: the same
    number of rows each), kv_len int32 [sequences], the new tokens included: rows cu_seqlens[b] .. of sequence b become
    its last tokens. One scale covers a page of a head; where a new token exceeds it, the page's older codes are
    rescaled. A page shared by two sequences must not be appended to. Bad page ids and lengths: ``device_error``
    0x501, 0x502, nothing written for them.
    """
    p, index, H, D = _kv8_problem(k_cache, v_cache, k_scale, v_scale, page_table, cu_seqlens, kv_len, k.dtype)
    p.k_stride = _head_rows(k, "k", H, D, index)
    p.v_stride = _head_rows(v, "v", H, D, index)
    if v.dtype != k.dtype or v.shape[0] != k.shape[0]:
        raise ValueError("k and v must have the same rows and dtype")
    p.tokens, p.k, p.v = k.shape[0], k.data_ptr(), v.data_ptr()
    _launch(index, _native.load().xrgpu_kv8_append, ctypes.byref(p))


def kv8_read(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
             page_table: torch.Tensor, cu_seqlens: Optional[torch.Tensor], kv_len: torch.Tensor, *, rows: int,
             dtype=torch.float16):
    """The values (k, v), each [rows, heads, head_dim], that the cache holds for the last tokens of each sequence
    (rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1; see ``kv8_append``). Rows of no sequence are zero."""
    p, index, H, D = _kv8_problem(k_cache, v_cache, k_scale, v_scale, page_table, cu_seqlens, kv_len, dtype)
    k = k_scale.new_empty((int(rows), H, D), dtype=dtype)
    v = torch.empty_like(k)
    p.tokens, p.k, p.v, p.zero_rest = int(rows), k.data_ptr(), v.data_ptr(), 1
    _launch(index, _native.load().xrgpu_kv8_read, ctypes.byref(p))
    return k, v


def attention_kv8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                  v_scale: torch.Tensor, page_table: torch.Tensor, cu_seqlens: Optional[torch.Tensor],
                  kv_len: torch.Tensor, *, scale: Optional[float] = None, causal: bool = True, window: int = 0,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of q [rows, query heads, head_dim] over the 8-bit cache (``kv8_append`` describes its tensors).

    Rows cu_seqlens[b] .. are the last positions of sequence b (kv_len counts them; append first). A row sees the
    tokens up to its own position (causal), the last `window` of them if given, or all kv_len (causal=False). Query
    head h reads key/value head h // (query heads // heads). scale defaults to head_dim ** -0.5. Pages in front of every
    row's window are not looked up (released ones may be -1). A row that sees nothing gives zeros; with ``out``, rows
    behind the last sequence are left as they were (without it they are zero). Sums are float32; for float16 rows the softmax's
    weights are rounded to float16 on their way to the values (2^-12 of each), for float32 rows they keep 2^-24.
    """
    p, index, H, D = _kv8_problem(k_cache, v_cache, k_scale, v_scale, page_table, cu_seqlens, kv_len, q.dtype)
    p.q_stride = _head_rows(q, "q", None, D, index)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        p.zero_rest = 1
    else:
        if out.dtype != q.dtype or out.shape != q.shape:
            raise ValueError("out must have q's shape and dtype")
        p.o_stride = _head_rows(out, "out", q.shape[1], D, index)
    p.tokens, p.heads_q, p.q, p.o = q.shape[0], q.shape[1], q.data_ptr(), out.data_ptr()
    p.causal, p.window = int(bool(causal)), int(window)
    p.scale = float(scale) if scale is not None else D ** -0.5
    lib = _native.load()
    need = _workspace_bytes(index, lib.xrgpu_kv8_attention_workspace_size, p)
    ws = q.new_empty(need, dtype=torch.uint8) if need else None
    _launch(index, lib.xrgpu_kv8_attention, ctypes.byref(p), ws.data_ptr() if ws is not None else None, need)
    return out
