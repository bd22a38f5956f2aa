"""Matrices in microscaled 4 bits (MXFP4): rows to 4 bits and back, products with a 4-bit matrix, the gated feed-forward's front half.

A row is cut into blocks of 32 neighbouring values (the last one filled up with zeros).  A block has a scale byte E, the power of two
2^(E - 127), and 32 codes of 4 bits (e2m1: a sign, then 0, 0.5, 1, 1.5, 2, 3, 4 or 6); a value is its code times its block's scale.  E is the
smallest with which no value of the block is cut off (|x| <= 6 * 2^(E - 127)); codes are rounded to nearest, ties to even.  A block that
holds an infinity or a NaN has E = 255, and all its values are NaN.

    w = quantize_mxfp4(weight)                        # or Mxfp4Matrix(codes, scales, columns) from a checkpoint that holds both
    gemm_mxfp4(x, w, out)                             # 16- or 32-bit activations: only the matrix is in 4 bits
    gemm_mxfp4(quantize_mxfp4(x), w, out)             # both operands in 4 bits
    gated_gemm_mxfp4(x, w, out, activation="silu")    # w: the gate's rows, then the up rows; out = act(gate) * up

As in kernels/ops.py every function checks its tensors, launches on the current CUDA stream and has no fallback off the GPU.  The reference
keeps 8-bit matrices beside scales per column (src/transformers_neuronx/quantize.py); 4-bit blocks are what this GPU's tensor cores multiply.
"""
from __future__ import annotations

from ctypes import c_int, c_longlong
from typing import Optional

import torch

from .ops import KernelError, _FLOATS, _check, _is_h16, _lib, _need, _p, _rows_2d, _sm_count, _state, _stream, activation_code

BLOCK = 32                                    # values that share a scale


class Mxfp4Matrix:
    """codes: uint8 [rows, blocks * 16], value 2j of a row in the low half of byte j; scales: uint8 [rows, blocks]; columns: values a row,
    blocks = ceil(columns / 32).  Both contiguous and on one device; codes behind the last column are zeros (0 times whatever stands there
    is what the products add).  The tensors are used as they are, not copied."""

    __slots__ = ("codes", "scales", "columns")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, columns: Optional[int] = None):
        for t, name in ((codes, "codes"), (scales, "scales")):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.uint8 or t.dim() != 2 or not t.is_contiguous():
                raise KernelError(f"{name} must be a contiguous 2-D uint8 tensor")
        rows, blocks = scales.shape
        if codes.shape[0] != rows or codes.shape[1] != blocks * 16 or codes.device != scales.device:
            raise KernelError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not fit: 16 bytes of codes a scale, one device")
        columns = blocks * BLOCK if columns is None else int(columns)
        if blocks < 1 or not (blocks - 1) * BLOCK < columns <= blocks * BLOCK:
            raise KernelError(f"{columns} columns do not make {blocks} blocks of {BLOCK}")
        self.codes, self.scales, self.columns = codes, scales, columns

    @property
    def shape(self):
        return torch.Size((self.codes.shape[0], self.columns))

    @property
    def device(self):
        return self.codes.device

    def numel(self) -> int:
        return self.codes.shape[0] * self.columns

    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def __repr__(self) -> str:
        return f"Mxfp4Matrix({self.codes.shape[0]} x {self.columns}, {self.device})"


def _here(device, *tensors) -> None:
    """All on one device, and it is the current one: the stream is the current device's."""
    if device.type != "cuda":
        raise KernelError("the 4-bit matrices' kernels need CUDA tensors: the engine has no CPU path")
    if device.index != torch.cuda.current_device():
        raise KernelError(f"the tensors are on {device}, the current device is cuda:{torch.cuda.current_device()}")
    for t in tensors:
        if t is not None and t.device != device:
            raise KernelError(f"tensors on {device} and {t.device} in one call")


def quantize_mxfp4(x: torch.Tensor, out: Optional[Mxfp4Matrix] = None) -> Mxfp4Matrix:
    """The rows of x [rows, columns] (16- or 32-bit floats; any row pitch) in 4 bits; `out`: the matrix to write."""
    _need(x, "x", _FLOATS, None, contiguous=False)
    rows, columns, pitch = _rows_2d(x, "x")
    _here(x.device)
    if columns < 1:
        raise KernelError("x has no columns")
    if out is None:
        blocks = -(-columns // BLOCK)
        out = Mxfp4Matrix(torch.empty((rows, blocks * 16), dtype=torch.uint8, device=x.device),
                          torch.empty((rows, blocks), dtype=torch.uint8, device=x.device), columns)
    else:
        _here(x.device, out.codes)
        if out.shape != x.shape:
            raise KernelError(f"out is {tuple(out.shape)}, x {tuple(x.shape)}")
        if out.codes.data_ptr() % 4:
            raise KernelError("out's codes must be 4-byte aligned")
    if rows:
        _check(_lib("mxfp4", x).tnx_mxfp4_quantize(_p(x), c_int(_is_h16(x)), c_longlong(pitch), _p(out.codes), _p(out.scales), c_int(rows),
                                                   c_int(columns), c_int(_sm_count(x.device)), _stream()), "quantize_mxfp4")
    return out


def dequantize_mxfp4(m: Mxfp4Matrix, dtype=torch.bfloat16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values of m: exact in float32 and bfloat16; float16 rounds what lies outside its range (infinity, subnormal numbers)."""
    _here(m.device)
    if m.codes.data_ptr() % 4:
        raise KernelError("the codes must be 4-byte aligned")
    if out is None:
        if dtype not in _FLOATS:
            raise KernelError(f"dtype {dtype}: expected one of {_FLOATS}")
        out = torch.empty(m.shape, dtype=dtype, device=m.device)
    else:
        _need(out, "out", _FLOATS, None, contiguous=False)
        _here(m.device, out)
        if out.shape != m.shape:
            raise KernelError(f"out is {tuple(out.shape)}, the matrix {tuple(m.shape)}")
    rows, columns, pitch = _rows_2d(out, "out")
    if rows:
        _check(_lib("mxfp4", out).tnx_mxfp4_dequantize(_p(m.codes), _p(m.scales), _p(out), c_int(_is_h16(out)), c_longlong(pitch), c_int(rows),
                                                       c_int(columns), c_int(_sm_count(m.device)), _stream()), "dequantize_mxfp4")
    return out


def gemm_mxfp4(a, w: Mxfp4Matrix, out: torch.Tensor, bias=None, residual=None, activation=None) -> torch.Tensor:
    """out = act(a @ w^T + bias) + residual.  a: [tokens, columns] 16- or 32-bit floats, or an Mxfp4Matrix (quantize_mxfp4); out:
    [tokens, rows of w], 32-bit or 16-bit (float activations in 16 bits: the same type); bias: 32-bit; residual: 32-bit with the shape and
    row pitch of a 32-bit out, which it may be.  Sums are 32-bit; each result is rounded once."""
    return _product(a, w, out, bias, residual, activation, False)


def gated_gemm_mxfp4(a, w: Mxfp4Matrix, out: torch.Tensor, bias=None, activation="silu") -> torch.Tensor:
    """out = act(a @ gate^T + bias[:F]) * (a @ up^T + bias[F:]): w holds the gate's F rows, then the F up rows; out [tokens, F].  The front half
    of a gated feed-forward in one kernel; neither projection is rounded before the product."""
    return _product(a, w, out, bias, None, activation, True)


def _product(a, w, out, bias, residual, activation, gated):
    act = activation_code(activation)
    if not isinstance(w, Mxfp4Matrix):
        raise KernelError("w must be an Mxfp4Matrix")
    quantized = isinstance(a, Mxfp4Matrix)
    if quantized:
        (M, K), lda = a.shape, 0
    else:
        _need(a, "a", _FLOATS, None, contiguous=False)
        M, K, lda = _rows_2d(a, "a")
    _need(out, "out", _FLOATS, None, contiguous=False)
    Mo, No, ldc = _rows_2d(out, "out")
    rows, Kw = w.shape
    if gated and rows % 2:
        raise KernelError(f"a gated product needs as many gate rows as up rows, got {rows} in all")
    N = rows // 2 if gated else rows
    if Kw != K or Mo != M or No != N:
        raise KernelError(f"shapes do not fit: a {(M, K)}, w {(rows, Kw)}{' (gated)' if gated else ''}, out {tuple(out.shape)}")
    _here(w.device, a.codes if quantized else a, out, bias, residual)
    if bias is not None:
        _need(bias, "bias", torch.float32, 1)
        if bias.shape[0] != rows:
            raise KernelError("bias length differs from the matrix's rows")
    if residual is not None:
        _need(residual, "residual", torch.float32, None, contiguous=False)
        if tuple(residual.shape) != (M, N) or _rows_2d(residual, "residual")[2] != ldc or out.dtype != torch.float32:
            raise KernelError("residual must be float32 with the shape and row stride of a float32 out")
    if M == 0 or N == 0:
        return out
    if not quantized and _is_h16(a) and (out.dtype == a.dtype or out.dtype == torch.float32) and lda % 8 == 0 \
            and a.data_ptr() % 16 == 0 and w.codes.data_ptr() % 16 == 0:
        st = _state(a.device)
        _check(_lib("gemm_mxfp4", a).tnx_gemm_mxfp4_16(_p(a), c_longlong(lda), _p(w.codes), _p(w.scales), _p(bias), _p(residual), _p(out), c_int(_is_h16(out)),
                                                       c_longlong(ldc), c_int(M), c_int(N), c_int(K), c_int(act), c_int(1 if gated else 0),
                                                       c_int(st["sms"]), _p(st["err"]), _stream()), "gemm_mxfp4")
        return out
    if quantized and a.codes.data_ptr() % 16 == 0 and w.codes.data_ptr() % 16 == 0:
        st = _state(w.device)
        _check(_lib("gemm_mxfp4", out).tnx_gemm_mxfp4_4(_p(a.codes), _p(a.scales), _p(w.codes), _p(w.scales), _p(bias), _p(residual), _p(out),
                                                        c_int(_is_h16(out)), c_longlong(ldc), c_int(M), c_int(N), c_int(K), c_int(act),
                                                        c_int(1 if gated else 0), c_int(st["sms"]), _p(st["err"]), _stream()), "gemm_mxfp4")
        return out
    lib = _lib("mxfp4", None if quantized else a, out)
    kind = 2 if quantized else 0 if _is_h16(a) else 1
    _check(lib.tnx_mxfp4_gemm_simt(_p(a.codes if quantized else a), c_int(kind), _p(a.scales if quantized else None), c_longlong(lda), _p(w.codes),
                                   _p(w.scales), _p(bias), _p(residual), _p(out), c_int(_is_h16(out)), c_longlong(ldc), c_int(M), c_int(N), c_int(K),
                                   c_int(act), c_int(1 if gated else 0), _stream()), "gemm_mxfp4")
    return out
