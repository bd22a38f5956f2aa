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

from ctypes import c_char_p, c_longlong
from struct import Struct
from typing import Optional

import torch

from . import build as _build
from . import ops as _ops
from .ops import ACTIVATIONS, KernelError, _FLOATS, _H16, _check, _state, activation_code

BLOCK = 32                                    # values that share a scale
TILE_TOKENS = 128                             # beyond these persistent blocks walk over tiles of up to 192 tokens (gemm_mxfp4_tiles.cu)
CHAIN = 5120                                  # 32-bit results of 16-bit activations: the columns that one accumulator adds up without a visible loss; beyond
                                              # them K is split (up to eight ways); 4-bit ones take an addition for 64 columns instead of 16 and are not split for it
MOST = 2**31 - 4096                           # rows or columns: kernels count both, rounded up to tiles, in 32 bits
FEW_TOKENS = 16                               # the most that the kernel which streams the matrix through registers takes at a time (gemv_mxfp4.cu)


class Mxfp4Matrix:
    """codes: uint8 [rows, blocks * 16], value 2j of a row in the low half of byte j; scales: uint8 [rows, blocks]; columns: values a row,
    blocks = ceil(columns / 32).  Both contiguous and on one device; codes behind the last column are zeros (0 times whatever stands there
    is what the products add).  The tensors are used as they are, not copied."""

    # _kind: the 16-bit type of the values that were brought into 4 bits, if it was one: where no 16-bit operand names it, it names the build of the kernels
    __slots__ = ("_codes", "_scales", "_buffer", "_device", "_blocks", "_kind", "rows", "columns")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, columns: Optional[int] = None):
        for t, name in ((codes, "codes"), (scales, "scales")):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.uint8 or t.dim() != 2 or not t.is_contiguous():
                raise KernelError(f"{name} must be a contiguous 2-D uint8 tensor")
        rows, blocks = scales.shape
        if codes.shape != (rows, blocks * 16) or codes.device != scales.device:
            raise KernelError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not fit: 16 bytes of codes a scale, one device")
        columns = blocks * BLOCK if columns is None else int(columns)
        if rows > MOST or columns > MOST:
            raise KernelError(f"{rows} x {columns} values: at most {MOST} either way")
        if blocks < 1 or not (blocks - 1) * BLOCK < columns <= blocks * BLOCK:
            raise KernelError(f"{columns} columns do not make {blocks} blocks of {BLOCK}")
        self._codes, self._scales, self._buffer = codes, scales, None
        self._device, self._blocks, self._kind, self.rows, self.columns = codes.get_device(), blocks, None, rows, columns

    @classmethod
    def _empty(cls, rows: int, columns: int, device: torch.device, number: int) -> "Mxfp4Matrix":
        """Codes and scales behind them in one allocation; the two tensors are made when they are asked for."""
        self = object.__new__(cls)
        blocks = (columns + BLOCK - 1) // BLOCK
        self._codes = self._scales = None
        self._buffer = torch.empty_strided((rows * blocks * 17,), (1,), dtype=torch.uint8, device=device)
        self._device, self._blocks, self._kind, self.rows, self.columns = number, blocks, None, rows, columns
        return self

    def _split(self) -> None:
        n = self.rows * self._blocks * 16
        self._codes = self._buffer[:n].view(self.rows, self._blocks * 16)
        self._scales = self._buffer[n:].view(self.rows, self._blocks)

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            self._split()
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            self._split()
        return self._scales

    def _pointers(self):
        if self._buffer is not None:
            p = self._buffer.data_ptr()
            return p, p + self.rows * self._blocks * 16
        return self._codes.data_ptr(), self._scales.data_ptr()

    @property
    def shape(self):
        return torch.Size((self.rows, self.columns))

    @property
    def device(self):
        return (self._buffer if self._buffer is not None else self._codes).device

    def numel(self) -> int:
        return self.rows * self.columns

    def nbytes(self) -> int:
        return self.rows * self._blocks * 17

    def __repr__(self) -> str:
        return f"Mxfp4Matrix({self.rows} x {self.columns}, {self.device})"


# Entry points take their parameters in one array, the stream last: a parameter of a ctypes call costs 0.1 us.
_PACK = {n: Struct(f"{n}q").pack for n in range(1, 24)}
_entries = {}


def _entry(library: str, name: str, dtype):
    """The entry point in the flavour of `dtype`'s 16-bit type."""
    fn = _entries.get((name, dtype))
    if fn is None:
        fn = getattr(_build.load(library, dtype if dtype in _H16 else None), name + "_packed")
        fn.argtypes = [c_char_p]
        _entries[(name, dtype)] = fn
    return fn


_devices = {}                                 # number -> (SMs, address of the error word)


def _device_info(number: int, device: torch.device):
    have = _devices.get(number)
    if have is None:
        st = _state(device)
        have = _devices[number] = (st["sms"], st["err"].data_ptr())
    return have


def _stream(device: int) -> int:
    scoped = _ops._scoped_stream
    return (scoped.value or 0) if scoped is not None else torch._C._cuda_getCurrentRawStream(device)


def _device_of(t: torch.Tensor, name: str) -> int:
    """The number of the tensor's device, which has to be the current one: the stream is the current device's."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise KernelError(f"{name} must be a CUDA tensor: the engine has no CPU path")
    d = t.get_device()
    if d != torch._C._cuda_getDevice():
        raise KernelError(f"{name} is on cuda:{d}, the current device is cuda:{torch._C._cuda_getDevice()}")
    return d


def _matrix_device(m: Mxfp4Matrix, name: str) -> int:
    d = m._device
    if d < 0:
        raise KernelError(f"{name} must be on a CUDA device: the engine has no CPU path")
    if d != torch._C._cuda_getDevice():
        raise KernelError(f"{name} is on cuda:{d}, the current device is cuda:{torch._C._cuda_getDevice()}")
    return d


def _floats(t, name: str, device: int):
    """(rows, columns, row pitch) of a 2-D tensor of 16- or 32-bit floats on `device` whose rows are contiguous."""
    if not isinstance(t, torch.Tensor) or t.dtype not in _FLOATS:
        raise KernelError(f"{name} must be a tensor of bfloat16, float16 or float32")
    if t.get_device() != device:
        raise KernelError(f"{name} is on {t.device}, other tensors of the call on cuda:{device}")
    if t.dim() != 2:
        raise KernelError(f"{name} has {t.dim()} dimensions, expected 2")
    rows, columns = t.shape
    pitch, step = t.stride()
    if step != 1 and columns > 1:
        raise KernelError(f"{name} must have contiguous rows")
    if rows > MOST or columns > MOST:
        raise KernelError(f"{name} is {rows} x {columns}: at most {MOST} either way")
    return rows, columns, pitch if rows > 1 else (columns + 7) // 8 * 8         # the pitch of one row means nothing


def _writable(t, name: str, device: int):
    """_floats() of a tensor that a kernel writes."""
    rows, columns, pitch = _floats(t, name, device)
    if pitch < columns and rows > 1:
        raise KernelError(f"{name}'s rows overlap: a pitch of {pitch} for {columns} columns")
    return rows, columns, pitch


def quantize_mxfp4(x: torch.Tensor, out: Optional[Mxfp4Matrix] = None) -> Mxfp4Matrix:
    """The rows of x [rows, columns] (16- or 32-bit floats; any row pitch) in 4 bits; `out`: the matrix to write."""
    device = _device_of(x, "x")
    rows, columns, pitch = _floats(x, "x", device)
    if columns < 1:
        raise KernelError("x has no columns")
    if out is None:
        out = Mxfp4Matrix._empty(rows, columns, x.device, device)
    elif not isinstance(out, Mxfp4Matrix) or (out.rows, out.columns, out._device) != (rows, columns, device):
        raise KernelError(f"out must be an Mxfp4Matrix of {rows} x {columns} on the device of x")
    codes, scales = out._pointers()
    if codes % 4:
        raise KernelError("out's codes must be 4-byte aligned")
    dtype = x.dtype
    out._kind = dtype if dtype in _H16 else None
    if rows:
        _check(_entry("mxfp4", "tnx_mxfp4_quantize", dtype)(_PACK[9](
            x.data_ptr(), 0 if dtype is torch.float32 else 1, pitch, codes, scales, rows, columns, _device_info(device, x.device)[0], _stream(device))),
            "quantize_mxfp4")
    return out


def dequantize_mxfp4(m: Mxfp4Matrix, dtype=torch.bfloat16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values of m: exact in float32 and bfloat16; float16 rounds what lies outside its range (infinity, subnormal numbers)."""
    if not isinstance(m, Mxfp4Matrix):
        raise KernelError("m must be an Mxfp4Matrix")
    device = _matrix_device(m, "m")
    codes, scales = m._pointers()
    if codes % 4:
        raise KernelError("the codes must be 4-byte aligned")
    rows, columns = m.rows, m.columns
    if out is None:
        if dtype not in _FLOATS:
            raise KernelError(f"dtype {dtype}: expected one of {_FLOATS}")
        out, pitch = torch.empty_strided((rows, columns), (columns, 1), dtype=dtype, device=m.device), columns
    else:
        have, width, pitch = _writable(out, "out", device)
        if have != rows or width != columns:
            raise KernelError(f"out is {tuple(out.shape)}, the matrix {rows} x {columns}")
        dtype = out.dtype
    if rows:
        _check(_entry("mxfp4", "tnx_mxfp4_dequantize", dtype)(_PACK[9](
            codes, scales, out.data_ptr(), 0 if dtype is torch.float32 else 1, pitch, rows, columns, _device_info(device, out.device)[0], _stream(device))),
            "dequantize_mxfp4")
    return out


def gemm_mxfp4(a, w: Mxfp4Matrix, out: torch.Tensor, bias=None, residual=None, activation=None) -> torch.Tensor:
    """out = act(a @ w^T + bias) + residual.  a: [tokens, columns] 16- or 32-bit floats, or an Mxfp4Matrix (quantize_mxfp4); out:
    [tokens, rows of w], 32-bit or 16-bit (float activations in 16 bits: the same type); bias: 32-bit; residual: 32-bit with the shape and
    row pitch of a 32-bit out, which it may be.  Sums are 32-bit; each result is rounded once.  out overlaps no other operand.

    Where operands become 16-bit ones, values far below their neighbours lose bits: with float16 activations values of a row of w below 2^-36 of
    the row's largest scale, and where few tokens are streamed (kernels' choice) activations below 2^-39 of the largest of the 256 around them.
    A value of the matrix that no 32-bit number holds (2^128 and more: codes 4 and 6 of scale byte 253, 2 to 6 of 254) counts as itself or as an infinity,
    as the kernel has it; every other scale byte is as good as any, and no step on the way to a result leaves 32 bits unless the sums do."""
    return _product(a, w, out, bias, residual, activation, False)


def gated_gemm_mxfp4(a, w: Mxfp4Matrix, out: torch.Tensor, bias=None, activation="silu") -> torch.Tensor:
    """out = act(a @ gate^T + bias[:F]) * (a @ up^T + bias[F:]): w holds the gate's F rows, then the F up rows; out [tokens, F].  The front half
    of a gated feed-forward in one kernel; neither projection is rounded before the product."""
    return _product(a, w, out, bias, None, activation, True)


_tiles = {}                                   # sizes -> whether persistent tiles are the faster kernel


def _in_tiles(M, N, K, gated, quantized, out_h16, kind, sms) -> bool:
    """More than TILE_TOKENS tokens: whether the kernel of persistent tiles takes them, or (few tiles, long K; 32-bit results of a long K) the one that
    splits K over clusters.  Whichever is estimated to be faster; 2,048 tokens by 16,384 x 4,096 223 to 240 us in tiles, 323 split; 200 by 5,120 x 20,480
    102 and 72."""
    key = (M, N, K, gated, quantized, out_h16, kind, sms)
    have = _tiles.get(key)
    if have is None:
        if not quantized and not out_h16 and K > CHAIN:
            have = False
        else:
            few, many = _build.load("gemm_mxfp4", kind), _build.load("gemm_mxfp4_tiles", kind)
            few.tnx_gemm_mxfp4_estimate.restype = many.tnx_gemm_mxfp4_tiles_estimate.restype = c_longlong
            g, q = int(gated), int(quantized)
            have = (many.tnx_gemm_mxfp4_tiles_estimate(M, N, K, g, q, sms) <= few.tnx_gemm_mxfp4_estimate(M, N, K, g, q, out_h16, sms))
        if len(_tiles) > 4096:
            _tiles.clear()
        _tiles[key] = have
    return have


def _product(a, w, out, bias, residual, activation, gated):
    act = ACTIVATIONS.get(activation)
    if act is None:
        act = activation_code(activation)                     # raises
    if not isinstance(w, Mxfp4Matrix):
        raise KernelError("w must be an Mxfp4Matrix")
    device = _matrix_device(w, "w")
    rows = w.rows
    quantized = isinstance(a, Mxfp4Matrix)
    if quantized:
        if a._device != device:
            raise KernelError(f"a is on {a.device}, w on {w.device}")
        M, K, lda, kind, a_kind = a.rows, a.columns, 0, a._kind or w._kind, 2
        a_p, as_p = a._pointers()
    else:
        M, K, lda = _floats(a, "a", device)
        kind = a.dtype
        a_kind = 0
        if kind is torch.float32:
            a_kind, kind = 1, w._kind
        a_p, as_p = a.data_ptr(), 0
    Mo, N, ldc = _writable(out, "out", device)
    if gated and rows % 2:
        raise KernelError(f"a gated product needs as many gate rows as up rows, got {rows} in all")
    if w.columns != K or Mo != M or (2 * N if gated else N) != rows:
        raise KernelError(f"shapes do not fit: a {(M, K)}, w {(rows, w.columns)}{' (gated)' if gated else ''}, out {tuple(out.shape)}")
    out_kind = out.dtype
    out_h16 = 0 if out_kind is torch.float32 else 1
    if out_h16:
        if a_kind == 0 and kind is not out_kind:
            raise KernelError(f"a is {kind}, out {out_kind}: 16-bit activations and results must agree")
        kind = out_kind
    bias_p = res_p = 0
    if bias is not None:
        if not isinstance(bias, torch.Tensor) or bias.dtype is not torch.float32 or bias.dim() != 1 or bias.get_device() != device or not bias.is_contiguous():
            raise KernelError("bias must be a contiguous 1-D float32 tensor on the device of w")
        if bias.shape[0] != rows:
            raise KernelError("bias length differs from the matrix's rows")
        bias_p = bias.data_ptr()
    if residual is not None:
        if _floats(residual, "residual", device) != (M, N, ldc) or residual.dtype is not torch.float32 or out_h16:
            raise KernelError("residual must be float32 with the shape and row stride of a float32 out")
        res_p = residual.data_ptr()
    if M == 0 or N == 0:
        return out
    w_p, s_p = w._pointers()
    sms, err = _device_info(device, out.device)
    kernels = 1
    tail = (w_p, s_p, bias_p, res_p, out.data_ptr(), out_h16, ldc, M, N, K, act, 1 if gated else 0)
    few = w_p % 16 == 0 and (a_kind != 2 or a_p % 4 == 0)
    tensor = (a_p | w_p) % 16 == 0 and (a_kind == 2 or (a_kind == 0 and lda % 8 == 0 and lda >= K))
    # 4-bit activations are always faster on the tensor cores (one to 16 tokens by 16,384 x 4,096 9 us, 13 to 27 streamed), 16-bit ones from nine tokens
    # on (8 tokens by 16,384 x 4,096 13 to 16 us streamed, 17 to 20 on the tensor cores, 12 tokens 19 to 22 and 17 to 20; by 2,304 x 768 5 to 6 and 6,
    # then 6 to 7.6 and 6); 32-bit ones are streamed, 16 tokens at a time
    if few and (not tensor or (a_kind == 0 and M <= 8)) and (M <= FEW_TOKENS or a_kind == 1):
        code = _entry("gemv_mxfp4", "tnx_gemv_mxfp4", kind)(_PACK[19](a_p, a_kind, as_p, lda, *tail, sms, err, _stream(device)))
        kernels = -(-M // FEW_TOKENS)
    elif tensor:
        tiles = M > TILE_TOKENS and _in_tiles(M, N, K, gated, quantized, out_h16, kind, sms)
        if tiles and quantized:
            # scales as the tensor cores read them: 1,024 bytes for 128 rows of W, 2,048 for 64 tokens, for every 256 columns
            nbytes = ((rows + 127) // 128 * 1024 + (M + 63) // 64 * 2048) * ((K + 255) // 256)
            scratch = torch.empty_strided((nbytes,), (1,), dtype=torch.uint8, device=out.device)
            code = _entry("gemm_mxfp4_tiles", "tnx_gemm_mxfp4_tiles_4", kind)(
                _PACK[18](a_p, as_p, *tail, scratch.data_ptr(), sms, err, _stream(device)))
            kernels = 2
        elif tiles:
            code = _entry("gemm_mxfp4_tiles", "tnx_gemm_mxfp4_tiles_16", kind)(_PACK[17](a_p, lda, *tail, sms, err, _stream(device)))
        elif quantized:
            code = _entry("gemm_mxfp4", "tnx_gemm_mxfp4_4", kind)(_PACK[17](a_p, as_p, *tail, sms, err, _stream(device)))
        else:
            code = _entry("gemm_mxfp4", "tnx_gemm_mxfp4_16", kind)(_PACK[17](a_p, lda, *tail, sms, err, _stream(device)))
    else:
        code = _entry("mxfp4", "tnx_mxfp4_gemm_simt", kind)(_PACK[17](a_p, a_kind, as_p, lda, *tail, _stream(device)))
    _check(code, "gemm_mxfp4", kernels)
    return out
