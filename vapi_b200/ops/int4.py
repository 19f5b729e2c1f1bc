"""Products with 4-bit weights and a scale and a zero for each group of columns (csrc/int4.cu)."""
from __future__ import annotations

import os
from typing import Optional, Tuple

import torch

from . import BF16, KernelError, _bias, _check, _cuda, _glu, _here, _lib, _native, _p, _stream, _DT
from . import linear as _linear
from . import linear_swiglu as _linear_swiglu
from . import swiglu as _swiglu

INT4_GROUPS = (32, 64, 128)
#: products of more bfloat16 rows than this take the weight as bfloat16 numbers through this package's and the library's products (and of fewer,
#: where :func:`_own` says so)
INT4_MAX_ROWS = int(os.environ.get("VAPI_INT4_MAX_ROWS", "2048"))


class Int4Weight:
    """A matrix [n, k] of numbers ``(code - zero) * scale`` as the kernels read it (:func:`int4_pack` and :func:`int4_quantize` make one): codes
    and zeros in 0..15, a bfloat16 scale and a zero for each group of ``group`` columns of a row."""

    __slots__ = ("codes", "scales", "n", "k", "group")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, n: int, k: int, group: int):
        self.codes, self.scales, self.n, self.k, self.group = codes, scales, int(n), int(k), int(group)
        n, k, group = self.n, self.k, self.group
        if n <= 0 or k <= 0 or group not in INT4_GROUPS or k % group:
            raise KernelError(f"a 4-bit weight of {n} x {k} in groups of {group}")
        tiles, chunks = -(-n // 16), -(-k // 64)
        for t, shape, what in ((codes, (tiles, chunks, 32, 4), "codes"), (scales, (tiles, 2 * chunks if group == 32 else k // group, 8, 2), "scales")):
            if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
                raise KernelError(f"the {what} of a 4-bit weight must be {shape} of int32 in one piece, got {tuple(t.shape)} of {t.dtype}")

    @property
    def shape(self) -> Tuple[int, int]:
        return self.n, self.k

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def nbytes(self) -> int:
        return (self.codes.numel() + self.scales.numel()) * 4


def int4_pack(codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None) -> Int4Weight:
    """Lay a 4-bit matrix out for the kernels, once: ``codes`` [n, k] uint8 in 0..15, ``scales`` [n, k / group] bfloat16,
    ``zeros`` [n, k / group] uint8 in 0..15 (None: 8 everywhere); the group is 32, 64 or 128 columns."""
    if codes.dim() != 2 or codes.dtype != torch.uint8 or codes.numel() == 0:
        raise KernelError(f"the codes must be [n, k] of uint8, got {tuple(codes.shape)} of {codes.dtype}")
    n, k = codes.shape
    if scales.dtype != torch.bfloat16 or scales.dim() != 2 or scales.shape[0] != n or scales.shape[1] == 0 or k % scales.shape[1]:
        raise KernelError(f"the scales must be [{n}, groups] of bfloat16, got {tuple(scales.shape)} of {scales.dtype}")
    groups = scales.shape[1]
    group = k // groups
    if group not in INT4_GROUPS:
        raise KernelError(f"groups of {group} columns are not one of {', '.join(map(str, INT4_GROUPS))}")
    if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape):
        raise KernelError(f"the zeros must be {tuple(scales.shape)} of uint8, got {tuple(zeros.shape)} of {zeros.dtype}")
    if codes.device != scales.device or (zeros is not None and codes.device != zeros.device):
        raise KernelError("codes, scales and zeros must be on one device")
    if codes.is_cuda:
        return _pack(codes, scales, zeros, group)
    if zeros is None:
        zeros = torch.full_like(scales, 8, dtype=torch.uint8)
    if int(codes.max()) > 15 or int(zeros.max()) > 15:
        raise KernelError("codes and zeros must be in 0..15")
    tiles, chunks = -(-n // 16), -(-k // 64)
    words = torch.empty((tiles, chunks, 32, 4), dtype=torch.int32, device=codes.device)
    step = max(1, (1 << 24) // (chunks * 1024))                    # tiles at a time: what stands beside the codes stays small
    for at in range(0, tiles, step):
        part = codes[at * 16:(at + step) * 16]
        m = -(-part.shape[0] // 16)
        part = torch.nn.functional.pad(part, (0, chunks * 64 - k, 0, m * 16 - part.shape[0])).to(torch.int32)
        # row 8h + g, column 64 ch + 16j + 8p + 2c + e  ->  lane 4g + c, word j, bits from 8p + 4h + 16e on
        part = part.view(m, 2, 8, chunks, 4, 2, 4, 2).permute(0, 3, 2, 6, 4, 1, 5, 7)
        got = torch.zeros((m, chunks, 8, 4, 4), dtype=torch.int32, device=codes.device)
        for h in range(2):
            for p in range(2):
                for e in range(2):
                    got |= part[..., h, p, e] << (8 * p + 4 * h + 16 * e)
        words[at:at + m] = got.view(m, chunks, 32, 4)
    bits = lambda t: t.to(torch.bfloat16).view(torch.int16).to(torch.int32) & 0xffff
    pairs = bits(scales) | bits(zeros.to(torch.float32) + 128.0) << 16
    wide = 2 * chunks if group == 32 else groups                   # (whole tiles of 64 columns)
    pairs = torch.nn.functional.pad(pairs, (0, wide - groups, 0, tiles * 16 - n)).view(tiles, 2, 8, wide).permute(0, 3, 2, 1).contiguous()
    return Int4Weight(words, pairs, n, k, group)


def _pack(codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor], group: int) -> Int4Weight:
    """The same on the device, by one kernel."""
    n, k = codes.shape
    _here(codes)
    codes, scales = codes.contiguous(), scales.contiguous()
    if codes.data_ptr() % 8:
        codes = codes.clone()
    zeros = None if zeros is None else zeros.contiguous()
    tiles, chunks = -(-n // 16), -(-k // 64)
    words = torch.empty((tiles, chunks, 32, 4), dtype=torch.int32, device=codes.device)
    pairs = torch.empty((tiles, 2 * chunks if group == 32 else k // group, 8, 2), dtype=torch.int32, device=codes.device)
    bad = torch.zeros(1, dtype=torch.int32, device=codes.device)
    lib = _lib("int4")
    _check(lib, lib.vapi_int4_pack(_p(codes), _p(scales), _p(zeros), n, k, group, _p(words), _p(pairs), _p(bad), _stream()))
    if int(bad):
        raise KernelError("codes and zeros must be in 0..15")
    return Int4Weight(words, pairs, n, k, group)


def int4_quantize(weight: torch.Tensor, group: int = 64) -> Int4Weight:
    """The nearest 4-bit matrix by each group's extremes: ``scale = (max - min) / 15`` rounded to bfloat16, ``zero = round(-min /
    scale)``, ``code = round(w / scale) + zero`` (min and max with 0 among them, so that zero stays zero)."""
    if weight.dim() != 2 or weight.numel() == 0 or not weight.dtype.is_floating_point:
        raise KernelError(f"a weight to quantise must be [n, k] of a floating type, got {tuple(weight.shape)} of {weight.dtype}")
    if group not in INT4_GROUPS or weight.shape[1] % group:
        raise KernelError(f"{weight.shape[1]} columns do not fall into groups of {group} (one of {', '.join(map(str, INT4_GROUPS))})")
    n, k = weight.shape
    codes = torch.empty((n, k), dtype=torch.uint8, device=weight.device)
    scales = torch.empty((n, k // group), dtype=torch.bfloat16, device=weight.device)
    zeros = torch.empty((n, k // group), dtype=torch.uint8, device=weight.device)
    step = max(1, (1 << 24) // k)
    for at in range(0, n, step):
        w = weight[at:at + step].to(torch.float32).view(-1, k // group, group)
        if not bool(torch.isfinite(w).all()):
            raise KernelError("a weight to quantise holds numbers that are not finite")
        lo, hi = w.amin(-1).clamp(max=0.0), w.amax(-1).clamp(min=0.0)
        # (an empty group, or one too small for a scale: codes are zeros then)
        s = (hi / 15 - lo / 15).clamp(min=1e-30).to(torch.bfloat16)
        z = torch.round(-lo / s.to(torch.float32)).clamp(0, 15)
        codes[at:at + step] = (torch.round(w / s.to(torch.float32)[..., None]) + z[..., None]).clamp(0, 15).to(torch.uint8).view(-1, k)
        scales[at:at + step], zeros[at:at + step] = s, z.to(torch.uint8)
    return int4_pack(codes, scales, zeros)


def _operands(x: torch.Tensor, w: Int4Weight) -> torch.Tensor:
    if not isinstance(w, Int4Weight):
        raise KernelError(f"a 4-bit product needs an Int4Weight, got {type(w).__name__}")
    if x.dim() != 2 or x.shape[1] != w.k or x.dtype not in _DT:
        raise KernelError(f"token operand {tuple(x.shape)} / {x.dtype} does not fit a 4-bit weight of {w.n}x{w.k}")
    _cuda(x, w.codes, w.scales)
    _here(x, w.codes, w.scales)
    return x if x.is_contiguous() and x.data_ptr() % 16 == 0 else x.clone(memory_format=torch.contiguous_format)


def int4_dequantize(w: Int4Weight, dtype: torch.dtype) -> torch.Tensor:
    """The numbers of a 4-bit weight, [n, k] in float32 (exactly) or bfloat16 (each rounded once: a scale times a whole number of
    four bits has four bits more than bfloat16).  Any kernel launched behind the call may read them as a weight."""
    if dtype not in _DT:
        raise KernelError(f"dtype {dtype} is not supported by the kernels (float32, bfloat16)")
    _cuda(w.codes, w.scales)
    _here(w.codes, w.scales)
    out = torch.empty((w.n, w.k), dtype=dtype, device=w.device)
    lib = _lib("int4")
    _check(lib, lib.vapi_int4_numbers(_p(w.codes), _p(w.scales), w.n, w.k, w.group, _p(out), _DT[dtype], _stream()), launches=2)
    return out


def _own(rows: int, w: Int4Weight) -> bool:
    """Whether a product of so many bfloat16 rows is csrc/int4.cu's.  Writing a weight out costs 0.43 us for each million of its numbers, and the
    kernel's lesser rate a part of the product, which is the larger the shorter K is (a block's start and end).  us of the kernel and of the other
    form: 2,048 x 2,048, 128 rows 8.0 / 8.7, 256 rows 11.3 / 9.0; 6,144 x 2,048, 256 rows 13.4 / 14.0, 512 rows 18.3 / 18.5, 1,024 rows 35 / 27;
    16,384 x 2,048, 768 rows 53.6 / 54.0, 1,024 rows 70 / 64; 2,048 x 8,192, 512 rows 20 / 26, 2,048 rows 49 / 54; 28,672 x 8,192 gated, 2,048 rows
    757 / 862."""
    numbers = w.n * w.k
    most = 128 if numbers < 1 << 23 else 512 if numbers < 1 << 24 else 768 if w.k < 4096 else 2048
    return rows <= min(most, INT4_MAX_ROWS)


def _rows(x: torch.Tensor, w: Int4Weight, bias, out: torch.Tensor, gated: int, act: int) -> torch.Tensor:
    lib = _lib("int4")
    f32 = out.dtype == torch.float32
    _check(lib, lib.vapi_int4_linear(_p(w.codes), _p(w.scales), w.n, w.k, w.group, _p(x), x.shape[0], _p(bias), None if f32 else _p(out),
                                     _p(out) if f32 else None, gated, act, -1, _stream()), launches=int(x.shape[0] > 0))
    return out


def int4_linear(x: torch.Tensor, w: Int4Weight, bias: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """:func:`linear` with a 4-bit weight: ``x @ W.T (+ bias)`` for ``x`` [n, k], in ``out_dtype`` (the type of ``x``, or float32).

    Up to 16 bfloat16 rows the codes are multiplied as the whole numbers they are, a group's sum is put on its scale in float32, and the
    result is rounded once.  More rows take the weight's numbers rounded to bfloat16, in the product itself up to 128 to INT4_MAX_ROWS rows (by the weight's size), else,
    as float32 ``x`` does with them in float32, through :func:`int4_dequantize` and :func:`linear`."""
    if type(w) is Int4Weight and x.is_cuda and x.dtype == torch.bfloat16 and _own(x.shape[0], w) and out_dtype in (None, torch.bfloat16, torch.float32):
        lib = _lib("int4")
        got = _native("int4", lib, "vapi_int4_linear", w.codes, w.scales, w.n, w.k, w.group, x, bias, 0, 0, int(out_dtype == torch.float32))
        if got is not NotImplemented:
            _check(lib, got if type(got) is int else 0, int(x.shape[0] > 0))
            return got
    x = _operands(x, w)
    _bias(bias, w.n)
    if out_dtype not in (None, x.dtype, torch.float32):
        raise KernelError(f"a 4-bit product of {x.dtype} gives {x.dtype} or float32, not {out_dtype}")
    if _DT[x.dtype] == BF16 and _own(x.shape[0], w):
        return _rows(x, w, bias, torch.empty((x.shape[0], w.n), dtype=out_dtype or x.dtype, device=x.device), 0, 0)
    return _linear(x, int4_dequantize(w, x.dtype), bias, out_dtype)


def int4_linear_swiglu(x: torch.Tensor, w: Int4Weight, act: str = "silu") -> torch.Tensor:
    """:func:`linear_swiglu` with a 4-bit weight [Wg; Wu]: ``act(x @ Wg.T) * (x @ Wu.T)``, the gate in the product's epilogue."""
    if type(w) is Int4Weight and x.is_cuda and x.dtype == torch.bfloat16 and _own(x.shape[0], w) and w.n % 32 == 0:
        lib = _lib("int4")
        got = _native("int4", lib, "vapi_int4_linear", w.codes, w.scales, w.n, w.k, w.group, x, None, 1, _glu(act), 0)
        if got is not NotImplemented:
            _check(lib, got if type(got) is int else 0, int(x.shape[0] > 0))
            return got
    x = _operands(x, w)
    if w.n % 2:
        raise KernelError("a gated product needs an even number of features")
    kind = _glu(act)
    if _DT[x.dtype] == BF16 and _own(x.shape[0], w):
        if w.n % 32 == 0:
            return _rows(x, w, None, torch.empty((x.shape[0], w.n // 2), dtype=x.dtype, device=x.device), 1, kind)
        return _swiglu(int4_linear(x, w), act)
    return _linear_swiglu(x, int4_dequantize(w, x.dtype), act)
