"""A paged cache of keys and values in 8 bits: the write, the read, and attention over it (csrc/cache8.cu)."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import KernelError, _check, _contig, _cuda, _dt, _f32, _held, _here, _i32, _least, _lib, _native, _p, _stream

#: tokens of a head that share a scale
CACHE8_BLOCK = 16


class Cache8(NamedTuple):
    """A layer's keys and values in 8 bits.  ``codes`` [pages, 2, nkv, page_size, d] are e4m3 numbers, ``exps``
    [pages, 2, nkv, page_size / 16] int8 the powers of two that blocks of 16 tokens of a head are scaled by: a number is
    ``code * 2^exp``.  A block's exponent is the smallest in -110..119 with which its largest magnitude fits 448."""

    codes: torch.Tensor
    exps: torch.Tensor


def cache8_empty(pages: int, nkv: int, page_size: int, d: int, device="cuda") -> Cache8:
    """Memory for a layer's cache (its contents undefined)."""
    if page_size <= 0 or page_size % CACHE8_BLOCK:
        raise KernelError(f"page size {page_size} must be a positive multiple of {CACHE8_BLOCK}")
    return Cache8(torch.empty((pages, 2, nkv, page_size, d), dtype=torch.float8_e4m3fn, device=device),
                  torch.empty((pages, 2, nkv, page_size // CACHE8_BLOCK), dtype=torch.int8, device=device))


def _cache8(cache: Cache8, nkv: int, d: int):
    """(pages, page size) of a cache, checked."""
    codes, exps = cache
    if codes.dtype != torch.float8_e4m3fn or codes.dim() != 5 or codes.shape[1] != 2 or codes.shape[2] != nkv or codes.shape[4] != d:
        raise KernelError(f"the codes must be [pages, 2, {nkv}, page_size, {d}] of float8_e4m3fn, got {tuple(codes.shape)} of {codes.dtype}")
    pages, page_size = codes.shape[0], codes.shape[3]
    if page_size % CACHE8_BLOCK or page_size == 0 or pages == 0:
        raise KernelError(f"a cache of {pages} pages of {page_size} tokens: pages must hold a positive multiple of {CACHE8_BLOCK}")
    if exps.dtype != torch.int8 or tuple(exps.shape) != (pages, 2, nkv, page_size // CACHE8_BLOCK):
        raise KernelError(f"the exponents must be {(pages, 2, nkv, page_size // CACHE8_BLOCK)} of int8, got {tuple(exps.shape)} of {exps.dtype}")
    _contig(codes, "codes")
    _contig(exps, "exponents")
    return pages, page_size


def qk_norm_rope_write8(qkv: torch.Tensor, nh: int, nkv: int, d: int, q_weight: Optional[torch.Tensor],
                        k_weight: Optional[torch.Tensor], eps: float, cos: Optional[torch.Tensor], sin: Optional[torch.Tensor],
                        rot: int, cache: Cache8, slot_mapping: torch.Tensor, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`qk_norm_rope_write` for a cache in 8 bits: per-head RMSNorm and rotate-half RoPE of q and k in a fused ``qkv``
    [n, (nh+2nkv)*d], which is left as it was; returns q [n, nh*d], and writes the keys (normed, rotated, rounded to the
    activations' type) and the values to ``cache`` at ``slot_mapping``.

    Tokens of one block of 16 must follow one another in the step, as a request's do, and no two name one slot (what such a block then
    holds is not said: its tokens may be on another's scale).  A block whose first token (place 0) is
    among them begins afresh; the older tokens of another one are rounded again when a new token needs a larger scale.  What
    is not finite is kept as NaN.  ``slot_mapping`` is index data: it is read ahead of the wait for the kernel before, and none of this package's
    kernels on its way may write it."""
    if qkv.is_cuda:
        lib = _lib("cache8")
        got = _native("write8", lib, "vapi_qk_norm_rope_write8", qkv, nh, nkv, d, q_weight, k_weight, eps, cos, sin, rot, cache[0], cache[1],
                      slot_mapping, _p(status))
        if got is not NotImplemented:
            _check(lib, got if type(got) is int else 0, int(qkv.shape[0] > 0))
            return got
    _contig(qkv, "qkv")
    for t, w in ((q_weight, "q norm weight"), (k_weight, "k norm weight"), (cos, "cos"), (sin, "sin")):
        _f32(t, w)
    _i32(slot_mapping, "slot mapping")
    _contig(slot_mapping, "slot mapping")
    if qkv.dim() != 2 or qkv.shape[1] != (nh + 2 * nkv) * d:
        raise KernelError(f"qkv is {tuple(qkv.shape)}, expected {(nh + 2 * nkv) * d} columns")
    n = qkv.shape[0]
    pages, page_size = _cache8(cache, nkv, d)
    _least(slot_mapping, n, "slot mapping")
    for t, w in ((q_weight, "q norm weight"), (k_weight, "k norm weight")):
        if t is not None and t.numel() != d:
            raise KernelError(f"the {w} must be [head_dim]")
    if (cos is None) != (sin is None) or (cos is not None and (tuple(cos.shape) != (n, rot // 2) or sin.shape != cos.shape)):
        raise KernelError("cos/sin must be [n, rot/2]")
    _cuda(qkv, q_weight, k_weight, cos, sin, cache.codes, cache.exps, slot_mapping)
    _here(qkv, q_weight, k_weight, cos, sin, cache.codes, cache.exps, slot_mapping)
    q = torch.empty((n, nh * d), dtype=qkv.dtype, device=qkv.device)
    lib = _lib("cache8")
    _check(lib, lib.vapi_qk_norm_rope_write8(_p(qkv), _dt(qkv), _p(q_weight), _p(k_weight), eps, _p(cos), _p(sin), rot, _p(q),
                                             _p(cache.codes), _p(cache.exps), _p(slot_mapping), n, nh, nkv, d, page_size, pages,
                                             _p(status), _stream()), launches=int(n > 0))
    return q


def cache8_read(cache: Cache8, pages: torch.Tensor, dtype: torch.dtype, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """What whole pages of a cache hold, [len(pages), 2, nkv, page_size, d] in ``dtype`` (bfloat16 holds every number of the
    cache exactly, and so does float32): to move a request's tokens to another cache, or to look at them."""
    if pages.is_cuda and dtype in (torch.bfloat16, torch.float32):
        lib = _lib("cache8")
        got = _native("read8", lib, "vapi_cache8_read", cache[0], cache[1], pages, int(dtype == torch.float32), _p(status))
        if got is not NotImplemented:
            _check(lib, got if type(got) is int else 0, int(pages.numel() > 0))
            return got
    _i32(pages, "pages")
    _contig(pages, "pages")
    nkv, d = (cache.codes.shape[2], cache.codes.shape[4]) if cache.codes.dim() == 5 else (0, 0)
    num_pages, page_size = _cache8(cache, nkv, d)
    _cuda(cache.codes, cache.exps, pages)
    _here(cache.codes, cache.exps, pages)
    out = torch.empty((pages.numel(), 2, nkv, page_size, d), dtype=dtype, device=cache.codes.device)
    lib = _lib("cache8")
    _check(lib, lib.vapi_cache8_read(_p(cache.codes), _p(cache.exps), _p(pages), _p(out), _dt(out), pages.numel(), nkv, d, page_size,
                                     num_pages, _p(status), _stream()), launches=int(pages.numel() > 0))
    return out


def attention8_splits(num_seqs: int, max_q: int, max_k: int, nh: int, nkv: int, d: int) -> int:
    """How many blocks (of eight warps) share the keys of one (sequence, kv head, tile of rows) in :func:`paged_attention8` when it is not
    told (the library's own rule): a power of two up to a cluster's 16, while all blocks are on the device at once and each warp still
    has two blocks of 16 tokens."""
    return int(_lib("cache8").vapi_attention8_splits(num_seqs, max_q, max_k, nh, nkv, d))


_IMPL8 = {"auto": 0, "general": 1, "tensor_core": 2, "tcgen05": 3}
#: portions shorter than this never go to the tcgen05 kernel beside other sequences (csrc/cache8_prompt.cuh)
_PORTION8_MIN_Q = 32


def paged_attention8(q: torch.Tensor, q_row_stride: int, cache: Cache8, block_table: torch.Tensor, cu_q: torch.Tensor,
                     seqlens_k: torch.Tensor, n: int, num_seqs: int, max_q: int, max_k: int, nh: int, nkv: int, d: int,
                     scale: float, window: int = 0, splits: Optional[int] = None, status: Optional[torch.Tensor] = None,
                     impl: str = "auto") -> torch.Tensor:
    """:func:`paged_attention` over a cache in 8 bits; returns [n, nh*d].  Arguments as there; the numbers of the cache are taken
    exactly, scores, softmax and sums are float32.  A query without a visible key gets zeros.  Pages before the window and behind a
    request's end are not looked at.  A value that is not a number reaches the queries that see its token, and on the tensor cores also those
    of the same portion that stand before it in one tile, as with :func:`paged_attention`.

    The cache may be the work of any kernel ahead on the stream.  Within ``one_stream(settled=True)`` what it holds before a sequence's own tokens of
    the call is read while kernels ahead still run, and must be none of theirs.  ``block_table``, ``cu_q`` and ``seqlens_k`` are index data, read
    ahead of that wait always: none of this package's kernels on its way may write them.

    ``impl``: "auto" picks: for bfloat16 and head size 64 or 128 the tcgen05 kernel for prompt portions (where rows and keys are enough for
    it), and the mma.sync kernel for the others, in both of which ``splits`` blocks (up to 16, and up to 8) share the keys as a cluster; the
    general kernel for every other type, head size (a multiple of 16 up to 256) and alignment.  "tcgen05", "tensor_core" and "general" force one (the first two raise where
    they do not apply)."""
    code = _IMPL8.get(impl)
    kernels = 1 if n > 0 else 0
    if (max_q >= _PORTION8_MIN_Q and num_seqs > 1 and code == 0 and q.dtype == torch.bfloat16 and d in (64, 128) and nkv > 0 and q.is_cuda and scale > 0
            and q_row_stride % 8 == 0 and q.data_ptr() % 16 == 0):
        kernels *= int(_lib("cache8").vapi_attention8_kernels(n, num_seqs, max_q, max_k, nh, nkv, d, window))
    if q.is_cuda and code is not None:
        lib = _lib("cache8")
        got = _native("attention8", lib, "vapi_paged_attention8", q, q_row_stride, cache[0], cache[1], block_table, cu_q, seqlens_k, n, num_seqs,
                      max_q, max_k, nh, nkv, d, scale, window, splits or 0, code, int(_held.settled), _p(status))
        if got is not NotImplemented:
            _check(lib, got if type(got) is int else 0, kernels)
            return got
    for t, w in ((block_table, "block table"), (cu_q, "cu_q"), (seqlens_k, "seqlens_k")):
        _i32(t, w)
    if impl not in _IMPL8:
        raise KernelError(f"impl `{impl}` is not one of {', '.join(_IMPL8)}")
    if nh <= 0 or nkv <= 0 or nh % nkv:
        raise KernelError(f"{nh} heads are not a multiple of {nkv} kv heads")
    if block_table.dim() != 2 or block_table.stride(1) != 1 or block_table.shape[0] < num_seqs:
        raise KernelError("block table must be [S, width] with unit inner stride")
    _contig(cu_q, "cu_q")
    _contig(seqlens_k, "seqlens_k")
    _least(cu_q, num_seqs + 1, "cu_q")
    _least(seqlens_k, num_seqs, "seqlens_k")
    if q.stride(-1) != 1 or q_row_stride < nh * d or (n > 0 and q.untyped_storage().nbytes() < (q.storage_offset() + (n - 1) * q_row_stride + nh * d) * q.element_size()):
        raise KernelError(f"q {tuple(q.shape)} does not hold {n} rows of {nh * d} at a stride of {q_row_stride}")
    pages, page_size = _cache8(cache, nkv, d)
    _cuda(q, cache.codes, cache.exps, block_table, cu_q, seqlens_k)
    _here(q, cache.codes, cache.exps, block_table, cu_q, seqlens_k)
    out = torch.empty((n, nh * d), dtype=q.dtype, device=q.device)
    lib = _lib("cache8")
    _check(lib, lib.vapi_paged_attention8(_p(q), q_row_stride, _p(cache.codes), _p(cache.exps), _dt(q), _p(block_table), block_table.stride(0),
                                          _p(cu_q), _p(seqlens_k), _p(out), n, num_seqs, max_q, max_k, nh, nkv, d, page_size, pages,
                                          scale, window, splits or 0, code, int(_held.settled), _p(status), _stream()), launches=kernels)
    return out
