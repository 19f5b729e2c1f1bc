"""The operators of serving in fewer bits from their definitions, in 64 bits on the host: what their kernels are tested against,
and (:data:`OPS`) what stands in for them where host logic runs without a device."""
import math

import torch

BLOCK = 16


def exponent(amax: float) -> int:
    """The smallest e in -110..119 with amax <= 448 * 2^e."""
    e = -110
    while e < 119 and amax > 448.0 * 2.0 ** e:
        e += 1
    return e


def code(x: torch.Tensor, e: int) -> torch.Tensor:
    """The nearest e4m3 numbers of x / 2^e (float64), magnitudes above 448 as 448, NaN for what is not finite."""
    y = x.double() * 2.0 ** -e
    y = torch.where(torch.isfinite(y), y.clamp(-448.0, 448.0), torch.full_like(y, math.nan))
    # (exactly: to the grid of the number's own binade, at least 2^-9 apart)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(y / step) * step).to(torch.float8_e4m3fn)


def write(codes, exps, k, v, slots):
    """The step's keys and values [n, nkv, d] into the cache (host tensors, in place), block by block."""
    page_size, pages = codes.shape[3], codes.shape[0]
    n, at = len(slots), 0
    while at < n:
        slot, count = int(slots[at]), 1
        while at + count < n and int(slots[at + count]) == slot + count and (slot + count) % BLOCK:
            count += 1
        page, off = slot // page_size, slot % page_size
        place = off % BLOCK
        if 0 <= page < pages and slot >= 0:
            for kind, x in ((0, k), (1, v)):
                for g in range(x.shape[1]):
                    new = x[at:at + count, g].double()
                    fin = new[torch.isfinite(new)].abs()
                    e = exponent(float(fin.max()) if fin.numel() else 0.0)
                    old = int(exps[page, kind, g, off // BLOCK])
                    first = off - place
                    if place:
                        if old < e:
                            older = codes[page, kind, g, first:off].double() * 2.0 ** max(old - e, -126)
                            codes[page, kind, g, first:off] = code(older, 0)
                        e = max(e, old)
                    exps[page, kind, g, off // BLOCK] = e
                    codes[page, kind, g, off:off + count] = code(new, e)
        at += count


def values(codes, exps):
    """What a cache holds, float64 [pages, 2, nkv, page_size, d]."""
    return codes.double() * torch.exp2(exps.double()).repeat_interleave(BLOCK, -1)[..., None]


def attention(q, kv, block_table, cu_q, seqlens_k, nh, nkv, d, scale, window=0):
    """(output, sum of weight * |value|, largest sum |q||k| * scale of a row) in float64; q [n, nh*d], kv as :func:`values` gives it."""
    page = kv.shape[3]
    out = torch.zeros((q.shape[0], nh * d), dtype=torch.float64)
    spread, most = torch.zeros_like(out), 0.0
    for s in range(len(seqlens_k)):
        q0, q1, klen = int(cu_q[s]), int(cu_q[s + 1]), int(seqlens_k[s])
        if q1 == q0 or klen <= 0:
            continue
        pages = block_table[s, :-(-klen // page)].long()
        both = kv[pages].permute(1, 2, 0, 3, 4).reshape(2, nkv, -1, d)[:, :, :klen]
        x = q[q0:q1].double().view(q1 - q0, nkv, nh // nkv, d)
        pos = torch.arange(klen - (q1 - q0), klen)[:, None]
        key = torch.arange(klen)[None]
        sees = (key <= pos) & ((key > pos - window) if window > 0 else True)
        for g in range(nkv):
            sc = torch.einsum("qrd,kd->qrk", x[:, g], both[0, g]) * scale
            sc = sc.masked_fill(~sees[:, None], -math.inf)
            top = sc.amax(-1, keepdim=True)
            w = torch.exp(sc - torch.where(torch.isfinite(top), top, 0.0))
            total = w.sum(-1, keepdim=True)
            w = torch.where(total > 0, w / total, 0.0)
            vals = torch.where(sees.any(0)[:, None], both[1, g], 0.0)
            out.view(-1, nkv, nh // nkv, d)[q0:q1, g] = torch.einsum("qrk,kd->qrd", w, vals)
            spread.view(-1, nkv, nh // nkv, d)[q0:q1, g] = torch.einsum("qrk,kd->qrd", w, vals.abs())
            keys = torch.where(sees.any(0)[:, None], both[0, g].abs(), 0.0)
            most = max(most, float((torch.einsum("qrd,kd->qrk", x[:, g].abs(), keys) * scale).max()))
    return out, spread, most


# ---- stand-ins for the framework's functions ----------------------------------------------------------

def qk_norm_rope_write8(qkv, nh, nkv, d, q_weight, k_weight, eps, cos, sin, rot, cache, slot_mapping, status=None):
    import plain_ops
    n, page = qkv.shape[0], cache.codes.shape[3]
    x = qkv.clone()
    room = torch.zeros((1, 2, nkv, max(16, -(-n // 16) * 16), d), dtype=qkv.dtype)
    plain_ops.qk_norm_rope_write(x, nh, nkv, d, q_weight, k_weight, eps, cos, sin, rot, room, torch.arange(n, dtype=torch.int32), None)
    k, v = (room[0, i, :, :n].transpose(0, 1) for i in (0, 1))
    assert page % BLOCK == 0
    write(cache.codes, cache.exps, k, v, slot_mapping[:n])
    return x[:, :nh * d].contiguous()


def paged_attention8(q, q_row_stride, cache, block_table, cu_q, seqlens_k, n, num_seqs, max_q, max_k, nh, nkv, d, scale, window=0,
                     splits=None, status=None, impl="auto"):
    assert q_row_stride == q.stride(0)
    return attention(q[:n, :nh * d], values(cache.codes, cache.exps), block_table, cu_q[:num_seqs + 1], seqlens_k[:num_seqs], nh, nkv, d,
                     scale, window)[0].to(q.dtype)


def attention8_splits(num_seqs, max_q, max_k, nh, nkv, d):
    return 1


OPS = ["qk_norm_rope_write8", "paged_attention8", "attention8_splits"]


def token_logprobs(logits, tokens, top=0, status=None, slices=0):
    from vapi_b200 import ops
    lp = torch.log_softmax(logits.double(), 1)
    ids = torch.argsort(-logits.double(), dim=1, stable=True)[:, :top]
    return ops.TokenLogprobs(lp.gather(1, tokens.long()[:, None])[:, 0].float(), -torch.where(lp > -math.inf, lp.exp() * lp, 0.0).sum(1).float(),
                             ids.to(torch.int32), lp.gather(1, ids).float())


OPS += ["token_logprobs"]


def unpack(w):
    """(codes, scales, zeros) of an Int4Weight, read from its words bit by bit (host)."""
    words, pairs = w.codes.cpu(), w.scales.cpu()
    tiles, chunks = words.shape[:2]
    codes = torch.zeros(tiles, 2, 8, chunks, 4, 2, 4, 2, dtype=torch.uint8)
    lanes = words.view(tiles, chunks, 8, 4, 4)
    for h in range(2):
        for p in range(2):
            for e in range(2):
                codes[:, h, :, :, :, p, :, e] = ((lanes >> (8 * p + 4 * h + 16 * e)) & 15).permute(0, 2, 1, 4, 3).to(torch.uint8)
    table = pairs.permute(0, 3, 2, 1).reshape(tiles * 16, -1)[:w.n, :w.k // w.group]
    number = lambda t: (t & 0xffff).to(torch.int16).view(torch.bfloat16)
    return codes.reshape(tiles * 16, chunks * 64)[:w.n, :w.k], number(table), number(table >> 16) - 128


def int4_numbers(w):
    codes, scales, zeros = unpack(w)
    return (codes.double() - zeros.double().repeat_interleave(w.group, 1)) * scales.double().repeat_interleave(w.group, 1)


def int4_linear(x, w, bias=None, out_dtype=None):
    y = x.double() @ int4_numbers(w).t()
    return (y if bias is None else y + bias.double()).to(out_dtype or x.dtype)


def int4_linear_swiglu(x, w, act="silu"):
    import plain_ops
    return plain_ops.swiglu(int4_linear(x, w, out_dtype=torch.float32), act).to(x.dtype)


OPS += ["int4_linear", "int4_linear_swiglu"]
