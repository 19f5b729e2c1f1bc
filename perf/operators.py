"""Operators of serving in fewer bits, as cases that can be timed and compared: a cache of keys and values held in
8 bits (the write and the attention that reads it), matrix products with 4-bit weights, and the log probabilities
of given tokens, by which a user sees what the fewer bits cost.

A case is one pass through one operator:

* ``write``: a step's fused q/k/v product is normed and rotated, and its keys and values are quantised into the
  cache: codes are e4m3 numbers, and every block of 16 tokens of a head has one scale, a power of two, the smallest
  that lets the block's largest magnitude fit 448.  A token that needs a larger one than its block has makes the
  block's older tokens be rounded again on it.
* ``attend``: causal attention of a step's queries over such a cache.
* ``int4``: ``x W^T`` where W's numbers are ``(code - zero) * scale``, code and zero in 0..15, scale and zero for
  each group of columns of a row; with "swiglu" W is [Wg; Wu] and the result silu(x Wg^T) * (x Wu^T).
* ``logprobs``: for every row of logits the log probability of a given token, the entropy, and the most likely
  tokens with theirs, ties to the lowest id.

Sizes are those of the LFM2 models that ``bench.py`` serves, and head size 128 beside their 64.
"""
import math

import torch

#: set: `run` calls the framework's operators; else it computes the same with elementary torch operations
own = False

PAGE, BLOCK = 64, 16
EPS, THETA = 1e-5, 1000000.0
LARGEST, LEAST_EXP, MOST_EXP = 448.0, -110, 119


# ---- the cases ----------------------------------------------------------------------------------------

def listed():
    return [
        # a decode step of the benchmark's batch writes eight tokens behind long contexts: latency
        {"name": "write-8x1@4090", "kind": "write", "requests": 8, "tokens": 1, "past": 4089, "heads": 32, "kv_heads": 8, "head": 64},
        # a prompt portion of the default configuration, its first token inside a block
        {"name": "write-1x2048@2047", "kind": "write", "requests": 1, "tokens": 2048, "past": 2047, "heads": 32, "kv_heads": 8, "head": 64},
        # one user's answer, deep in a context: the smallest pass over a cache
        {"name": "attend-1x1@4090", "kind": "attend", "requests": 1, "shortest": 4090, "longest": 4090, "portion": 0,
         "heads": 32, "kv_heads": 8, "head": 64, "window": 0},
        # a full server: 64 requests of lengths 128 to 2,048
        {"name": "attend-64x1@128..2048", "kind": "attend", "requests": 64, "shortest": 128, "longest": 2048, "portion": 0,
         "heads": 32, "kv_heads": 8, "head": 64, "window": 0},
        # what an 8-bit cache is bought for: eight long contexts side by side
        {"name": "attend-8x1@32000", "kind": "attend", "requests": 8, "shortest": 31000, "longest": 32000, "portion": 0,
         "heads": 32, "kv_heads": 8, "head": 64, "window": 0},
        # the last portion of a document of 8,000 tokens
        {"name": "attend-1x2048@8000", "kind": "attend", "requests": 1, "shortest": 8000, "longest": 8000, "portion": 2048,
         "heads": 32, "kv_heads": 8, "head": 64, "window": 0},
        # one token through an output projection: the smallest product
        {"name": "int4-1x2048x2048", "kind": "int4", "rows": 1, "out": 2048, "inner": 2048, "group": 64, "form": "plain", "bias": False},
        # the gate|up product of the benchmark's batch, where most of a decode step's weights are
        {"name": "int4-8x16384x2048-swiglu", "kind": "int4", "rows": 8, "out": 16384, "inner": 2048, "group": 128, "form": "swiglu", "bias": False},
        # the down product of the 700M size with an odd number of requests, fine groups and a bias
        {"name": "int4-19x1536x6912", "kind": "int4", "rows": 19, "out": 1536, "inner": 6912, "group": 32, "form": "plain", "bias": True},
        # a prompt portion through the down product
        {"name": "int4-2048x2048x8192", "kind": "int4", "rows": 2048, "out": 2048, "inner": 8192, "group": 128, "form": "plain", "bias": False},
        # a decode step whose requests report log probabilities
        {"name": "logprobs-8x65536-top5", "kind": "logprobs", "rows": 8, "vocab": 65536, "top": 5, "dtype": "float32"},
        # scoring a document: every position of a portion
        {"name": "logprobs-2047x65536-top20", "kind": "logprobs", "rows": 2047, "vocab": 65536, "top": 20, "dtype": "float32"},
    ]


def draw(rng):
    def log_between(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    heads, kv_heads, head = rng.choice([(32, 8, 64), (24, 8, 64), (16, 8, 64), (32, 4, 64), (16, 4, 128), (32, 8, 128), (12, 2, 128)])
    kind = rng.choice(["write", "attend", "attend", "attend", "int4", "int4", "int4", "logprobs", "logprobs"])
    if kind == "write":
        if rng.random() < 0.5:
            return {"kind": "write", "requests": log_between(1, 64), "tokens": 1, "past": rng.randint(0, 1500),
                    "heads": heads, "kv_heads": kv_heads, "head": head}
        requests = rng.choice([1, 1, 2, 3])
        return {"kind": "write", "requests": requests, "tokens": log_between(2, 2048 // requests), "past": rng.randint(0, 1500),
                "heads": heads, "kv_heads": kv_heads, "head": head}
    if kind == "attend":
        form = rng.choice(["decode", "decode", "portion", "mixed"])
        window = rng.choice([0, 0, 0, rng.randint(1, 1500)])
        if form == "decode":
            requests = log_between(1, 64)
            longest = min(log_between(1, 32000), 250000 // requests)
            return {"kind": "attend", "requests": requests, "shortest": rng.randint(max(1, longest // 8), longest), "longest": longest,
                    "portion": 0, "heads": heads, "kv_heads": kv_heads, "head": head, "window": window}
        requests = 1 if form == "portion" else log_between(2, 32)
        portion = log_between(2, 2000) if requests == 1 else log_between(2, 500)
        longest = portion + rng.randint(0, 5000 if requests == 1 else 1500)
        return {"kind": "attend", "requests": requests, "shortest": max(1, longest // rng.randint(1, 8)), "longest": longest,
                "portion": portion, "heads": heads, "kv_heads": kv_heads, "head": head, "window": window}
    if kind == "int4":
        group = rng.choice([32, 64, 128])
        rows = log_between(1, 64) if rng.random() < 0.7 else log_between(65, 2048)
        out, inner = rng.choice([(2048, 2048), (6144, 2048), (16384, 2048), (2048, 8192), (1536, 1536), (4608, 1536), (13824, 1536),
                                 (1536, 6912), (16 * rng.randint(4, 500), 128 * rng.randint(2, 60))])
        form = "swiglu" if out >= 4608 and rng.random() < 0.5 else "plain"
        return {"kind": "int4", "rows": rows, "out": out, "inner": inner, "group": group, "form": form,
                "bias": form == "plain" and rng.random() < 0.3}
    rows = log_between(1, 2000)
    vocab = rng.choice([65536, 65536, 509, 1003, 4099, 128256, 151936])
    rows = min(rows, 2000 * 65536 // max(vocab, 65536))
    return {"kind": "logprobs", "rows": rows, "vocab": vocab, "top": rng.choice([0, 1, 5, 20, rng.randint(2, 20)]),
            "dtype": rng.choice(["float32", "float32", "bfloat16"])}


def lengths(case):
    """The requests' lengths: spread evenly from the shortest to the longest, long and short ones in turn."""
    n, lo, hi = case["requests"], case["shortest"], case["longest"]
    even = [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]
    return [even[n - 1 - i // 2] if i % 2 == 0 else even[i // 2] for i in range(n)]


def portions(case):
    """How many tokens each request brings: one, and the longest (the first) its portion."""
    lens = lengths(case)
    return [min(case["portion"], lens[0]) if case["portion"] and i == 0 else 1 for i in range(len(lens))]


# ---- inputs -------------------------------------------------------------------------------------------

def pages_of(lens, generator):
    """A block table [S, width] of pages taken in random order, and how many pages there are."""
    need = [-(-n // PAGE) for n in lens]
    order = torch.randperm(sum(need) + 1, generator=generator)
    table = torch.zeros((len(lens), max(need)), dtype=torch.int32)
    at = 0
    for s, k in enumerate(need):
        table[s, :k] = order[at:at + k].int()
        at += k
    return table, sum(need) + 1


def scale_exponent(amax):
    """The smallest e in LEAST_EXP .. MOST_EXP with amax <= 448 * 2^e (448 = 1.75 * 2^8), from amax = m * 2^x, m in [1/2, 1)."""
    m, x = torch.frexp(amax)
    return (x - 9 + (m > 0.875)).clamp(LEAST_EXP, MOST_EXP)


def power_of_two(e):
    """2^e in float32, from its bits (e in -126 .. 127)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def to_codes(x, exps):
    """e4m3 numbers of x / 2^exps, rounded to nearest even, no magnitude above 448; NaN for what is not finite."""
    y = x.float() * power_of_two(-exps.int())
    y = torch.where(torch.isfinite(y), y.clamp(-LARGEST, LARGEST), torch.full_like(y, float("nan")))
    return y.to(torch.float8_e4m3fn)


def random_cache(pages, kv_heads, head, g):
    """A cache whose every block was written whole: channels and tokens of unlike size, as keys and values have them."""
    shape = (pages, 2, kv_heads, PAGE // BLOCK, BLOCK, head)
    x = torch.randn(shape, generator=g, device="cuda")
    x *= torch.exp(0.7 * torch.randn((1, 2, kv_heads, 1, 1, head), generator=g, device="cuda"))
    x *= torch.exp(0.3 * torch.randn((pages, 2, kv_heads, PAGE // BLOCK, BLOCK, 1), generator=g, device="cuda"))
    exps = scale_exponent(x.abs().amax((-1, -2))).to(torch.int8)
    codes = to_codes(x, exps[..., None, None])
    return codes.view(pages, 2, kv_heads, PAGE, head), exps


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    dev = lambda t: t.cuda()
    s = {"case": case}
    if case["kind"] in ("write", "attend"):
        nh, nkv, d = case["heads"], case["kv_heads"], case["head"]
        if case["kind"] == "write":
            news = [case["tokens"]] * case["requests"]
            lens = [case["past"] + case["tokens"]] * case["requests"]
        else:
            lens, news = lengths(case), portions(case)
        table, pages = pages_of(lens, host)
        codes, exps = random_cache(pages, nkv, d, g)
        s.update(codes=codes, exps=exps, table=dev(table), n=sum(news), requests=len(lens), max_q=max(news), max_k=max(lens))
        cu = [0]
        for q in news:
            cu.append(cu[-1] + q)
        s["cu_q"] = dev(torch.tensor(cu, dtype=torch.int32))
        s["seqlens_k"] = dev(torch.tensor(lens, dtype=torch.int32))
        seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(news))
        pos = torch.cat([torch.arange(n - q, n) for n, q in zip(lens, news)])
        if case["kind"] == "write":
            s["qkv"] = torch.randn(s["n"], (nh + 2 * nkv) * d, generator=g, device="cuda").bfloat16()
            s["q_weight"], s["k_weight"] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda") for _ in range(2))
            angle = pos[:, None].float() * torch.pow(THETA, -2.0 * torch.arange(d // 2, dtype=torch.float64) / d).float()
            s["cos"], s["sin"] = dev(angle.cos()), dev(angle.sin())
            slots = table[seq, pos // PAGE] * PAGE + pos % PAGE
            s["slots"] = dev(slots.to(torch.int32))
            # the pages that the step writes to (what comes back as the updated state)
            s["pages"] = dev(torch.unique(slots // PAGE).to(torch.int32))
        else:
            s["q"] = (1.2 * torch.randn(s["n"], (nh + 2 * nkv) * d, generator=g, device="cuda")).bfloat16()
            # what lies behind a request's end in its last page was never written: it may be anything, NaN among it
            tail = torch.arange(PAGE)
            for i, n in enumerate(lens):
                if n % PAGE:
                    codes.view(torch.uint8)[int(table[i, (n - 1) // PAGE]), :, :, dev(tail[n % PAGE:])] = 0x7f
        if own:
            from vapi_b200 import ops
            s["cache"] = ops.Cache8(codes, exps)
    elif case["kind"] == "int4":
        n, k, group = case["out"], case["inner"], case["group"]
        w = torch.randn(n, k // group, group, generator=g, device="cuda") * (k ** -0.5)
        w *= torch.exp(0.4 * torch.randn(n, 1, 1, generator=g, device="cuda"))
        lo, hi = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
        scales = ((hi - lo) / 15).clamp(min=1e-8).bfloat16()
        zeros = torch.round(-lo / scales.float()).clamp(0, 15)
        s["codes"] = (torch.round(w / scales.float()[..., None]) + zeros[..., None]).clamp(0, 15).to(torch.uint8).view(n, k)
        s["scales"], s["zeros"] = scales, zeros.to(torch.uint8)
        x = torch.randn(case["rows"], k, generator=g, device="cuda")
        x[:, torch.randint(0, k, (max(1, k // 256),), generator=g, device="cuda")] *= 8      # a few channels stand out
        s["x"] = x.bfloat16()
        s["bias"] = torch.randn(n, generator=g, device="cuda") if case["bias"] else None
        if own:
            from vapi_b200 import ops
            s["weight"] = ops.int4_pack(s["codes"], s["scales"], s["zeros"])
            del s["codes"], s["scales"], s["zeros"]
    else:
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn(rows, vocab, generator=g, device="cuda") * 2.5
        x[torch.arange(rows, device="cuda"), torch.randint(0, vocab, (rows,), generator=g, device="cuda")] += 9
        # half of the given tokens are likely ones, as a text's are
        tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        tokens[::2] = x[::2].argmax(1)
        s["logits"] = x.to(getattr(torch, case["dtype"]))
        s["tokens"] = tokens.to(torch.int32)
    return s


# ---- one pass -----------------------------------------------------------------------------------------

def run(s):
    case = s["case"]
    if case["kind"] == "write":
        return run_write(s, case)
    if case["kind"] == "attend":
        return run_attend(s, case)
    return run_int4(s, case) if case["kind"] == "int4" else run_logprobs(s, case)


def normed_and_rotated(x, weight, cos, sin):
    """Per-head RMS norm and rotation of the pairs (i, i + d/2), rounded to bfloat16; x is [n, heads, d] in float32."""
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).bfloat16()


def run_write(s, case):
    nh, nkv, d = case["heads"], case["kv_heads"], case["head"]
    if own:
        from vapi_b200 import ops
        q = ops.qk_norm_rope_write8(s["qkv"], nh, nkv, d, s["q_weight"], s["k_weight"], EPS, s["cos"], s["sin"], d, s["cache"], s["slots"])
        return {"q": q, "pages": ops.cache8_read(s["cache"], s["pages"], torch.bfloat16)}
    n, codes, exps = s["n"], s["codes"], s["exps"]
    x = s["qkv"].float().view(n, nh + 2 * nkv, d)
    cos, sin = s["cos"][:, None], s["sin"][:, None]
    q = normed_and_rotated(x[:, :nh], s["q_weight"], cos, sin)
    kv = torch.stack([normed_and_rotated(x[:, nh:nh + nkv], s["k_weight"], cos, sin).float(), x[:, nh + nkv:]], 1)      # [n, 2, nkv, d]
    # a token's block: its number among all blocks of the cache, and the token's place in it
    slots = s["slots"].long()
    block, place = slots // BLOCK, slots % BLOCK
    pages, blocks = codes.shape[0], codes.shape[0] * (PAGE // BLOCK)
    first = torch.full((blocks,), BLOCK, device="cuda").scatter_reduce(0, block, place, "amin")
    amax = kv.abs().amax(-1)                                                               # [n, 2, nkv]
    amax = torch.zeros((blocks, 2, nkv), device="cuda").scatter_reduce(0, block[:, None, None].expand_as(amax), amax, "amax")
    old = exps.permute(0, 3, 1, 2).reshape(blocks, 2, nkv).int()
    need = scale_exponent(amax).int()
    new = torch.where((first < BLOCK)[:, None, None], torch.where((first > 0)[:, None, None], torch.maximum(old, need), need), old)
    # older tokens of a block, on its new scale
    c = codes.view(pages, 2, nkv, PAGE // BLOCK, BLOCK, d).permute(0, 3, 1, 2, 4, 5).reshape(blocks, 2, nkv, BLOCK, d)
    touched = torch.unique(block)
    older = torch.arange(BLOCK, device="cuda") < first[touched][:, None]
    again = to_codes(c[touched].float(), (new - old).clamp(0, 126)[touched][..., None, None])      # (2^-126 of any code rounds to zero)
    page, part = touched // (PAGE // BLOCK), touched % (PAGE // BLOCK)
    whole = torch.where(older[:, None, None, :, None], again.float(), c[touched].float()).to(torch.float8_e4m3fn)
    codes.view(torch.uint8).view(pages, 2, nkv, PAGE // BLOCK, BLOCK, d)[page, :, :, part] = whole.view(torch.uint8)
    exps[page, :, :, part] = new[touched].to(torch.int8)
    codes.view(torch.uint8)[slots // PAGE, :, :, slots % PAGE] = to_codes(kv, new[block][..., None]).view(torch.uint8)
    return {"q": q.view(n, nh * d), "pages": values_of(codes, exps, s["pages"]).bfloat16()}


def values_of(codes, exps, pages):
    """What the codes of these pages stand for, [pages, 2, kv heads, PAGE, head]."""
    pages = pages.long()
    c = codes.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float()
    return c * power_of_two(exps[pages]).repeat_interleave(BLOCK, -1)[..., None]


def run_attend(s, case):
    nh, nkv, d, window = case["heads"], case["kv_heads"], case["head"], case["window"]
    width = (nh + 2 * nkv) * d
    if own:
        from vapi_b200 import ops
        return ops.paged_attention8(s["q"], width, s["cache"], s["table"], s["cu_q"], s["seqlens_k"], s["n"], s["requests"], s["max_q"],
                                    s["max_k"], nh, nkv, d, d ** -0.5, window)
    S, max_q, max_k = s["requests"], s["max_q"], s["max_k"]
    kv = values_of(s["codes"], s["exps"], s["table"].reshape(-1)).view(S, -1, 2, nkv, PAGE, d)
    kv = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, S, nkv, -1, d)[:, :, :, :max_k]
    klen, q0 = s["seqlens_k"].long(), s["cu_q"].long()
    qlen = q0[1:] - q0[:-1]
    # queries one sequence a row, padded to the longest portion
    j = torch.arange(max_q, device="cuda")
    rows = torch.where(j < qlen[:, None], q0[:-1, None] + j, 0)
    q = s["q"][:, :nh * d].float()[rows].view(S, max_q, nkv, nh // nkv, d).permute(0, 2, 3, 1, 4)      # [S, nkv, rep, max_q, d]
    at = (klen - qlen)[:, None] + j
    key = torch.arange(kv.shape[3], device="cuda")
    sees = (key <= at[..., None]) & (key < klen[:, None, None]) & (j < qlen[:, None])[..., None]
    if window:
        sees &= key > at[..., None] - window
    used = (key < klen[:, None])[:, None, :, None]
    k, v = torch.where(used, kv[0], 0), torch.where(used, kv[1], 0)
    scores = (q.reshape(S, nkv, -1, d) @ k.transpose(-1, -2)).view(S, nkv, nh // nkv, max_q, -1) * d ** -0.5
    scores = scores.masked_fill_(~sees[:, None, None], float("-inf"))
    scores = scores.sub_(scores.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = (scores.view(S, nkv, -1, scores.shape[-1]) @ v).view(S, nkv, nh // nkv, max_q, d) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(S, max_q, nh * d)
    return out[j < qlen[:, None]].to(s["q"].dtype)


def run_int4(s, case):
    if own:
        from vapi_b200 import ops
        if case["form"] == "swiglu":
            return ops.int4_linear_swiglu(s["x"], s["weight"])
        return ops.int4_linear(s["x"], s["weight"], s["bias"])
    n, k = s["codes"].shape
    w = (s["codes"].float().view(n, -1, case["group"]) - s["zeros"].float()[..., None]) * s["scales"].float()[..., None]
    y = s["x"].float() @ w.view(n, k).t()
    if s["bias"] is not None:
        y = y + s["bias"]
    if case["form"] == "swiglu":
        gate, up = y.chunk(2, 1)
        y = gate / (1 + torch.exp(-gate)) * up
    return y.to(s["x"].dtype)


def run_logprobs(s, case):
    if own:
        from vapi_b200 import ops
        r = ops.token_logprobs(s["logits"], s["tokens"], case["top"])
        return {"logprob": r.logprob, "entropy": r.entropy, "top_ids": r.top_ids, "top_logprobs": r.top_logprobs}
    x = s["logits"].float()
    lp = x - x.amax(1, keepdim=True)
    lp = lp - lp.exp().sum(1, keepdim=True).log()
    best, ids = torch.sort(x, dim=1, descending=True, stable=True)
    ids = ids[:, :case["top"]]
    return {"logprob": lp.gather(1, s["tokens"].long()[:, None])[:, 0], "entropy": -(lp.exp() * lp).sum(1),
            "top_ids": ids.to(torch.int32), "top_logprobs": lp.gather(1, ids)}


# ---- what a pass cannot do without --------------------------------------------------------------------

def work(case):
    if case["kind"] in ("write", "attend"):
        nh, nkv, d = case["heads"], case["kv_heads"], case["head"]
    if case["kind"] == "write":
        n = case["requests"] * case["tokens"]
        pages = case["requests"] * ((case["past"] + case["tokens"] - 1) // PAGE - case["past"] // PAGE + 1)
        moved = n * ((nh + 2 * nkv) * d * 2 + nh * d * 2 + 2 * nkv * d + 4 * d + 4)
        return {"bytes": moved + pages * 2 * nkv * PAGE * d * 3, "flops": n * (nh + 2 * nkv) * d * 8}
    if case["kind"] == "attend":
        pairs = keys = 0
        for k, q in zip(lengths(case), portions(case)):
            w = case["window"] or k
            keys += min(k, w + q - 1)
            # sum over the portion's queries of the keys each sees
            full = max(0, min(q, k - max(w, k - q)))
            pairs += full * w + sum(range(k - q + 1, k - full + 1))
        n = sum(portions(case))
        return {"bytes": keys * 2 * nkv * (d + 1 / BLOCK) + 4 * n * nh * d, "flops": 4 * pairs * nh * d}
    if case["kind"] == "int4":
        m, n, k = case["rows"], case["out"], case["inner"]
        wide = n // 2 if case["form"] == "swiglu" else n
        return {"bytes": n * k // 2 + n * (k // case["group"]) * 2.5 + 2 * m * k + 2 * m * wide, "flops": 2 * m * n * k}
    r, v = case["rows"], case["vocab"]
    return {"bytes": r * v * (4 if case["dtype"] == "float32" else 2) + r * (12 + 8 * case["top"]), "flops": 5 * r * v}


# ---- the same in 64 bits, from the definitions --------------------------------------------------------

def exact(case, seed):
    global own
    before, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = before
    return {"write": exact_write, "attend": exact_attend, "int4": exact_int4, "logprobs": exact_logprobs}[case["kind"]](s, case)


def exact_write(s, case):
    """The queries; what the cache then holds is a choice among 8-bit numbers, not a value of its own."""
    nh, d = case["heads"], case["head"]
    x = s["qkv"].double()[:, :nh * d].view(-1, nh, d)
    x = x / (x.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * s["q_weight"].double()
    c, sn = s["cos"].double()[:, None], s["sin"].double()[:, None]
    half = d // 2
    y = torch.empty_like(x)
    y[..., :half] = x[..., :half] * c - x[..., half:] * sn
    y[..., half:] = x[..., half:] * c + x[..., :half] * sn
    return {"q": y.reshape(-1, nh * d), "pages": None}


def exact_attend(s, case):
    nh, nkv, d, window = case["heads"], case["kv_heads"], case["head"], case["window"]
    rep, out, at = nh // nkv, [], 0
    for i, (n, new) in enumerate(zip(lengths(case), portions(case))):
        pages = s["table"][i, :-(-n // PAGE)].long()
        power = torch.pow(2.0, s["exps"][pages].double())
        codes = s["codes"].view(torch.uint8)[pages].view(torch.float8_e4m3fn).double()
        kv = codes.view(len(pages), 2, nkv, PAGE // BLOCK, BLOCK, d) * power[..., None, None]
        kv = kv.permute(1, 2, 0, 3, 4, 5).reshape(2, nkv, -1, d)[:, :, :n]
        q = s["q"][at:at + new, :nh * d].double().view(new, nkv, rep, d)
        place = torch.arange(n - new, n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")[None]
        hidden = key > place
        if window:
            hidden |= key <= place - window
        heads = []
        for g in range(nkv):
            score = torch.einsum("qrd,kd->rqk", q[:, g], kv[0, g]) / math.sqrt(d)
            p = torch.softmax(score.masked_fill(hidden, float("-inf")), -1)
            heads.append(torch.einsum("rqk,kd->qrd", p, kv[1, g]))
        out.append(torch.cat(heads, 1).reshape(new, nh * d))
        at += new
    return torch.cat(out)


def exact_int4(s, case):
    group = case["group"]
    scale = s["scales"].double().repeat_interleave(group, 1)
    w = scale * (s["codes"].double() - s["zeros"].double().repeat_interleave(group, 1))
    y = torch.einsum("mk,nk->mn", s["x"].double(), w)
    if s["bias"] is not None:
        y += s["bias"].double()
    if case["form"] == "swiglu":
        half = y.shape[1] // 2
        return y[:, :half] * torch.sigmoid(y[:, :half]) * y[:, half:]
    return y


def exact_logprobs(s, case):
    top = case["top"]
    logprob, entropy, ids, tops = [], [], [], []
    for x, t in zip(s["logits"].split(256), s["tokens"].long().split(256)):
        lse = torch.logsumexp(x.double(), 1, keepdim=True)
        lp = x.double() - lse
        logprob.append(lp[torch.arange(len(t), device="cuda"), t])
        entropy.append((lse[:, 0] - (lp.exp() * x.double()).sum(1)))
        order = torch.argsort(-x.float(), dim=1, stable=True)[:, :top]
        ids.append(order.to(torch.int32))
        tops.append(torch.take_along_dim(lp, order, 1))
    return {"logprob": torch.cat(logprob), "entropy": torch.cat(entropy), "top_ids": torch.cat(ids), "top_logprobs": torch.cat(tops)}
