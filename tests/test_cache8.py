"""The cache in 8 bits (csrc/cache8.cu): what the write quantises, what the read gives back, attention over it, and refusals."""
import math

import pytest
import torch

import plain_fewer_bits as plain

gpu = pytest.mark.gpu


def _ops():
    from vapi_b200 import ops
    return ops


# ---- refusals (no device) -----------------------------------------------------------------------------

def _step(n=3, nh=4, nkv=2, d=64, pages=2, page=32, dtype=torch.bfloat16):
    cache = _ops().cache8_empty(pages, nkv, page, d, "cpu")
    return dict(qkv=torch.zeros(n, (nh + 2 * nkv) * d, dtype=dtype), cache=cache, slots=torch.arange(n, dtype=torch.int32), nh=nh, nkv=nkv, d=d)


def _write(s, **kw):
    a = dict(q_weight=None, k_weight=None, eps=1e-5, cos=None, sin=None, rot=s["d"])
    a.update(kw)
    return _ops().qk_norm_rope_write8(s["qkv"], s["nh"], s["nkv"], s["d"], a["q_weight"], a["k_weight"], a["eps"], a["cos"], a["sin"], a["rot"],
                                      s["cache"], s["slots"])


def test_the_write_refuses_what_does_not_fit():
    ops = _ops()
    with pytest.raises(ops.KernelError, match="multiple of 16"):
        ops.cache8_empty(2, 2, 24, 64, "cpu")
    for change, words in ((dict(qkv=torch.zeros(3, 500)), "columns"), (dict(slots=torch.arange(3)), "int32"),
                          (dict(slots=torch.arange(2, dtype=torch.int32)), "fewer than 3"),
                          (dict(qkv=torch.zeros(512, 3).t()), "contiguous"), (dict(d=32), "columns"),
                          (dict(cache=ops.Cache8(torch.zeros(2, 2, 2, 32, 64), torch.zeros(2, 2, 2, 2, dtype=torch.int8))), "float8"),
                          (dict(cache=ops.Cache8(_step()["cache"].codes, torch.zeros(2, 2, 2, 1, dtype=torch.int8))), "exponents"),
                          (dict(cache=ops.Cache8(_step()["cache"].codes.transpose(2, 3).contiguous().transpose(2, 3), _step()["cache"].exps)), "contiguous")):
        with pytest.raises(ops.KernelError, match=words):
            _write({**_step(), **change})
    for kw, words in ((dict(q_weight=torch.ones(32)), "head_dim"), (dict(k_weight=torch.ones(64, dtype=torch.bfloat16)), "float32"),
                      (dict(cos=torch.zeros(3, 32)), "cos/sin"), (dict(cos=torch.zeros(3, 16), sin=torch.zeros(3, 16)), "cos/sin")):
        with pytest.raises(ops.KernelError, match=words):
            _write(_step(), **kw)
    with pytest.raises(ops.KernelError, match="CUDA"):
        _write(_step())


def test_attention_and_the_read_refuse_what_does_not_fit():
    ops = _ops()
    s = _step()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    good = dict(q=torch.zeros(3, 256, dtype=torch.bfloat16), stride=256, cache=s["cache"], table=i32(0, 1).view(1, 2), cu=i32(0, 3), kl=i32(5),
                n=3, S=1, nh=4, nkv=2, d=64, impl="auto")

    def call(**kw):
        a = {**good, **kw}
        return ops.paged_attention8(a["q"], a["stride"], a["cache"], a["table"], a["cu"], a["kl"], a["n"], a["S"], 3, 5, a["nh"], a["nkv"], a["d"],
                                    0.125, impl=a["impl"])
    for kw, words in ((dict(impl="fast"), "not one of"), (dict(nh=3), "multiple of 2"), (dict(table=i32(0, 1)), "block table"), (dict(S=2), "block table"),
                      (dict(cu=i32(3)), "cu_q"), (dict(cu=torch.tensor([0, 3])), "int32"), (dict(stride=512), "does not hold"), (dict(stride=128), "does not hold"),
                      (dict(n=4), "does not hold"), (dict(d=32), "codes"), (dict(), "CUDA")):
        with pytest.raises(ops.KernelError, match=words):
            call(**kw)
    with pytest.raises(ops.KernelError, match="int32"):
        ops.cache8_read(s["cache"], torch.tensor([0]), torch.bfloat16)
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.cache8_read(s["cache"], i32(0), torch.bfloat16)


def test_the_plain_codes_are_the_types_own_rounding():
    """(the stand-in's arithmetic against torch's conversion, on every kind of number)"""
    x = torch.cat([torch.randn(2000, generator=torch.Generator().manual_seed(1)) * 10 ** torch.linspace(-4, 2.5, 2000),
                   torch.tensor([0.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -6, 448.0, 447.0, 17.0, 19.0, -18.0])]).clamp(-448, 448)
    assert torch.equal(plain.code(x, 0).float(), x.to(torch.float8_e4m3fn).float())
    for a in (0.0, 1e-38, 1.0, 448.0, 449.0, 3.3e38, 447.9 * 2.0 ** 20):
        e = plain.exponent(a)
        assert (a <= 448 * 2.0 ** e or e == 119) and (e == -110 or a > 448 * 2.0 ** (e - 1))


# ---- the write ----------------------------------------------------------------------------------------

def _same(a, b, what=""):
    a, b = a.float().cpu(), b.float().cpu()
    assert torch.equal(torch.isnan(a), torch.isnan(b)), what
    assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)), (what, int((torch.nan_to_num(a) != torch.nan_to_num(b)).sum()))


def _random_qkv(n, nh, nkv, d, seed, dtype):
    """Rows whose magnitudes go from tiny to huge, so that blocks' scales grow from step to step; some rows of zeros."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, nh + 2 * nkv, d, generator=g) * torch.exp(3 * torch.randn(n, nh + 2 * nkv, 1, generator=g))
    x[torch.rand(n, nh + 2 * nkv, generator=g) < 0.1] = 0
    return x.view(n, -1).to(dtype)


# steps of these many tokens, one after the other, of two requests side by side
@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nh,nkv,d,page", [(4, 2, 64, 64), (3, 1, 16, 16), (2, 2, 128, 32), (6, 3, 48, 48), (1, 1, 256, 16)])
def test_the_write_is_the_definition_bit_by_bit(nh, nkv, d, page, dtype):
    ops = _ops()
    # (the last one is a prompt's, where a warp takes 16 tokens)
    steps, pages = (1, 1, 5, 16, 1, 30, 2, 17, 1, 600), -(-700 // page)
    g = torch.Generator().manual_seed(d)
    order = torch.randperm(2 * pages + 1, generator=g)
    codes = torch.randint(0, 256, (2 * pages + 1, 2, nkv, page, d), generator=g, dtype=torch.uint8)      # pages are never cleared
    exps = torch.randint(-128, 128, (2 * pages + 1, 2, nkv, page // 16), generator=g).to(torch.int8)
    cache = ops.Cache8(codes.cuda().view(torch.float8_e4m3fn), exps.cuda())
    want_c, want_e = codes.view(torch.float8_e4m3fn).clone(), exps.clone()
    at = 0
    for i, n in enumerate(steps):
        qkv = _random_qkv(2 * n, nh, nkv, d, 100 * d + i, dtype)
        pos = torch.arange(at, at + n)
        slots = torch.cat([order[r * pages + pos // page] * page + pos % page for r in (0, 1)]).to(torch.int32)
        before = qkv.cuda()
        q = ops.qk_norm_rope_write8(before, nh, nkv, d, None, None, 0.0, None, None, d, cache, slots.cuda())
        assert torch.equal(q.cpu(), qkv[:, :nh * d]) and torch.equal(before.cpu(), qkv)
        x = qkv.view(2 * n, nh + 2 * nkv, d)
        plain.write(want_c, want_e, x[:, nh:nh + nkv], x[:, nh + nkv:], slots)
        at += n
        assert torch.equal(cache.exps.cpu(), want_e), i
        _same(cache.codes, want_c, i)                        # (what no token was written to is as it was, too)
    for dt in (torch.bfloat16, torch.float32):
        ids = torch.randperm(2 * pages + 1, generator=g).to(torch.int32)
        got = ops.cache8_read(cache, ids.cuda(), dt)
        # (pages that nothing was written to may hold exponents that are not ones: only those that were)
        mine = torch.isin(ids, order[:2 * pages].to(torch.int32))
        used = torch.ones(2 * pages + 1, dtype=torch.bool)
        for r in (0, 1):
            for j in range(pages):
                if (j + 1) * page > at:
                    used[order[r * pages + j]] = False
        mine &= used[ids.long()]
        _same(got[mine.cuda()], plain.values(want_c, want_e)[ids.long()][mine].to(dt))


@gpu
@pytest.mark.parametrize("d,rot", [(64, 64), (128, 64), (48, 48), (16, 8)])
def test_norm_and_rotation_before_the_write(d, rot):
    """q within its rounding of the formula; k within its two: to bfloat16 and to the code (half a step each: 2^-8 of the value, 2^-4
    of it or half the smallest step of the block), and float32's few steps in norm and rotation on the larger partner."""
    ops = _ops()
    n, nh, nkv, page = 37, 3, 2, 64
    g = torch.Generator().manual_seed(d)
    qkv = torch.randn(n, (nh + 2 * nkv) * d, generator=g).bfloat16()
    qw, kw = 1 + 0.3 * torch.randn(d, generator=g), 1 + 0.3 * torch.randn(d, generator=g)
    ang = torch.rand(n, rot // 2, generator=g) * 6
    cos, sin = ang.cos(), ang.sin()
    cache = ops.cache8_empty(1, nkv, page, d)
    q = ops.qk_norm_rope_write8(qkv.cuda(), nh, nkv, d, qw.cuda(), kw.cuda(), 1e-5, cos.cuda(), sin.cuda(), rot, cache,
                                torch.arange(n, dtype=torch.int32).cuda())
    x = qkv.double().view(n, nh + 2 * nkv, d)

    def formula(y, w):
        y = y / (y.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * w.double()
        a, b, rest = y[..., :rot // 2], y[..., rot // 2:rot], y[..., rot:]
        c, s = cos.double()[:, None], sin.double()[:, None]
        size = torch.cat([a.abs() + b.abs(), a.abs() + b.abs(), rest.abs()], -1)
        return torch.cat([a * c - b * s, b * c + a * s, rest], -1), size
    want, size = formula(x[:, :nh], qw)
    assert ((q.cpu().double().view(n, nh, d) - want).abs() <= 2.0 ** -8 * want.abs() + (d + 16) * 2.0 ** -24 * size).all()
    want, size = formula(x[:, nh:nh + nkv], kw)
    got = plain.values(cache.codes.cpu(), cache.exps.cpu())[0, :, :, :n].transpose(1, 2)
    step = torch.exp2(cache.exps.cpu().double()).repeat_interleave(16, -1)[0, :, :, :n].transpose(1, 2)[..., None] * 2.0 ** -9
    near = (1 + 2.0 ** -4) * (1 + 2.0 ** -8) - 1
    assert ((got[0] - want).abs() <= torch.maximum(near * want.abs(), 2.0 ** -8 * want.abs() + step[0] / 2) + (d + 16) * 2.0 ** -23 * size).all()
    v = x[:, nh + nkv:]
    assert ((got[1] - v).abs() <= torch.maximum(2.0 ** -4 * v.abs(), step[1] / 2)).all()


@gpu
def test_what_is_not_finite_stays_seen_and_extremes_saturate():
    ops = _ops()
    d, page = 64, 16
    big = torch.finfo(torch.bfloat16).max
    x = torch.zeros(4, 3, d)
    x[0, 1, :5] = torch.tensor([math.inf, -math.inf, math.nan, 2.0, -3.0])
    x[1, 1, :3] = torch.tensor([big, -big, 1.0])
    x[2, 2, :4] = torch.tensor([1e-38, -2.0 ** -120, 2.0 ** -118, 0.0])
    x[3, 2, 0] = math.nan
    qkv = x.view(4, -1).bfloat16()
    cache = ops.cache8_empty(1, 1, page, d)
    ops.qk_norm_rope_write8(qkv.cuda(), 1, 1, d, None, None, 0.0, None, None, d, cache, torch.arange(4, dtype=torch.int32).cuda())
    c, e = torch.zeros(1, 2, 1, page, d).to(torch.float8_e4m3fn), torch.zeros(1, 2, 1, 1, dtype=torch.int8)
    y = qkv.view(4, 3, d)
    plain.write(c, e, y[:, 1:2], y[:, 2:3], torch.arange(4))
    assert torch.equal(cache.exps.cpu(), e) and int(e[0, 0]) == 119 and int(e[0, 1]) == -110
    _same(cache.codes[:, :, :, :4], c[:, :, :, :4])
    assert torch.isnan(cache.codes[0, 0, 0, 0, :3].float()).all() and float(cache.codes[0, 0, 0, 1, 0].float()) == 448.0


@gpu
def test_bad_slots_are_refused_and_the_rest_written():
    ops = _ops()
    d, page = 64, 16
    qkv = _random_qkv(4, 1, 1, d, 5, torch.bfloat16)
    cache = ops.Cache8(torch.zeros(2, 2, 1, page, d, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn),
                       torch.zeros(2, 2, 1, 1, dtype=torch.int8, device="cuda"))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    slots = torch.tensor([-1, 32, 2 ** 31 - 1, 17], dtype=torch.int32)
    ops.qk_norm_rope_write8(qkv.cuda(), 1, 1, d, None, None, 0.0, None, None, d, cache, slots.cuda(), status)
    assert int(status) == 2
    c, e = torch.zeros(2, 2, 1, page, d).to(torch.float8_e4m3fn), torch.zeros(2, 2, 1, 1, dtype=torch.int8)
    x = qkv.view(4, 3, d)
    plain.write(c, e, x[:, 1:2], x[:, 2:3], slots)
    _same(cache.codes, c)
    status.zero_()
    got = ops.cache8_read(cache, torch.tensor([1, -1, 2], dtype=torch.int32).cuda(), torch.float32, status)
    assert int(status) == 4 and not got[1:].any()
    _same(got[:1], plain.values(c, e)[1:].float())
    assert ops.cache8_read(cache, torch.zeros(0, dtype=torch.int32, device="cuda"), torch.float32).shape[0] == 0
    assert _write({**_step(0), "cache": ops.cache8_empty(2, 2, 32, 64), "qkv": torch.zeros(0, 512, dtype=torch.bfloat16, device="cuda"),
                   "slots": torch.zeros(0, dtype=torch.int32, device="cuda")}).shape == (0, 256)


# ---- attention ----------------------------------------------------------------------------------------

def _attention_case(lens, news, nh, nkv, d, page, dtype, seed, extra_columns=0):
    """Random pages in a random order; what lies behind a request's end, and in pages of nobody, is NaN."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-k // page) for k in lens]
    pages = sum(need) + 1
    order = torch.randperm(pages, generator=g)
    x = torch.randn(pages, 2, nkv, page // 16, 16, d, generator=g) * torch.exp(2 * torch.randn(pages, 2, nkv, page // 16, 1, 1, generator=g))
    exps = torch.tensor([plain.exponent(float(a)) for a in x.abs().amax((-1, -2)).reshape(-1)]).view(pages, 2, nkv, page // 16)
    codes = (x.double() * torch.exp2(-exps.double())[..., None, None]).to(torch.float8_e4m3fn).view(pages, 2, nkv, page, d)
    # keys small enough for scores that matter
    exps[:, 0] = torch.randint(-9, -7, exps[:, 0].shape, generator=g)
    exps = exps.to(torch.int8)
    table = torch.full((len(lens), max(need + [1])), pages - 1, dtype=torch.int32)
    at = 0
    raw = codes.view(torch.uint8)
    raw[order[pages - 1]] = 0x7f
    for s, k in enumerate(need):
        table[s, :k] = order[at:at + k].int()
        table[s, k:] = int(order[pages - 1])
        at += k
        if lens[s] % page:
            raw[table[s, k - 1].long(), :, :, lens[s] % page:] = 0xff
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1], nh * d + extra_columns, generator=g).to(dtype)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)
    return dict(q=q, codes=codes, exps=exps, table=table, cu=i32(cu), kl=i32(lens), n=cu[-1], S=len(lens), max_q=max(news), max_k=max(lens), nh=nh, nkv=nkv, d=d)


def _run_attention(c, scale, window=0, splits=None, impl="auto", status=None):
    ops = _ops()
    q = c["q"].cuda()
    return ops.paged_attention8(q, q.stride(0), ops.Cache8(c["codes"].cuda(), c["exps"].cuda()), c["table"].cuda(), c["cu"].cuda(), c["kl"].cuda(),
                                c["n"], c["S"], c["max_q"], c["max_k"], c["nh"], c["nkv"], c["d"], scale, window, splits, status, impl)


def _check_attention(c, got, scale, window=0, tensor_cores=True):
    """Rounding of the output (half a step); each weight's: to f16 on the tensor cores (2^-11, once in the sum and once where it is divided by
    the sum of unrounded weights), 2^-22 of the base-2 exponential, and the error of its score, which is a float32 sum of d products
    (a tensor core adds 16 at a time and cuts off instead of rounding: 2^-22 a step)."""
    want, spread, most = plain.attention(c["q"][:, :c["nh"] * c["d"]], plain.values(c["codes"], c["exps"]), c["table"], c["cu"], c["kl"], c["nh"], c["nkv"], c["d"],
                                         scale, window)
    eps = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}[c["q"].dtype]
    score = most * ((c["d"] / 16 + 6) * 2.0 ** -22 if tensor_cores else (c["d"] + 6) * 2.0 ** -24)
    weight = 2 * (score + 2.0 ** -20) + (2.0 ** -10 if tensor_cores else 0.0)
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    over = (got - want).abs() - (eps * want.abs() + (1 + eps) * weight * spread)
    assert (over <= 0).all(), (float(over.max()), most)


LENGTHS = [([1], [1]), ([16, 17, 15], [1, 1, 1]), ([63, 64, 65, 1], [1, 1, 1, 1]), ([300, 5, 129], [1, 3, 2]), ([700], [1]), ([40, 33], [17, 33]),
           ([200, 90, 1], [70, 0, 1])]              # (forced onto the mma.sync kernel, portions too)


@gpu
@pytest.mark.parametrize("lens,news", LENGTHS)
@pytest.mark.parametrize("nh,nkv,d,page", [(8, 2, 64, 64), (4, 4, 64, 16), (6, 2, 128, 64), (32, 2, 64, 32), (4, 1, 128, 48)])
@pytest.mark.parametrize("window", [0, 1, 37])
def test_attention_on_the_tensor_cores(lens, news, nh, nkv, d, page, window):
    c = _attention_case(lens, news, nh, nkv, d, page, torch.bfloat16, 7 * d + len(lens) + page)
    _check_attention(c, _run_attention(c, d ** -0.5, window, impl="tensor_core"), d ** -0.5, window)


def _portion_check(c, got, scale, window):
    """The tcgen05 kernel's P is bfloat16 (half a step 2^-8, once in the product and once against the sum of unrounded weights: twice)
    and its values code * 2^e are exact; the rest as for the mma.sync kernel."""
    want, spread, most = plain.attention(c["q"][:, :c["nh"] * c["d"]], plain.values(c["codes"], c["exps"]), c["table"], c["cu"], c["kl"], c["nh"], c["nkv"], c["d"],
                                         scale, window)
    weight = 2 * (most * (c["d"] / 16 + 6) * 2.0 ** -22 + 2.0 ** -20) + 2.0 ** -7
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    over = (got - want).abs() - (2.0 ** -8 * want.abs() + (1 + 2.0 ** -8) * weight * spread)
    assert (over <= 0).all(), float(over.max())
    # (and on average far nearer: rounding errors of both signs; a value left out or taken twice would not be)
    assert (got - want).norm() <= 2.0 ** -7 * want.norm()


PORTIONS = [([1], [1]), ([64], [64]), ([65], [65]), ([300], [129]), ([40, 33, 100], [17, 33, 1]), ([1000, 90, 700], [70, 0, 512]), ([190], [2])]


@gpu
@pytest.mark.parametrize("lens,news", PORTIONS)
@pytest.mark.parametrize("nh,nkv,d,page", [(8, 2, 64, 64), (4, 4, 64, 16), (6, 2, 128, 64), (32, 2, 64, 48), (4, 1, 128, 16), (3, 1, 64, 128)])
@pytest.mark.parametrize("window", [0, 1, 37])
def test_portions_on_tcgen05(lens, news, nh, nkv, d, page, window):
    c = _attention_case(lens, news, nh, nkv, d, page, torch.bfloat16, 11 * d + len(lens) + page)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    _portion_check(c, _run_attention(c, d ** -0.5, window, impl="tcgen05", status=status), d ** -0.5, window)
    _portion_check(c, _run_attention(c, d ** -0.5, window, status=status), d ** -0.5, window)
    assert int(status) == 0


@gpu
@pytest.mark.parametrize("d,window", [(64, 0), (64, 100), (128, 0)])
def test_long_portions_beside_single_tokens(d, window):
    """Portions long enough for the tcgen05 kernel in one step with shorter ones and single tokens, which go to the mma.sync kernel."""
    c = _attention_case([1700, 60, 900, 33, 1], [1650, 1, 31, 32, 1], 16, 4, d, 64, torch.bfloat16, d)
    ops = _ops()
    before = ops.launch_count
    got = _run_attention(c, d ** -0.5, window)
    assert ops.launch_count == before + 2
    _portion_check(c, got, d ** -0.5, window)


@gpu
@pytest.mark.parametrize("splits", [1, 2, 3, 4, 8, 16])
@pytest.mark.parametrize("nh,nkv,d,window", [(8, 2, 64, 0), (6, 2, 128, 0), (3, 1, 64, 150), (8, 1, 128, 70)])
def test_portions_split_over_a_cluster(splits, nh, nkv, d, window):
    """Blocks of a cluster with several tiles of keys, with one and with none (30 keys are one tile), rows behind a sequence's last, and
    tokens before a sequence's first key, which see nothing."""
    c = _attention_case([1500, 30, 130], [45, 30, 130], nh, nkv, d, 64, torch.bfloat16, 3 * splits + d)
    first = _run_attention(c, d ** -0.5, window, splits=splits, impl="tcgen05")
    _portion_check(c, first, d ** -0.5, window)
    assert torch.equal(first, _run_attention(c, d ** -0.5, window, splits=splits, impl="tcgen05"))
    c["kl"] = torch.tensor([1500, 12, 0], dtype=torch.int32)
    blind = _run_attention(c, d ** -0.5, window, splits=splits, impl="tcgen05")
    assert torch.equal(blind[:45], first[:45])
    assert not blind[45:45 + 18].any() and not blind[75:].any()
    assert torch.isfinite(blind).all() and blind[63:75].any()


@gpu
@pytest.mark.parametrize("splits", [1, 2, 4, 8, 16])
@pytest.mark.parametrize("rows", [1, 3])
def test_attention_split_over_a_cluster(splits, rows):
    """(fewer blocks of keys than warps, and more than 32 a warp, where the look-up is made again)"""
    for lens in ([5, 130], [9000, 77]):
        c = _attention_case(lens, [rows, rows], 8, 2, 64, 64, torch.bfloat16, splits)
        first = _run_attention(c, 0.125, splits=splits)
        _check_attention(c, first, 0.125)
        assert torch.equal(first, _run_attention(c, 0.125, splits=splits))
        big = _attention_case(lens, [rows, rows], 6, 2, 128, 64, torch.bfloat16, splits)
        _check_attention(big, _run_attention(big, 0.125, splits=splits), 0.125)


@gpu
@pytest.mark.parametrize("d,nh,nkv", [(64, 16, 8), (128, 8, 4)])
@pytest.mark.parametrize("rows,window", [(1, 0), (1, 40), (5, 0)])
def test_many_requests_of_few_keys(d, nh, nkv, rows, window):
    """More blocks than the device holds at once, which then have four warps; requests of one key and of none among them."""
    S = 100
    lens = [1 + (37 * i) % 300 for i in range(S)]
    lens[3] = 1000
    news = [min(rows, k) if i % 5 else 1 for i, k in enumerate(lens)]
    c = _attention_case(lens, news, nh, nkv, d, 16, torch.bfloat16, rows + d)
    c["kl"][7] = 0
    got = _run_attention(c, d ** -0.5, window)
    _check_attention(c, got, d ** -0.5, window)
    assert torch.equal(got, _run_attention(c, d ** -0.5, window))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nh,nkv,d,page", [(4, 2, 64, 64), (3, 1, 16, 16), (2, 2, 128, 32), (6, 3, 48, 48), (2, 1, 256, 16)])
@pytest.mark.parametrize("window", [0, 20])
def test_attention_on_the_general_kernel(nh, nkv, d, page, dtype, window):
    for lens, news in LENGTHS[1:]:
        c = _attention_case(lens, news, nh, nkv, d, page, dtype, d + len(lens))
        _check_attention(c, _run_attention(c, d ** -0.5, window, impl="general"), d ** -0.5, window, tensor_cores=False)


@gpu
@pytest.mark.parametrize("splits", [None, 1, 3, 8, 16])
@pytest.mark.parametrize("nh,nkv,d,dtype,rows", [(4, 1, 80, torch.float32, 1), (2, 2, 64, torch.float32, 7), (8, 1, 256, torch.bfloat16, 3)])
def test_the_general_kernel_over_a_cluster(splits, nh, nkv, d, dtype, rows):
    """Blocks with several tiles of keys, one and none; tokens before the first key beside others of their tile."""
    c = _attention_case([2500, 9, 40], [rows, rows, rows], nh, nkv, d, 16, dtype, d + rows)
    got = _run_attention(c, d ** -0.5, splits=splits, impl="general")
    _check_attention(c, got, d ** -0.5, tensor_cores=False)
    assert torch.equal(got, _run_attention(c, d ** -0.5, splits=splits, impl="general"))
    c["kl"] = torch.tensor([2500, 0, rows - 1], dtype=torch.int32)
    blind = _run_attention(c, d ** -0.5, splits=splits, impl="general")
    assert torch.equal(blind[:rows], got[:rows]) and not blind[rows:2 * rows + 1].any() and torch.isfinite(blind).all()


@gpu
def test_queries_at_any_stride_and_place():
    for extra, tensor_cores in ((64, True), (8, True), (4, False), (1, False)):
        c = _attention_case([70, 30], [2, 30], 4, 2, 64, 64, torch.bfloat16, extra, extra)
        _check_attention(c, _run_attention(c, 0.125), 0.125, tensor_cores=tensor_cores)
    c = _attention_case([70, 30], [2, 30], 4, 2, 64, 64, torch.bfloat16, 3)
    whole = torch.randn(33, 256).bfloat16().cuda().view(-1)
    whole[3:3 + 32 * 256] = c["q"].cuda().view(-1)
    ops = _ops()
    q = whole[3:3 + 32 * 256].view(32, 256)
    got = ops.paged_attention8(q, 256, ops.Cache8(c["codes"].cuda(), c["exps"].cuda()), c["table"].cuda(), c["cu"].cuda(), c["kl"].cuda(), 32, 2, 30, 70, 4, 2, 64, 0.125)
    _check_attention(c, got, 0.125)


@gpu
def test_a_query_without_keys_gets_zeros_and_a_bad_page_a_status():
    for d, impl in ((64, "auto"), (64, "general"), (64, "tcgen05"), (128, "tcgen05")):
        c = _attention_case([40, 16, 20], [1, 1, 2], 4, 2, d, 16, torch.bfloat16, 1)
        c["kl"] = torch.tensor([40, 0, 1], dtype=torch.int32)           # the third request's first query lies before position 0
        got = _run_attention(c, 0.125, impl=impl)
        assert not got[1].any() and not got[2].any()
        if impl == "tcgen05":
            _portion_check(c, got, 0.125, 0)
        else:
            _check_attention(c, got, 0.125, tensor_cores=impl == "auto")
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        c["table"][0, 1] = 10 ** 6
        _run_attention(c, 0.125, impl=impl, status=status)
        assert int(status) == 4
    with pytest.raises(_ops().KernelError, match="tensor-core"):
        _run_attention(_attention_case([5], [1], 2, 1, 48, 16, torch.bfloat16, 1), 0.1, impl="tensor_core")
    with pytest.raises(_ops().KernelError, match="splits"):
        _run_attention(_attention_case([5], [1], 2, 1, 64, 16, torch.bfloat16, 1), 0.1, splits=17)


@gpu
@pytest.mark.parametrize("d,impl", [(64, "tensor_core"), (128, "tensor_core"), (64, "tcgen05"), (128, "tcgen05"), (64, "general"), (48, "auto")])
@pytest.mark.parametrize("lens,news", [([200, 333], [1, 1]), ([500, 99], [150, 40])])
def test_what_a_window_has_left_behind_is_not_looked_up(d, impl, lens, news):
    """Pages before every row's window are no pages any more, and what no row sees in the first that is one, or behind the last, is NaN."""
    window, dtype = 21, torch.bfloat16
    c = _attention_case(lens, news, 4, 2, d, 16, dtype, d + len(impl))
    raw = c["codes"].view(torch.uint8)
    for s, (k, n) in enumerate(zip(lens, news)):
        least = k - n - window + 1                       # the first key that a row sees
        c["table"][s, :least // 16] = -1
        raw[c["table"][s, least // 16].long(), :, :, :least % 16] = 0x7f
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for splits in (1, 4):
        got = _run_attention(c, d ** -0.5, window, splits=splits, impl=impl, status=status)
        assert int(status) == 0
        _portion_check(_seen_only(c), got, d ** -0.5, window)


def _seen_only(c):
    """The case with numbers where there is no page and where nothing is seen (the plain form takes 0 * NaN)."""
    c = dict(c)
    raw = c["codes"].view(torch.uint8).clone()
    raw[(raw & 0x7f) == 0x7f] = 0
    c["codes"], c["table"] = raw.view(torch.float8_e4m3fn), c["table"].clamp(min=0)
    return c


@gpu
def test_pages_beyond_32_bits_of_offset():
    """A cache of 4.6 GB, of which the first and the last pages are written, read and attended to."""
    ops = _ops()
    nh, nkv, d, page, pages = 8, 2, 128, 64, 141_000
    cache = ops.cache8_empty(pages, nkv, page, d)
    assert cache.codes.numel() > 2 ** 32
    n = 3 * page
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(n, (nh + 2 * nkv) * d, generator=g).bfloat16().cuda()
    ids = torch.tensor([pages - 1, 0, pages - 2], dtype=torch.int32)
    slots = (ids[:, None].long() * page + torch.arange(page)).view(-1).int().cuda()
    q = ops.qk_norm_rope_write8(qkv, nh, nkv, d, None, None, 0.0, None, None, 0, cache, slots)
    back = ops.cache8_read(cache, ids.cuda(), torch.bfloat16)
    small = ops.cache8_empty(3, nkv, page, d)
    assert torch.equal(q, ops.qk_norm_rope_write8(qkv, nh, nkv, d, None, None, 0.0, None, None, 0, small, torch.arange(n, dtype=torch.int32, device="cuda")))
    assert torch.equal(back, ops.cache8_read(small, torch.arange(3, dtype=torch.int32, device="cuda"), torch.bfloat16))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    for impl in ("tensor_core", "tcgen05", "general"):
        a, b = (ops.paged_attention8(q, nh * d, where, table[None], i32(0, n), i32(n), n, 1, n, n, nh, nkv, d, d ** -0.5, impl=impl)
                for where, table in ((cache, ids.cuda()), (small, i32(0, 1, 2))))
        assert torch.equal(a, b), impl


@gpu
def test_queries_of_unlike_size_and_blocks_of_unlike_scale():
    """Rows of queries from 2^-60 to 2^60 (their scores scaled back), values from 2^-80 to 2^80 in neighbouring blocks: no row loses its own."""
    c = _attention_case([100], [1], 8, 2, 64, 16, torch.bfloat16, 9)
    power = torch.tensor([-60, -20, -3, 0, 0, 7, 25, 60])
    plain_q = c["q"].clone()
    c["q"] = (c["q"].view(8, 64).float() * torch.exp2(power.float())[:, None]).bfloat16().view(1, -1)
    c["exps"][:, 1] = torch.randint(-80, 80, c["exps"][:, 1].shape, generator=torch.Generator().manual_seed(3)).to(torch.int8)
    for h in range(8):
        # one head at a time, so that the scale takes its power off again
        scale = 0.125 * 2.0 ** -int(power[h])
        got = _run_attention(c, scale).double().cpu().view(8, 64)[h]
        want, spread, most = plain.attention(plain_q, plain.values(c["codes"], c["exps"]), c["table"], c["cu"], c["kl"], 8, 2, 64, 0.125)
        weight = 2 * (most * 10 * 2.0 ** -22 + 2.0 ** -20) + 2.0 ** -10
        w, sp = want.view(8, 64)[h], spread.view(8, 64)[h]
        assert ((got - w).abs() <= 2.0 ** -8 * w.abs() + 1.01 * weight * sp).all(), h


@gpu
def test_captured_and_on_another_stream():
    c = _attention_case([900, 33, 64], [1, 1, 1], 8, 2, 64, 64, torch.bfloat16, 2)
    ops = _ops()
    q, cache = c["q"].cuda(), ops.Cache8(c["codes"].cuda(), c["exps"].cuda())
    table, cu, kl = c["table"].cuda(), c["cu"].cuda(), c["kl"].cuda()
    call = lambda: ops.paged_attention8(q, q.stride(0), cache, table, cu, kl, 3, 3, 1, 900, 8, 2, 64, 0.125)
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(call(), want)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    kl.copy_(torch.tensor([700, 20, 64], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    c["kl"] = kl.cpu()
    _check_attention(c, got, 0.125)
