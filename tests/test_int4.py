"""Products with 4-bit weights (csrc/int4.cu)."""
import pytest
import torch

import plain_fewer_bits as plain

gpu = pytest.mark.gpu


def _ops():
    from vapi_b200 import ops
    return ops


def _random(n, k, group, seed):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    zeros = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8)
    scales = (torch.exp(torch.randn(n, k // group, generator=g)) * 0.05).bfloat16()
    return codes, scales, zeros


def test_a_packed_weight_holds_what_went_in():
    ops = _ops()
    for n, k, group in ((1, 32, 32), (16, 64, 64), (17, 96, 32), (40, 384, 128), (2000, 128, 64)):
        codes, scales, zeros = _random(n, k, group, n)
        w = ops.int4_pack(codes, scales, zeros)
        assert w.shape == (n, k) and w.group == group
        for a, b in zip(plain.unpack(w), (codes, scales, zeros.bfloat16())):
            assert torch.equal(a, b)
        assert torch.equal(plain.unpack(ops.int4_pack(codes, scales))[2], torch.full_like(scales, 8))


def test_quantising_is_off_by_half_a_step_at_most():
    """scale = (hi - lo) / 15 rounded by at most 2^-8 of it, so codes reach to within 15 * 2^-8 steps of either end; the zero is
    rounded by half a step, which shifts the ends and so can cut off half a step more there."""
    ops = _ops()
    g = torch.Generator().manual_seed(1)
    for group in (32, 64, 128):
        w = torch.randn(50, 256, generator=g) * torch.exp(torch.randn(50, 1, generator=g))
        w[3], w[4], w[5] = 0, w[4].abs() + 5, -w[5].abs()
        q = ops.int4_quantize(w, group)
        scale = plain.unpack(q)[1].double().repeat_interleave(group, 1)
        assert ((plain.int4_numbers(q) - w.double()).abs() <= (1.0 + 15 * 2.0 ** -8) * scale).all()
        assert not plain.int4_numbers(q)[3].any()
        inside = (w.double() / scale + plain.unpack(q)[2].double().repeat_interleave(group, 1))
        inside = (inside >= 0) & (inside <= 15)
        assert ((plain.int4_numbers(q) - w.double()).abs() <= (0.5 + 1e-4) * scale)[inside].all()


def test_what_does_not_fit_is_refused():
    ops = _ops()
    codes, scales, zeros = _random(16, 128, 64, 1)
    for args, words in (((codes.int(), scales), "uint8"), ((codes, scales.float()), "bfloat16"), ((codes, scales[:8]), "scales"),
                        ((codes, scales[:, :1].expand(16, 8).contiguous()), "groups of 16"), ((codes, scales, zeros.int()), "zeros"),
                        ((codes, scales, zeros[:, :1]), "zeros"), ((codes + 8, scales, zeros), "0..15"), ((codes, scales, zeros + 8), "0..15"),
                        ((codes[:, :0], scales), "codes")):
        with pytest.raises(ops.KernelError, match=words):
            ops.int4_pack(*args)
    for args, words in (((torch.zeros(4, 100),), "groups of 64"), ((torch.zeros(4, 128), 16), "groups of 16"), ((torch.zeros(4, 128, dtype=torch.int32),), "floating"),
                        ((torch.full((4, 128), float("nan")),), "finite")):
        with pytest.raises(ops.KernelError, match=words):
            ops.int4_quantize(*args)
    w = ops.int4_pack(codes, scales, zeros)
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    for call, words in ((lambda: ops.int4_linear(x, codes), "Int4Weight"), (lambda: ops.int4_linear(x[:, :64], w), "does not fit"), (lambda: ops.int4_linear(x.half(), w), "does not fit"),
                        (lambda: ops.int4_linear(x, w), "CUDA"), (lambda: ops.linear(x, w), "CUDA"), (lambda: ops.linear_swiglu(x, w), "CUDA"),
                        (lambda: ops.int4_dequantize(w, torch.float16), "dtype")):
        with pytest.raises(ops.KernelError, match=words):
            call()
    assert not ops.few_rows_applies(1, w)


def test_a_weight_of_another_layout_is_refused():
    ops = _ops()
    for group in (32, 64):
        w = ops.int4_pack(*_random(24, 192, group, 2))
        same = ops.Int4Weight(w.codes, w.scales, 24, 192, group)
        assert same.shape == (24, 192)
        for args, words in (((w.codes, w.scales, 40, 192, group), "codes"), ((w.codes, w.scales, 24, 256, group), "codes"), ((w.codes, w.scales, 24, 192, 48), "groups of 48"),
                            ((w.codes, w.scales[:, :1], 24, 192, group), "scales"), ((w.codes.float(), w.scales, 24, 192, group), "int32"), ((w.codes, w.scales, 0, 192, group), "0 x 192"),
                            ((w.codes[:, ::2], w.scales, 24, 128, group), "codes")):
            with pytest.raises(ops.KernelError, match=words):
                ops.Int4Weight(*args)


def _to_device(w):
    return _ops().Int4Weight(w.codes.cuda(), w.scales.cuda(), w.n, w.k, w.group)


def _check(x, w, got, bias=None, rounded=False, act=None):
    """Half a step of the result; the float32 sums of k products, which tensor cores cut off instead of rounding (2^-23 of the sum of
    magnitudes a step of 16, and one a group and a few for the warps); with ``rounded`` a weight's half step of bfloat16 too."""
    numbers = plain.int4_numbers(w)
    y, size = x.double() @ numbers.t(), x.double().abs() @ numbers.abs().t()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    # (the codes less their zero, up to 15, enter the sums before the scale: the same relative size)
    err = size * ((w.k / 16 + w.k / w.group + 20) * 2.0 ** -23 + (2.0 ** -8 if rounded else 0.0))
    if act:
        half = w.n // 2
        gate, up, eg, eu = y[:, :half], y[:, half:], err[:, :half], err[:, half:]
        if rounded:                      # (the unfused form stores gate and up as bfloat16)
            eg, eu = eg + 2.0 ** -8 * gate.abs(), eu + 2.0 ** -8 * up.abs()
        f = (lambda z: z * torch.sigmoid(z)) if act == "silu" else (lambda z: z * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3)))
        y = f(gate) * up
        # (the slope of either gate is below 1.2; exponential and division of the fast kind: 2^-20 of the result)
        err = 1.2 * eg * (up.abs() + eu) + f(gate).abs() * eu + 2.0 ** -20 * y.abs()
    eps = 2.0 ** -24 if got.dtype == torch.float32 else 2.0 ** -8
    over = (got.double().cpu() - y).abs() - (eps * y.abs() + (1 + eps) * err + 1e-38)
    assert torch.isfinite(got).all() and (over <= 0).all(), float(over.max())


SIZES = [(16, 32, 32), (1, 64, 64), (48, 128, 128), (33, 96, 32), (200, 512, 64), (96, 1152, 128), (1000, 160, 32), (10016, 256, 64), (64, 8192, 128)]


@gpu
@pytest.mark.parametrize("n,k,group", SIZES)
def test_packing_on_the_device_is_the_hosts(n, k, group):
    ops = _ops()
    codes, scales, zeros = _random(n, k, group, 3)
    for z in (zeros, None):
        a, b = ops.int4_pack(codes, scales, z), ops.int4_pack(codes.cuda(), scales.cuda(), None if z is None else z.cuda())
        assert torch.equal(a.codes, b.codes.cpu()) and torch.equal(a.scales, b.scales.cpu())
    wide = torch.zeros(n, k + 3, dtype=torch.uint8)
    wide[:, 3:] = codes
    b = ops.int4_pack(wide.cuda()[:, 3:], scales.cuda(), zeros.cuda())
    assert torch.equal(ops.int4_pack(codes, scales, zeros).codes, b.codes.cpu())
    for which in (0, 1):
        bad = [codes.clone(), zeros.clone()]
        bad[which][-1, -1] = 16
        with pytest.raises(ops.KernelError, match="0..15"):
            ops.int4_pack(bad[0].cuda(), scales.cuda(), bad[1].cuda())



@gpu
@pytest.mark.parametrize("n,k,group", SIZES)
@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 16, 17, 24, 25, 32, 33, 64])
def test_few_rows(n, k, group, rows):
    ops = _ops()
    w = ops.int4_pack(*_random(n, k, group, n + k))
    d = _to_device(w)
    g = torch.Generator().manual_seed(rows)
    x = (torch.randn(rows, k, generator=g) * torch.exp(torch.randn(1, k, generator=g))).bfloat16()
    bias = torch.randn(n, generator=g)
    # (above 16 rows a weight's number is rounded to bfloat16: half a step, at most 2^-8 of the number, so of the sum of magnitudes)
    rounded = rows > 16
    got = ops.int4_linear(x.cuda(), d)
    assert got.dtype == torch.bfloat16
    _check(x, w, got, rounded=rounded)
    assert torch.equal(ops.linear(x.cuda(), d), got)
    _check(x, w, ops.int4_linear(x.cuda(), d, bias.cuda()), bias, rounded=rounded)
    _check(x, w, ops.int4_linear(x.cuda(), d, bias.cuda(), torch.float32), bias, rounded=rounded)
    if n % 2 == 0:
        for act in ("silu", "gelu_tanh"):
            _check(x, w, ops.linear_swiglu(x.cuda(), d, act), act=act, rounded=rounded or n % 32 != 0)


@gpu
@pytest.mark.parametrize("n,k,group", [(2048, 8192, 128), (16416, 1024, 64), (8200, 2080, 32)])
@pytest.mark.parametrize("rows", [30, 100, 129, 300, 512])
def test_rows_enough_for_a_tile(n, k, group, rows):
    """Weights large enough for the tcgen05 kernel at any of these rows; all the same a second time, and in a graph."""
    ops = _ops()
    w = ops.int4_pack(*_random(n, k, group, n + rows))
    d = _to_device(w)
    g = torch.Generator().manual_seed(rows)
    x = (torch.randn(rows, k, generator=g) * torch.exp(torch.randn(1, k, generator=g))).bfloat16()
    bias, dev = torch.randn(n, generator=g), x.cuda()
    db = bias.cuda()
    before = ops.launch_count
    got = ops.int4_linear(dev, d, db)
    assert ops.launch_count == before + 1
    _check(x, w, got, bias, rounded=True)
    wide = ops.int4_linear(dev, d, db, torch.float32)
    assert torch.equal(wide.bfloat16(), got) and torch.equal(ops.int4_linear(dev, d, db), got)
    if n % 32 == 0:
        _check(x, w, ops.int4_linear_swiglu(dev, d), rounded=True, act="silu")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = ops.int4_linear(dev, d, db)
    dev.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, bias.bfloat16().cuda().expand(rows, n))
    dev.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, got)


@gpu
@pytest.mark.parametrize("n,k,group", SIZES)
def test_more_rows_and_float32(n, k, group):
    ops = _ops()
    w = ops.int4_pack(*_random(n, k, group, n + k))
    d = _to_device(w)
    numbers = plain.int4_numbers(w)
    assert torch.equal(ops.int4_dequantize(d, torch.float32).cpu(), numbers.float()) and torch.equal(numbers.float().double(), numbers)
    assert torch.equal(ops.int4_dequantize(d, torch.bfloat16).cpu(), numbers.float().bfloat16())
    for rows in (65, 300):
        x = torch.randn(rows, k, generator=torch.Generator().manual_seed(rows)).bfloat16()
        _check(x, w, ops.int4_linear(x.cuda(), d), rounded=True)
        if n % 16 == 0:
            _check(x, w, ops.int4_linear_swiglu(x.cuda(), d), rounded=True, act="silu")
    for rows in (1, 40):
        x = torch.randn(rows, k, generator=torch.Generator().manual_seed(rows))
        _check(x, w, ops.int4_linear(x.cuda(), d))


@gpu
def test_rows_in_other_places_and_nothing():
    ops = _ops()
    w = ops.int4_pack(*_random(64, 128, 64, 5))
    d = _to_device(w)
    wide = torch.randn(9, 300).bfloat16()
    for view in (wide[:, 3:131], wide[:, 8:136], wide.t().contiguous().t()[:, 100:228], wide[::2, :128]):
        _check(view, w, ops.int4_linear(view.cuda() if view.is_contiguous() else torch.empty_strided(view.shape, view.stride(), dtype=view.dtype, device="cuda").copy_(view), d))
    assert ops.int4_linear(torch.zeros(0, 128, dtype=torch.bfloat16, device="cuda"), d).shape == (0, 64)
    assert ops.int4_linear_swiglu(torch.zeros(0, 128, dtype=torch.bfloat16, device="cuda"), d).shape == (0, 32)
    x = torch.randn(3, 128).bfloat16()
    x[1, 5] = float("nan")
    got = ops.int4_linear(x.cuda(), d)
    assert torch.isnan(got[1]).all() and torch.isfinite(got[[0, 2]]).all()


@gpu
def test_captured_and_on_another_stream():
    ops = _ops()
    w = ops.int4_pack(*_random(2048, 2048, 64, 5))
    d = _to_device(w)
    x = torch.randn(4, 2048).bfloat16().cuda()
    want = ops.int4_linear(x, d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(ops.int4_linear(x, d), want)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.int4_linear(x, d)
    x.copy_(x.flip(1))
    graph.replay()
    torch.cuda.synchronize()
    _check(x.cpu(), w, got)
