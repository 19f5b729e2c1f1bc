"""Operators of serving in fewer bits straight behind the kernels whose results they read: launched without a pause, and captured."""
import pytest
import torch

from test_int4 import _check, _random, _to_device

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture
def ops():
    from vapi_b200 import ops
    return ops


def _played(body):
    """The body's results run eagerly, and those of its third replay as a graph."""
    body()
    torch.cuda.synchronize()
    yield [t.clone() for t in body()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = body()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    yield out


# ---- a weight that is written out ----------------------------------------------------------------------

@pytest.mark.parametrize("n,k,group", [(2048, 2048, 64), (8192, 2048, 128), (2048, 8192, 32)])
@pytest.mark.parametrize("rows", [1, 8, 16, 40])
@pytest.mark.parametrize("gated", [False, True])
def test_a_weight_written_out_is_read_when_it_is_there(ops, n, k, group, rows, gated):
    """float32 rows take a 4-bit weight as numbers in memory, which are another weight's or NaN until they have been written."""
    hosts = [ops.int4_pack(*_random(n, k, group, s)) for s in (1, 2)]
    weights = [_to_device(w) for w in hosts]
    x = torch.randn(rows, k, generator=torch.Generator().manual_seed(rows))
    dev = x.cuda()

    def body():
        out = []
        for turn in range(2):
            for w in weights:
                torch.full((n * k,), float("nan"), device="cuda")           # (its memory goes back at once)
                out.append(ops.int4_linear_swiglu(dev, w) if gated else ops.int4_linear(dev, w))
        return out
    for got in _played(body):
        for i in (0, 1):
            _check(x, hosts[i], got[i], act="silu" if gated else None)
            assert torch.equal(got[i], got[2 + i])


@pytest.mark.parametrize("rows", [3, 24])
@pytest.mark.parametrize("gated", [False, True])
def test_the_same_in_bfloat16(ops, monkeypatch, rows, gated):
    """What rows do where the products of few rows are switched off (VAPI_INT4_MAX_ROWS)."""
    monkeypatch.setattr(ops.int4, "INT4_MAX_ROWS", 0)
    n, k, group = 8192, 2048, 64
    hosts = [ops.int4_pack(*_random(n, k, group, s)) for s in (1, 2)]
    weights = [_to_device(w) for w in hosts]
    x = torch.randn(rows, k, generator=torch.Generator().manual_seed(rows)).bfloat16()
    dev = x.cuda()

    def body():
        out = []
        for w in weights:
            torch.full((n * k // 2,), float("nan"), device="cuda")
            out.append(ops.int4_linear_swiglu(dev, w) if gated else ops.int4_linear(dev, w))
        return out
    for got in _played(body):
        for w, y in zip(hosts, got):
            _check(x, w, y, rounded=True, act="silu" if gated else None)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows", [2, 20, 40])
def test_a_product_with_a_weight_of_int4_dequantize(ops, dtype, rows):
    """The public pieces, with a kernel between them too."""
    n, k, group = 8192, 2048, 64
    hosts = [ops.int4_pack(*_random(n, k, group, s)) for s in (1, 2)]
    weights = [_to_device(w) for w in hosts]
    x = torch.randn(rows, k, generator=torch.Generator().manual_seed(rows)).to(dtype)
    dev = x.cuda()

    def body():
        out = []
        for w in weights:
            for between in (False, True):
                torch.full((n * k * dev.element_size() // 4,), float("nan"), device="cuda")
                numbers = ops.int4_dequantize(w, dtype)
                if between:
                    ops.swiglu(dev)
                out.append(ops.linear(dev, numbers))
        return out
    for got in _played(body):
        for i, y in enumerate(got):
            _check(x, hosts[i // 2], y, rounded=dtype == BF)
