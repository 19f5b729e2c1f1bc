"""Operators of serving in fewer bits straight behind the kernels whose results they read: launched without a pause, and captured."""
import sys
import threading

import pytest
import torch

from test_int4 import _check, _random, _to_device

pytestmark = pytest.mark.gpu
BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32


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

# ---- a cache that is written -------------------------------------------------------------------------

class Prompt:
    """A prompt's rows, its cache, and what is done with them: 32 / 8 heads.  (Rows that are not 16-byte aligned are the general write's, a warp of which
    takes 16 tokens one after the other: it ends late.)"""

    def __init__(self, ops, d, n):
        self.ops, self.d, self.n = ops, d, n
        g = torch.Generator().manual_seed(4)
        self.qkv = torch.randn(n * 48 * d + 1, generator=g).bfloat16().cuda()[1:].view(n, 48 * d)
        self.cache = ops.cache8_empty(-(-n // 64), 8, 64, d)
        self.slots = torch.arange(n, dtype=I32, device="cuda")
        self.table = torch.arange(-(-n // 64), dtype=I32, device="cuda")[None]
        self.lens = torch.tensor([n], dtype=I32, device="cuda")

    def clear(self):
        self.cache.codes.view(torch.uint8).fill_(0x7f)
        self.cache.exps.zero_()

    def write(self, a, b, rows=None):
        return self.ops.qk_norm_rope_write8(self.qkv[a:b] if rows is None else rows, 32, 8, self.d, None, None, 0.0, None, None, 0, self.cache, self.slots[a:b])

    def attend(self, q, ends, impl="auto"):
        rows = q.shape[0]
        return self.ops.paged_attention8(q, q.stride(0), self.cache, self.table, ends, self.lens, rows, 1, rows, self.n, 32, 8, self.d, self.d ** -0.5, impl=impl)


def _ends(rows):
    return torch.tensor([0, rows], dtype=I32, device="cuda")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows,impl", [(1, "auto"), (7, "tensor_core"), (200, "tcgen05"), (200, "auto"), (1, "general")])
def test_attention_of_the_last_tokens_of_what_was_just_written(ops, d, rows, impl):
    """One write of a whole prompt, and attention of its last tokens straight behind it."""
    n, ends = 6000, _ends(rows)
    p = Prompt(ops, d, n)
    q = p.write(0, n)[n - rows:]
    torch.cuda.synchronize()
    want = p.attend(q, ends, impl)
    assert torch.isfinite(want).all()

    def body():
        p.clear()
        return [p.attend(p.write(0, n)[n - rows:], ends, impl)]
    for turn in range(5):
        for got in _played(body):
            assert torch.equal(got[0], want)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [1, 1000])
def test_attention_behind_two_writes(ops, d, rows):
    """A prompt in two portions, both written before the second's attention; and a portion, a token, the token's attention."""
    n, ends = 7000, _ends(rows)
    p = Prompt(ops, d, n)
    p.write(0, n - rows)
    torch.cuda.synchronize()
    q = p.write(n - rows, n)
    torch.cuda.synchronize()
    want = p.attend(q, ends)
    assert torch.isfinite(want).all()

    def body():
        p.clear()
        p.write(0, n - rows)
        return [p.attend(p.write(n - rows, n), ends)]
    for turn in range(5):
        for got in _played(body):
            assert torch.equal(got[0], want)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows,impl", [(1, "auto"), (300, "tcgen05")])
def test_settled_steps_read_their_own_tokens_when_they_are_written(ops, d, rows, impl):
    """Within one_stream(settled=True), as in an engine's step: older keys ahead of the wait, the step's own behind its write."""
    n, ends = 7000, _ends(rows)
    p = Prompt(ops, d, n)
    p.write(0, n - rows)
    torch.cuda.synchronize()
    q = p.write(n - rows, n)
    torch.cuda.synchronize()
    want = p.attend(q, ends, impl)
    zeros = torch.zeros(rows, 48 * d, dtype=BF, device="cuda")
    for turn in range(5):
        p.write(n - rows, n, zeros)
        torch.cuda.synchronize()
        with ops.one_stream(settled=True):
            assert ops._held.settled
            p.write(n - rows, n)
            got = p.attend(q, ends, impl)
        assert torch.equal(got, want) and not ops._held.settled


@pytest.mark.parametrize("d,rows,impl", [(64, 1, "auto"), (128, 1, "tensor_core"), (64, 40, "tcgen05"), (64, 1, "general")])
def test_index_data_of_the_kernel_just_before(ops, d, rows, impl):
    """Lengths and pages that another library's kernels write right ahead of the call, other ones each time."""
    n, ends = 1536, _ends(rows)                              # (whole pages: in another order they hold numbers too)
    p = Prompt(ops, d, n)
    q = p.write(0, n)[n - rows:]
    lengths = [torch.tensor([k], dtype=I32, device="cuda") for k in (n, 700, 64, n - 1)]
    tables = [p.table.clone(), p.table.flip(1).contiguous()]
    torch.cuda.synchronize()

    def body(between=lambda: None):
        out = []
        for table in tables:
            for length in lengths:
                torch.add(table, 0, out=p.table)
                torch.mul(length, 1, out=p.lens)
                between()
                out.append(p.attend(q, ends, impl))
        return out
    want = body(torch.cuda.synchronize)
    assert all(torch.isfinite(y).all() for y in want)
    for turn in range(20):
        for got in _played(body):
            assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- a wait that is given up ----------------------------------------------------------------------------

@pytest.mark.parametrize("gated", [0, 1])
@pytest.mark.parametrize("n,k,splits", [(2048, 2048, 4), (256, 4096, 8), (40000, 256, 1)])
def test_a_product_one_of_whose_blocks_gives_up_is_nan(ops, n, k, splits, gated):
    """The blocks of one rank of their clusters take no wait: every result that their sums would have entered is NaN, and the next call is unaffected."""
    w = _to_device(ops.int4_pack(*_random(n, k, 64, 7)))
    x = torch.randn(50, k, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    call = ops.int4_linear_swiglu if gated else ops.int4_linear
    want, lib = call(x, w), ops._lib("int4")
    for trial in (-1, *range(splits), 8):
        out = torch.zeros_like(want)
        rc = lib.vapi_int4_linear(w.codes.data_ptr(), w.scales.data_ptr(), n, k, 64, x.data_ptr(), 50, None, out.data_ptr(), None, gated, 0, trial,
                                  torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        if 0 <= trial < splits:
            assert torch.isnan(out).all(), trial
        else:
            assert torch.equal(out, want)
        assert torch.equal(call(x, w), want)


# ---- calls of several threads ---------------------------------------------------------------------------

def test_threads_with_unlike_head_sizes(ops):
    """Head sizes that share a kernel but not an amount of shared memory, from four threads at a time."""
    i32 = lambda *v: torch.tensor(v, dtype=I32, device="cuda")

    def case(d):
        g = torch.Generator().manual_seed(d)
        cache = ops.Cache8(torch.randn(4, 2, 1, 16, d, generator=g).to(torch.float8_e4m3fn).cuda(), torch.zeros(4, 2, 1, 1, dtype=torch.int8, device="cuda"))
        q, table, cu, kl = torch.randn(2, 8 * d, generator=g).cuda(), i32(0, 1, 2, 3)[None], i32(0, 2), i32(50)
        return lambda: ops.paged_attention8(q, 8 * d, cache, table, cu, kl, 2, 1, 2, 50, 8, 1, d, 0.1)
    calls = [case(d) for d in (176, 256, 176, 256)]
    want, wrong, interval = [f() for f in calls], [], sys.getswitchinterval()

    def run(call, right, stream):
        try:
            with torch.cuda.stream(stream):
                for _ in range(20000):
                    got = call()
                if not torch.equal(got, right):
                    wrong.append("another result")
        except Exception as e:
            wrong.append(str(e))
    torch.cuda.synchronize()
    sys.setswitchinterval(1e-6)
    try:
        for _ in range(4):
            threads = [threading.Thread(target=run, args=(f, y, torch.cuda.Stream())) for f, y in zip(calls, want)]
            for t in threads:
                t.start()
            for t in threads:
                t.join()
    finally:
        sys.setswitchinterval(interval)
    torch.cuda.synchronize()
    assert not wrong, wrong


@pytest.mark.parametrize("d,dtype", [(64, BF), (128, BF), (64, F32), (48, BF)])
@pytest.mark.parametrize("requests,tokens", [(64, 1), (3, 5), (1, 40)])
def test_writes_one_after_the_other(ops, d, dtype, requests, tokens):
    """Steps of the same requests without a pause, each larger than the last, so that blocks' exponents, which lie side by side, keep growing; then the read."""
    nkv, nh, page, steps = 8, 8, 64, 20
    per = -(-steps * tokens // page)
    g = torch.Generator().manual_seed(d)
    x = torch.randn(steps, requests * tokens, (nh + 2 * nkv), d, generator=g)
    grow = torch.rand(steps, requests * tokens, nh + 2 * nkv, 1, generator=g).cumsum(0)
    x = (x * torch.exp2(2 * grow)).view(steps, requests * tokens, -1).to(dtype).cuda()
    order = torch.randperm(requests * per, generator=g).view(requests, per)
    pos = torch.arange(steps * tokens)
    slots = (order[:, pos // page] * page + pos % page).view(requests, steps, tokens).transpose(0, 1).reshape(steps, -1).to(I32).contiguous().cuda()
    cache, pages = ops.cache8_empty(requests * per, nkv, page, d), torch.arange(requests * per, dtype=I32, device="cuda")

    def body(between=lambda: None):
        cache.codes.view(torch.uint8).zero_()
        cache.exps.fill_(-110)
        for i in range(steps):
            between()
            ops.qk_norm_rope_write8(x[i], nh, nkv, d, None, None, 0.0, None, None, 0, cache, slots[i])
        between()
        return [ops.cache8_read(cache, pages, F32), cache.exps.clone()]
    want = body(torch.cuda.synchronize)
    for turn in range(10):
        for got in _played(body):
            assert all(torch.equal(a, b) for a, b in zip(got, want))
