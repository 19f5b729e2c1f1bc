"""Log probabilities of given tokens, entropy and alternatives (csrc/logprobs.cu)."""
import math

import pytest
import torch

import plain_fewer_bits as plain

gpu = pytest.mark.gpu


def _ops():
    from vapi_b200 import ops
    return ops


def test_what_does_not_fit_is_refused():
    ops = _ops()
    x, t = torch.zeros(3, 7), torch.zeros(3, dtype=torch.int32)
    for args, words in (((x[0], t), "R, V"), ((x.t(), t), "inner stride"), ((x.double(), t), "dtype"), ((x, t.long()), "int32"), ((x, t[:2]), "tokens must be"),
                        ((x, t, 8), "alternatives"), ((x, t, -1), "alternatives"), ((torch.zeros(3, 100), t, 65), "alternatives"), ((x, t, 2), "CUDA")):
        with pytest.raises(ops.KernelError, match=words):
            ops.token_logprobs(*args)


def _check(x, tokens, got, top, what=""):
    """ids exactly.  A log probability is x_j - m - ln s: half a float32 step of x_j - m and of the difference each, and s to within 2^-20 (a sum of
    V positive float32 terms added 16 of them, then threads, then warps deep, each 2^-24, the terms themselves 2^-22 of the
    base-2 exponential, and x - m times log2 e to half a step of at most 200).  The entropy is ln s - t / s with the same errors, t's
    on sum of p |x - m|."""
    want = plain.token_logprobs(x.cpu(), tokens, top)
    d = x.double().cpu()
    m = d.amax(1)
    mean = (torch.softmax(d, 1) * torch.where(d > -math.inf, (d - m[:, None]).abs(), 0.0)).sum(1)
    sums = 200 * 2.0 ** -24 + 2.0 ** -19 + d.shape[1] ** 0.5 * 2.0 ** -24
    ids = got.top_ids.cpu()
    assert torch.equal(ids, want.top_ids), what
    for a, b, far in ((got.logprob, want.logprob, (d.gather(1, tokens.long()[:, None])[:, 0] - m).abs()),
                      (got.top_logprobs, want.top_logprobs, (d.gather(1, want.top_ids.long()) - m[:, None]).abs())):
        a, b = a.double().cpu(), b.double()
        inf = b == -math.inf
        assert torch.equal(a[inf], b[inf]), what
        tol = sums + 2.0 ** -22 * (far + math.log(d.shape[1]) + 1)
        assert ((a - b).abs() <= tol)[~inf].all(), (what, float((a - b).abs()[~inf].max()))
    tol = sums * (2 + mean) + 2.0 ** -22 * (mean + math.log(d.shape[1]) + 1)
    assert ((got.entropy.double().cpu() - want.entropy.double()).abs() <= tol).all(), what


def _logits(rows, vocab, seed, dtype, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g) * spread).to(dtype), torch.randint(0, vocab, (rows,), generator=g).to(torch.int32)


# vocabularies shorter than a 16-byte piece, odd ones (rows begin anywhere), about one piece a thread, several batches
@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 2, 3, 7, 63, 509, 1027, 2049, 4099, 16385, 65536, 128256])
@pytest.mark.parametrize("top", [0, 1, 5, 20, 64])
def test_against_the_definition(vocab, top, dtype):
    ops = _ops()
    top = min(top, vocab)
    for rows in (1, 5, 37):
        x, t = _logits(rows, vocab, vocab + rows, dtype)
        dev = x.cuda()
        for slices in sorted({0, 1, 2, 8}):
            _check(x, t, ops.token_logprobs(dev, t.cuda(), top, slices=slices), top, (rows, slices))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_at_any_stride_and_many_rows(dtype):
    ops = _ops()
    x, t = _logits(700, 1003, 3, dtype)
    wide = torch.zeros(700, 1003 + 5, dtype=dtype)
    wide[:, 2:-3] = x
    got = ops.token_logprobs(wide.cuda()[:, 2:-3], t.cuda(), 9)
    _check(x, t, got, 9)
    for a, b in zip(got, ops.token_logprobs(wide.cuda()[:, 2:-3], t.cuda(), 9)):
        assert torch.equal(a, b)
    assert ops.token_logprobs(x.cuda()[:0], t.cuda()[:0], 3).top_ids.shape == (0, 3)
    assert ops.token_logprobs(x.cuda()[:, :1], torch.zeros(700, dtype=torch.int32).cuda(), 1).logprob.abs().max() == 0


@gpu
def test_rows_further_apart_than_32_bits():
    ops = _ops()
    x, t = _logits(2, 5000, 8, torch.bfloat16)
    stride = 2 ** 31 + 8
    wide = torch.empty(stride + 5000, dtype=torch.bfloat16, device="cuda").as_strided((2, 5000), (stride, 1))
    wide.copy_(x)
    _check(x, t, ops.token_logprobs(wide, t.cuda(), 7), 7)


@gpu
@pytest.mark.parametrize("slices", [1, 2, 8])
def test_ties_and_rows_made_to_fill_the_list(slices):
    """Equal logits go by id; descending and ascending rows; the largest all in the elements of a few threads (more above the bound
    than the list holds); zeros of both signs are one number."""
    ops = _ops()
    vocab = 40000
    rows = [torch.zeros(vocab), torch.arange(vocab).float() * -1e-3, torch.arange(vocab).float() * 1e-3, (torch.arange(vocab) % 7).float(),
            torch.where(torch.arange(vocab) % 2 == 0, 0.0, -0.0)]
    crowded = torch.randn(vocab, generator=torch.Generator().manual_seed(1))
    for j in range(20):                                  # element 4 * (512 * p + 8 * j) ..: one thread of each of 20 groups
        for p in range(0, vocab // 2048):
            crowded[2048 * p + 32 * j:2048 * p + 32 * j + 4] += 20
    for j in range(20):
        crowded[32 * j] += 9                             # ... and a bound below all of those
    rows += [crowded, torch.where(crowded > 15, 30.0, crowded)]
    x = torch.stack(rows)
    t = torch.randint(0, vocab, (len(rows),), generator=torch.Generator().manual_seed(2)).to(torch.int32)
    for top in (1, 20, 64):
        _check(x, t, ops.token_logprobs(x.cuda(), t.cuda(), top, slices=slices), top, top)


@gpu
def test_infinities_and_nan():
    ops = _ops()
    vocab = 3000
    x = torch.randn(6, vocab, generator=torch.Generator().manual_seed(4))
    x[0, 100:] = -math.inf                               # most of the row masked: fewer numbers than threads
    x[1, :] = -math.inf
    x[1, 2999] = 2.0
    x[2] = torch.finfo(torch.float32).min                # a mask of the type's lowest value
    x[2, 5] = 1.0
    t = torch.tensor([7, 0, 5, 1, 2, 3], dtype=torch.int32)
    for slices in (1, 2):
        got = ops.token_logprobs(x.cuda(), t.cuda(), 8, slices=slices)
        _check(x[[0, 1, 3]], t[[0, 1, 3]], ops.TokenLogprobs(*(v[[0, 1, 3]] for v in got)), 8)
        assert got.top_ids[1].tolist() == [2999, 0, 1, 2, 3, 4, 5, 6]
        assert got.logprob[2] == 0 and got.entropy[2] == 0 and got.top_ids[2].tolist() == [5, 0, 1, 2, 3, 4, 6, 7]
        assert got.logprob[1] == -math.inf and got.entropy[1] == 0
    x[3, 17], x[4, 17], x[5] = math.nan, math.inf, -math.inf
    got = ops.token_logprobs(x.cuda(), t.cuda(), 8)
    assert torch.isnan(got.logprob[3:]).all() and torch.isnan(got.entropy[3:]).all()
    assert torch.isfinite(got.entropy[:3]).all()


@gpu
def test_a_token_outside_the_vocabulary_leaves_a_status():
    ops = _ops()
    x, t = _logits(3, 100, 1, torch.float32)
    t[1] = 100
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = ops.token_logprobs(x.cuda(), t.cuda(), 2, status)
    assert int(status) == 1 and torch.isnan(got.logprob[1]) and torch.isfinite(got.logprob[[0, 2]]).all()
    t[1] = -1
    assert torch.isnan(ops.token_logprobs(x.cuda(), t.cuda(), 2).logprob[1])


@gpu
def test_captured_and_on_another_stream():
    ops = _ops()
    x, t = _logits(8, 65536, 1, torch.float32)
    x, t = x.cuda(), t.cuda()
    want = ops.token_logprobs(x, t, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a, b in zip(ops.token_logprobs(x, t, 5), want):
            assert torch.equal(a, b)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.token_logprobs(x, t, 5)
    x.copy_(x.flip(1))
    graph.replay()
    torch.cuda.synchronize()
    _check(x, t.cpu(), got, 5)
