"""The native calls (csrc/calls.cpp) of the operators of serving in fewer bits against the same steps in Python, and what neither takes."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32


@pytest.fixture
def ops():
    from vapi_b200 import ops
    return ops


def _calls(ops):
    """name -> (a call by keyword, its good arguments)."""
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    i = lambda *v: torch.tensor(v, dtype=I32, device="cuda")
    cache = ops.Cache8(r(3, 2, 2, 32, 64).to(torch.float8_e4m3fn), torch.zeros(3, 2, 2, 2, dtype=torch.int8, device="cuda"))
    w = ops.int4_quantize(r(64, 128), 64)
    ang = r(3, 32)
    return {
        "write": (lambda **k: ops.qk_norm_rope_write8(k["qkv"], 4, 2, 64, k["qw"], k["kw"], 1e-5, k["cos"], k["sin"], 64, k["cache"], k["slots"]),
                  dict(qkv=r(3, 512).to(BF), qw=r(64), kw=r(64), cos=ang.cos(), sin=ang.sin(), cache=cache, slots=i(5, 6, 40))),
        "read": (lambda **k: ops.cache8_read(k["cache"], k["pages"], k["dtype"]), dict(cache=cache, pages=i(2, 0), dtype=BF)),
        "attention": (lambda **k: ops.paged_attention8(k["q"], k["stride"], k["cache"], k["table"], k["cu"], k["kl"], 3, 2, 2, 40, 4, 2, 64, 0.125, k["window"]),
                      dict(q=r(3, 512).to(BF), stride=512, cache=cache, table=i(1, 2, 0, 0).view(2, 2), cu=i(0, 2, 3), kl=i(40, 7), window=0)),
        "int4": (lambda **k: ops.int4_linear(k["x"], k["w"], k["bias"], k["dtype"]), dict(x=r(5, 128).to(BF), w=w, bias=r(64), dtype=None)),
        "gated": (lambda **k: ops.int4_linear_swiglu(k["x"], k["w"], k["act"]), dict(x=r(5, 128).to(BF), w=w, act="silu")),
        "logprobs": (lambda **k: ops.token_logprobs(k["x"], k["t"], k["top"]), dict(x=r(5, 100), t=i(1, 2, 3, 4, 99), top=3)),
    }


def _copy(args):
    return {k: type(v)(*(t.clone() for t in v)) if isinstance(v, tuple) else v for k, v in args.items()}


VARIANTS = [("write", {}), ("write", dict(qw=None, kw=None, cos=None, sin=None)), ("read", {}), ("read", dict(dtype=F32)), ("attention", {}), ("attention", dict(window=9)),
            ("int4", {}), ("int4", dict(bias=None, dtype=F32)), ("gated", {}), ("gated", dict(act="gelu_tanh")), ("logprobs", {}), ("logprobs", dict(top=0))]


@pytest.mark.parametrize("name,change", VARIANTS)
def test_native_and_python_calls_are_one(ops, monkeypatch, name, change):
    call, good = _calls(ops)[name]
    got, caches, counts = [], [], []
    for native in (True, False):
        if not native:
            monkeypatch.setattr(ops, "_calls_module", ops._NoCalls)
        else:
            ops._calls()
            real = ops._calls_module
            answers = []

            class Heard:
                def __getattr__(self, which):
                    def fn(*a):
                        answers.append(getattr(real, which)(*a))
                        return answers[-1]
                    return fn
            monkeypatch.setattr(ops, "_calls_module", Heard())
        args = _copy({**good, **change})
        before = ops.launch_count
        out = call(**args)
        counts.append(ops.launch_count - before)
        got.append(out if isinstance(out, tuple) else (out,))
        caches.append(args.get("cache"))
        monkeypatch.undo()
        if native:
            assert answers and all(x is not NotImplemented for x in answers)
    assert counts == [1, 1] and type(got[0]) is type(got[1])
    for a, b in zip(*got):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)
    if name == "write":
        assert torch.equal(caches[0].codes.view(torch.uint8), caches[1].codes.view(torch.uint8)) and torch.equal(caches[0].exps, caches[1].exps)


def _bad(ops):
    f = lambda *s, dt=F32: torch.zeros(*s, device="cuda", dtype=dt)
    good = {name: args for name, (_, args) in _calls(ops).items()}
    cache = good["read"]["cache"]
    caches = [dict(cache=ops.Cache8(cache.codes.view(torch.uint8), cache.exps)), dict(cache=ops.Cache8(cache.codes, cache.exps[:, :, :, :1])),
              dict(cache=ops.Cache8(cache.codes.cpu(), cache.exps)), dict(cache=ops.Cache8(cache.codes[:, :, :, ::2], cache.exps)),
              dict(cache=ops.Cache8(cache.codes, cache.exps.int()))]
    w = good["int4"]["w"]
    return ([("write", c) for c in caches] + [("read", c) for c in caches] + [("attention", c) for c in caches]
            + [("write", c) for c in (dict(qkv=f(3, 511, dt=BF)), dict(qkv=f(3, 512, dt=torch.float16)), dict(qkv=f(512, 3, dt=BF).t()), dict(qw=f(63)), dict(kw=f(64, dt=BF)),
                                      dict(cos=None), dict(cos=f(2, 32)), dict(sin=f(3, 31)), dict(slots=f(2, dt=I32)), dict(slots=f(3, dt=torch.int64)), dict(slots=f(6, dt=I32)[::2]),
                                      dict(slots=torch.zeros(3, dtype=I32)))]
            + [("read", c) for c in (dict(pages=f(2)), dict(pages=f(4, dt=I32)[::2]), dict(dtype=torch.float16), dict(pages=torch.zeros(2, dtype=I32)))]
            + [("attention", c) for c in (dict(q=f(3, 512, dt=torch.float16)), dict(stride=255), dict(stride=1024), dict(table=f(1, 2, dt=I32)), dict(table=f(2, 2, dt=I32).t()[:, :1].t()[:1]),
                                          dict(cu=f(2, dt=I32)), dict(kl=f(1, dt=I32)), dict(kl=f(2)), dict(cu=torch.zeros(3, dtype=I32)), dict(q=f(1, 512, dt=BF)))]
            + [("int4", c) for c in (dict(x=f(5, 64, dt=BF)), dict(x=f(5, 128, dt=torch.float16)), dict(bias=f(63)), dict(bias=f(64, dt=BF)), dict(dtype=torch.float16),
                                     dict(w=w.codes), dict(x=torch.zeros(5, 128, dtype=BF)), dict(w=ops.Int4Weight(w.codes.cpu(), w.scales, w.n, w.k, w.group)))]
            + [("gated", c) for c in (dict(x=f(5, 64, dt=BF)), dict(act="relu"))]
            + [("logprobs", c) for c in (dict(t=f(4, dt=I32)), dict(t=f(5, dt=torch.int64)), dict(top=65), dict(top=-1), dict(x=f(5, 2)), dict(x=f(100, 5).t()), dict(x=f(5, 100, dt=torch.float16)))])


@pytest.mark.parametrize("native", [True, False])
def test_what_does_not_fit_is_refused_by_both(ops, monkeypatch, native):
    if not native:
        monkeypatch.setattr(ops, "_calls_module", ops._NoCalls)
    calls = _calls(ops)
    for n, (name, change) in enumerate(_bad(ops)):
        call, good = calls[name]
        before = ops.launch_count
        with pytest.raises(ops.KernelError):
            call(**{**good, **change})
            pytest.fail(f"{n}: {name} {list(change)}")
        assert ops.launch_count == before, (n, name)


def test_the_c_functions_own_refusals(ops):
    f = lambda *s, dt=F32: torch.zeros(*s, device="cuda", dtype=dt)
    i = lambda *v: torch.tensor(v, dtype=I32, device="cuda")
    for d in (8, 24, 272):
        cache = ops.cache8_empty(1, 1, 16, d)
        with pytest.raises(ops.KernelError, match="multiple of 16"):
            ops.qk_norm_rope_write8(f(1, 3 * d), 1, 1, d, None, None, 0.0, None, None, d, cache, i(0))
        with pytest.raises(ops.KernelError, match="multiple of 16"):
            ops.cache8_read(cache, i(0), F32)
        with pytest.raises(ops.KernelError, match="multiple of 16"):
            ops.paged_attention8(f(1, d), d, cache, i(0).view(1, 1), i(0, 1), i(1), 1, 1, 1, 1, 1, 1, d, 1.0)
    cache = ops.cache8_empty(1, 1, 16, 64)
    with pytest.raises(ops.KernelError, match="rotation"):
        ops.qk_norm_rope_write8(f(1, 192), 1, 1, 64, None, None, 0.0, f(1, 40), f(1, 40), 80, cache, i(0))
    with pytest.raises(ops.KernelError, match="positive"):
        ops.paged_attention8(f(1, 64, dt=BF), 64, cache, i(0).view(1, 1), i(0, 1), i(1), 1, 1, 1, 1, 1, 1, 64, -1.0, impl="tcgen05")
    for slices in (3, 16, -1):
        with pytest.raises(ops.KernelError, match="power of two"):
            ops.token_logprobs(f(1, 10), i(0), 1, slices=slices)


def test_operators_on_two_streams_at_once(ops):
    """Kernels that hold tensor memory and wait for their cluster, beside one another and in turn."""
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(4)
    cache = ops.cache8_empty(20, 8, 64, 64)
    qkv = torch.randn(1280, 48 * 64, generator=g).bfloat16().cuda()
    ops.qk_norm_rope_write8(qkv, 32, 8, 64, None, None, 0.0, None, None, 0, cache, torch.arange(1280, dtype=torch.int32, device="cuda"))
    q, table, cu, kl = qkv[:200], torch.arange(20, dtype=torch.int32, device="cuda")[None], i32(0, 200), i32(1280)
    w = ops.int4_quantize(torch.randn(2048, 2048, generator=g).cuda())
    x, logits, tokens = torch.randn(64, 2048, generator=g).bfloat16().cuda(), torch.randn(8, 30000, generator=g).cuda(), i32(*range(8))
    calls = [lambda: ops.paged_attention8(q, qkv.stride(0), cache, table, cu, kl, 200, 1, 200, 1280, 32, 8, 64, 0.125),
             lambda: ops.int4_linear(x, w), lambda: ops.int4_linear_swiglu(x[:3], w), lambda: ops.token_logprobs(logits, tokens, 5).top_logprobs]
    want = [f() for f in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for turn in range(40):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got.append([calls[(j + 2 * i) % 4]() for j in range(4)])
    torch.cuda.synchronize()
    for n, outs in enumerate(got):
        for j, o in enumerate(outs):
            assert torch.equal(o, want[(j + 2 * (n % 2)) % 4]), (n, j)
