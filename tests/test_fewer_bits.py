"""Serving in fewer bits through the engine: 8-bit keys and values, 4-bit weights, scoring, log probabilities of generated tokens."""
import json
import math

import pytest
import torch

import plain_fewer_bits as plain
from conftest import TINY_A

gpu = pytest.mark.gpu


@pytest.fixture()
def plain_fewer(plain_kernels, monkeypatch):
    """The plain restatements of these operators too, and products that take either kind of weight."""
    from vapi_b200 import ops
    for name in plain.OPS:
        monkeypatch.setattr(ops, name, getattr(plain, name))
    four = lambda w: isinstance(w, ops.Int4Weight)
    linear, swiglu = plain_kernels.linear, plain_kernels.swiglu
    monkeypatch.setattr(ops, "linear", lambda x, w, b=None, dt=None: plain.int4_linear(x, w, b, dt) if four(w) else linear(x, w, b, dt))
    monkeypatch.setattr(ops, "linear_swiglu", lambda x, w, act="silu": plain.int4_linear_swiglu(x, w, act) if four(w) else swiglu(linear(x, w), act))
    return plain


def _runner(cfg, device="cpu", dtype="float32", seed=3, pages=24, std=0.1, **kw):
    from vapi_b200.engine.runner import ModelRunner
    return ModelRunner.from_random(cfg, seed, dtype=dtype, device=device, std=std, norm_init="perturbed", num_pages=pages, max_requests=8, max_batched_tokens=256,
                                   page_size=kw.pop("page_size", 16 if device == "cpu" else 64), **kw)


def _prompt(n, vocab=256, seed=0):
    return torch.randint(8, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def _logits(runner, tokens, portions):
    """Logits of every place, the text taken in these portions."""
    from vapi_b200.engine.step import StepEntry
    rc, out, at = runner.cache.open("x"), [], 0
    for n in portions:
        assert runner.cache.reserve(rc, at + n)
        out.append(runner.step([StepEntry(rc, tokens[at:at + n], range(n))]).float().cpu().clone())
        at += n
    if runner.device.type == "cuda":
        runner.check_status()
    return torch.cat(out), rc


# ---- what is refused ----------------------------------------------------------------------------------

def test_options_that_have_no_such_form_are_refused():
    from vapi_b200.config.runtime import RuntimeConfig, RuntimeConfigError
    for kw, words in ((dict(kv_cache_dtype="int8"), "kv_cache_dtype"), (dict(weight_dtype="fp4"), "weight_dtype"), (dict(weight_group=16), "weight_group"),
                      (dict(weight_dtype="int4", weight_group=128), "groups of 128")):
        with pytest.raises(ValueError, match=words):
            _runner(TINY_A, **kw)
    for section, body, words in (("model", {"weight_dtype": "int8"}, "weight_dtype"), ("model", {"weight_group": 48}, "weight_group"), ("cache", {"dtype": "int4"}, "cache.dtype")):
        with pytest.raises(RuntimeConfigError, match=words):
            RuntimeConfig.from_dict({section: body})
    cfg = RuntimeConfig.from_dict({"model": {"weight_dtype": "int4", "weight_group": 32}, "cache": {"dtype": "fp8"}})
    assert (cfg.model.weight_dtype, cfg.model.weight_group, cfg.cache.dtype) == ("int4", 32, "fp8")


def test_models_that_have_no_such_form_are_refused():
    from vukavik_util import TINY as vukavik
    for kw, words in ((dict(kv_cache_dtype="fp8"), "cache in 8 bits"), (dict(weight_dtype="int4", weight_group=32), "4-bit weights")):
        with pytest.raises(ValueError, match=words):
            _runner(vukavik, **kw)


def test_a_cache_of_codes_takes_half_the_bytes():
    full, half = _runner(TINY_A), _runner(TINY_A, kv_cache_dtype="fp8")
    # two attention layers of two kv heads of 16: 128 numbers a token and a byte for each 16 of their rows
    assert full.cache.bytes_per_token() == 2 * 64 * 4 and half.cache.bytes_per_token() == -(-(2 * 64 * 16 + 2 * 4) // 16)
    (group,) = half.cache.paged
    assert group.tensor.dtype == torch.float8_e4m3fn and group.exps.shape == (2, 24, 4) and full.cache.paged[0].exps is None


# ---- host logic on the plain operators ----------------------------------------------------------------

def test_scores_are_the_models_own_distribution(plain_kernels, plain_fewer):
    from vapi_b200.engine.score import score_texts
    runner = _runner(TINY_A)
    texts = [_prompt(45), _prompt(1, seed=1), _prompt(2, seed=2)]
    scores = score_texts(runner, texts, top=3, portion=16)
    want, rc = _logits(runner, texts[0], [45])
    runner.cache.close(rc)
    lp = torch.log_softmax(want.double(), 1)
    assert [len(s.logprobs) for s in scores] == [44, 0, 1] and math.isnan(scores[1].perplexity)
    s = scores[0]
    assert s.tokens == texts[0]
    for i in range(44):
        assert abs(s.logprobs[i] - float(lp[i, texts[0][i + 1]])) < 1e-4
        assert abs(s.entropies[i] + float((lp[i].exp() * lp[i]).sum())) < 1e-4
        ids = torch.argsort(-lp[i], stable=True)[:3]
        assert [t for t, _ in s.top[i]] == ids.tolist() and all(abs(v - float(lp[i, t])) < 1e-4 for t, v in s.top[i])
    assert abs(math.log(s.perplexity) + sum(s.logprobs) / 44) < 1e-9
    runner.cache.check_invariants()
    for bad, words in (([[]], "no tokens"), ([[256]], "vocabulary"), ([[-1]], "vocabulary"), ([[1] * 400], "context")):
        with pytest.raises(ValueError, match=words):
            score_texts(runner, bad)
    with pytest.raises(ValueError, match="alternatives"):
        score_texts(runner, [[1, 2]], top=21)
    small = _runner(TINY_A, pages=24)
    held = small.cache.open("held")
    assert small.cache.reserve(held, 23 * 16)
    with pytest.raises(RuntimeError, match="pages"):
        score_texts(small, [_prompt(40)])
    small.cache.close(held)
    assert len(score_texts(small, [_prompt(40)])[0].logprobs) == 39            # (what it held has gone back)
    small.cache.check_invariants()


@pytest.mark.parametrize("kw", [dict(kv_cache_dtype="fp8"), dict(weight_dtype="int4", weight_group=32), dict(kv_cache_dtype="fp8", weight_dtype="int4", weight_group=64)])
def test_the_engine_generates_and_scores_in_fewer_bits(plain_kernels, plain_fewer, kw):
    from vapi_b200.engine.engine import Engine
    from vapi_b200.engine.scheduler import SchedulerConfig
    from vapi_b200.engine.score import score_texts
    from vapi_b200.sampling.params import SamplingParams
    runner = _runner(TINY_A, **kw)
    eng = Engine(runner, SchedulerConfig(prefill_chunk_tokens=20))
    p = _prompt(37)
    eng.admit("a", p, SamplingParams(temperature=0.0, max_tokens=6, ignore_eos=True, logprobs=2))
    (done,) = eng.run()
    s = score_texts(runner, [p + done.tokens])[0]
    # the text's scores at the generated places are the generated tokens' own (4-bit weights alone: the same numbers; with codes the
    # blocks of a text taken at once begin on the scale of all their tokens, a generated one's on that of the first)
    for lp, again in zip(done.logprobs, s.logprobs[36:]):
        assert abs(lp.logprob - again) < (1e-4 if "kv_cache_dtype" not in kw else 0.3)
        assert lp.entropy is not None and lp.top[0] == (lp.token, pytest.approx(lp.logprob))
    runner.cache.check_invariants()


def test_the_command_scores(tmp_path, capsys, monkeypatch, plain_kernels, plain_fewer):
    from vapi_b200 import api, cli
    path = tmp_path / "cfg.json"
    path.write_text(json.dumps(TINY_A))
    real = api.ModelRunner.from_random
    monkeypatch.setattr(api.ModelRunner, "from_random", classmethod(lambda cls, c, seed, **kw: real(
        c, seed, **{**kw, "device": "cpu", "dtype": "float32", "num_pages": 24, "max_requests": 4, "max_batched_tokens": 64, "page_size": 16})))
    args = ["--random-weights", "0", "--config-json", str(path), "--prompt-ids", "9,10,11,12", "--prompt-ids", "30"]
    assert cli.main(args + ["--score", "--logprobs", "2", "--kv-cache-dtype", "fp8", "--weight-dtype", "int4", "--weight-group", "32"]) == 0
    one, two = (json.loads(l) for l in capsys.readouterr().out.splitlines())
    assert len(one["logprobs"]) == len(one["entropies"]) == len(one["top"]) == 3 and one["perplexity"] > 1 and two["perplexity"] is None
    assert cli.main(args + ["--score", "--logprobs", "40"]) == 2 and "alternatives" in capsys.readouterr().err
    assert cli.main(args + ["--weight-dtype", "int4", "--weight-group", "128"]) == 2 and "groups of 128" in capsys.readouterr().err


# ---- on the device ------------------------------------------------------------------------------------

def _from_dir(path, device, dtype="float32", **kw):
    from vapi_b200.engine.runner import ModelRunner
    return ModelRunner.from_dir(path, dtype=dtype, device=device, num_pages=24, max_requests=8, max_batched_tokens=256, page_size=kw.pop("page_size", 16), **kw)


@pytest.fixture()
def on_the_host(tiny_dirs):
    """A function that runs a text on the plain operators, and leaves the kernels in place behind it."""
    import plain_ops
    from vapi_b200 import ops

    def run(model, tokens, portions, **kw):
        with pytest.MonkeyPatch.context() as m:
            for name in plain_ops.ALL:
                m.setattr(ops, name, getattr(plain_ops, name))
            for name in plain.OPS:
                m.setattr(ops, name, getattr(plain, name))
            four = lambda w: isinstance(w, ops.Int4Weight)
            m.setattr(ops, "linear", lambda x, w, b=None, dt=None: plain.int4_linear(x, w, b, dt) if four(w) else plain_ops.linear(x, w, b, dt))
            m.setattr(ops, "linear_swiglu", lambda x, w, act="silu": plain.int4_linear_swiglu(x, w, act) if four(w) else plain_ops.swiglu(plain_ops.linear(x, w), act))
            return _logits(_from_dir(tiny_dirs[model], "cpu", **kw), tokens, portions)[0]
    return run


@gpu
@pytest.mark.parametrize("model", ["A", "B", "D", "E"])
def test_float32_models_match_the_plain_operators(model, tiny_dirs, on_the_host):
    """4-bit weights: the same numbers on both sides, float32 sums apart.  With the cache's codes: a key or value within 2^-20 of the
    border between two codes may fall either way (float32 sums apart), one of some 10^4 here at most, and moves its one
    product by an eighth: a hundredth of the largest logit covers several."""
    for kw, tol in ((dict(weight_dtype="int4", weight_group=32), 2e-4), (dict(kv_cache_dtype="fp8"), 1e-2),
                    (dict(kv_cache_dtype="fp8", weight_dtype="int4", weight_group=32), 1e-2)):
        tokens, portions = _prompt(60), [23, 1, 1, 30, 1, 4]
        want = on_the_host(model, tokens, portions, **kw)
        got, _ = _logits(_from_dir(tiny_dirs[model], "cuda", **kw), tokens, portions)
        assert (got - want).abs().max() <= tol * want.abs().max(), (kw, float((got - want).abs().max()), float(want.abs().max()))


@gpu
@pytest.mark.parametrize("model", ["D", "E"])
def test_the_first_layers_codes_are_those_of_the_whole_cache(model, tiny_dirs):
    """What reaches the first attention layer does not depend on how it caches: its codes stand for the keys and values that the
    16-bit cache holds, within half a step of the code (2^-4 of the number, or half the block's smallest step) and one of bfloat16."""
    tokens, n = _prompt(90), 90
    caches = []
    for kw in (dict(), dict(kv_cache_dtype="fp8")):
        r = _from_dir(tiny_dirs[model], "cuda", "bfloat16", page_size=64, **kw)
        _, rc = _logits(r, tokens, [n])
        site = min(s for s in r._site_buffers if r.cache.site_kind(s)[0] == "paged")
        table = rc.tables[0]
        caches.append((r, site, table))
    from vapi_b200 import ops
    (full, site, table), (half, site8, table8) = caches
    d, nkv = full.cache.site_spec(site).buffers[0].width, full.cache.site_spec(site).buffers[0].rows
    whole = full.cache.site_tensor(site).view(-1, 2, nkv, 64, d)[table].double().cpu()
    codes = ops.Cache8(half.cache.site_tensor(site8).view(-1, 2, nkv, 64, d), half.cache.site_exps(site8).view(-1, 2, nkv, 4))
    got = ops.cache8_read(codes, torch.tensor(table8, dtype=torch.int32).cuda(), torch.float32).double().cpu()
    step = torch.exp2(codes.exps[table8].double().cpu()).repeat_interleave(16, -1)[..., None] * 2.0 ** -9
    over = (got - whole).abs() - torch.maximum((2.0 ** -4 + 2.0 ** -7) * whole.abs(), 2.0 ** -7 * whole.abs() + step / 2)
    flat = lambda t: t.permute(1, 2, 0, 3, 4).reshape(2, nkv, -1, d)[:, :, :n]
    assert (flat(over) <= 0).all() and flat(whole).abs().max() > 0


BOTH = dict(kv_cache_dtype="fp8", weight_dtype="int4", weight_group=32)


@gpu
@pytest.mark.parametrize("dtype,tol", [("bfloat16", 0.05), ("float32", 0.01)])
@pytest.mark.parametrize("kw", [dict(kv_cache_dtype="fp8"), BOTH], ids=["cache", "both"])
def test_captured_and_batched_decoding_is_what_single_steps_give(kw, dtype, tol, tiny_dirs):
    """Requests of unlike lengths given the same tokens: side by side and captured (padded to eight, their keys cut as for the longest
    context), side by side, and each alone.  Sums are taken in other orders, so a key or value next to the border of two codes may fall
    either way, an eighth of it: a hundredth of the largest logit in float32, where few do; bfloat16 activations differ by a step of 2^-7
    now and then, in four layers."""
    from vapi_b200.engine.step import StepEntry
    texts = [_prompt(n + 18, seed=n) for n in (5, 16, 17, 40, 63)]

    def run(graphs, together):
        r = _from_dir(tiny_dirs["D"], "cuda", dtype, page_size=64, **kw)
        out = [[] for _ in texts]
        for group in ([list(enumerate(texts))] if together else [[x] for x in enumerate(texts)]):
            held = [r.cache.open(i) for i, _ in group]
            for step in range(19):
                entries = []
                for (i, t), rc in zip(group, held):
                    part = t[:len(t) - 18] if step == 0 else t[len(t) - 19 + step:len(t) - 18 + step]
                    assert r.cache.reserve(rc, rc.num_tokens + len(part))
                    entries.append(StepEntry(rc, part, [len(part) - 1]))
                got = r.step_decode_graph(entries) if graphs and step else r.step(entries)
                for (i, _), row in zip(group, got.float().cpu().clone()):
                    out[i].append(row)
            r.check_status()
        return torch.stack([torch.stack(o) for o in out])
    whole = run(True, True)
    for other in (run(False, True), run(False, False)):
        assert torch.isfinite(other).all() and (other - whole).abs().max() <= tol * whole.abs().max(), float((other - whole).abs().max() / whole.abs().max())


@gpu
@pytest.mark.parametrize("graphs", [True, False])
def test_the_engine_generates_to_the_end(graphs, tiny_dirs):
    from vapi_b200.engine.engine import Engine
    from vapi_b200.engine.scheduler import SchedulerConfig
    from vapi_b200.sampling.params import SamplingParams
    r = _from_dir(tiny_dirs["D"], "cuda", "bfloat16", page_size=64, **BOTH)
    eng = Engine(r, SchedulerConfig(prefill_chunk_tokens=24), use_graphs=graphs)
    for n in (5, 16, 17, 40, 63):
        eng.admit(n, _prompt(n, seed=n), SamplingParams(temperature=0.0, max_tokens=20, ignore_eos=True))
    done = eng.run()
    assert len(done) == 5 and all(len(f.tokens) == 20 and f.reason.value == "length" for f in done) and eng.stats.failed_steps == 0
    r.cache.check_invariants()


@gpu
def test_preempted_requests_come_back(tiny_dirs):
    """Too few pages for all: a request that is put off is computed again, its blocks on the scales of the portions it then comes in."""
    from vapi_b200.engine.engine import Engine
    from vapi_b200.engine.scheduler import SchedulerConfig
    from vapi_b200.sampling.params import SamplingParams
    from vapi_b200.engine.runner import ModelRunner

    def run(pages):
        r = ModelRunner.from_dir(tiny_dirs["D"], dtype="float32", device="cuda", num_pages=pages, max_requests=4, max_batched_tokens=256, page_size=16, **BOTH)
        eng = Engine(r, SchedulerConfig(prefill_chunk_tokens=64))
        for i in range(3):
            eng.admit(i, [11 + i] * 30, SamplingParams(temperature=0.0, max_tokens=30, ignore_eos=True))
        done = {f.request_id: f for f in eng.run()}
        r.cache.check_invariants()
        return done
    few, many = run(9), run(24)
    assert sum(f.preemptions for f in few.values()) > 0
    assert all(len(f.tokens) == 30 and f.reason.value == "length" for f in few.values()) and all(f.preemptions == 0 for f in many.values())


@gpu
def test_scores_and_generated_log_probabilities_on_the_device(tiny_dirs):
    from vapi_b200 import LLM, SamplingParams
    llm = LLM(tiny_dirs["D"], dtype="float32", num_blocks=24, page_size=64, max_concurrent_seqs=4, max_batched_tokens=256, prefill_chunk_tokens=50)
    text = _prompt(130, 1000)
    s = llm.score([text, [5]], top=4)
    want, rc = _logits(llm.runner, text, [130])
    llm.runner.cache.close(rc)
    lp = torch.log_softmax(want.double(), 1)
    assert len(s[0].logprobs) == 129 and s[1].logprobs == []
    for i in range(129):
        assert abs(s[0].logprobs[i] - float(lp[i, text[i + 1]])) < 1e-3 and abs(s[0].entropies[i] + float((lp[i].exp() * lp[i]).sum())) < 1e-3
        assert abs(s[0].top[i][0][1] - float(lp[i].max())) < 1e-3 and len(s[0].top[i]) == 4
    # requests with and without penalties side by side: log probabilities are of the raw logits
    pen = SamplingParams(temperature=0.0, max_tokens=6, ignore_eos=True, logprobs=3, presence_penalty=1.5, repetition_penalty=1.3)
    got = llm.generate([text[:40], text[:40], text[:30]], [pen, SamplingParams(temperature=0.8, seed=3, max_tokens=6, ignore_eos=True),
                                                          SamplingParams(temperature=0.0, max_tokens=6, ignore_eos=True, logprobs=0)])
    assert got[1].logprobs is None
    for c, prompt, k in ((got[0], text[:40], 3), (got[2], text[:30], 0)):
        again = llm.score([prompt + c.tokens], top=3)[0]
        for i, rec in enumerate(c.logprobs):
            j = len(prompt) - 1 + i
            assert rec.token == c.tokens[i] and abs(rec.logprob - again.logprobs[j]) < 1e-3 and abs(rec.entropy - again.entropies[j]) < 1e-3
            assert len(rec.top) == k and all(abs(a[1] - b[1]) < 1e-3 for a, b in zip(rec.top, again.top[j]))
    with pytest.raises(ValueError, match="vocabulary"):
        llm.score([[10 ** 6]])
    llm.engine.admit("live", text[:10], SamplingParams(max_tokens=2))
    with pytest.raises(RuntimeError, match="between"):
        llm.score([text])
    llm.engine.run()


@gpu
def test_serving_widths_in_fewer_bits():
    """Layers as wide as the 1.2B and the 700M size: decode, short and long portions through the kernels that serve them.  The same
    weights in 16 and in fewer bits say nearly the same of a text: the largest parts of what is lost are 2^-4 steps of keys and
    values and steps of a fifteenth of a group's width, against layers whose outputs add to a stream that keeps the embedding."""
    from conftest import serving_width_config
    from vapi_b200.engine.score import score_texts
    for sizes in ("1.2b", "700m"):
        cfg = serving_width_config(sizes)
        text = _prompt(700, 4096)
        scores = []
        for kw in (dict(), dict(kv_cache_dtype="fp8"), dict(kv_cache_dtype="fp8", weight_dtype="int4", weight_group=64)):
            r = _runner(cfg, "cuda", "bfloat16", pages=16, std=0.02, max_context=1024, **kw)
            whole = score_texts(r, [text], portion=256)[0]
            split = score_texts(r, [text[:300]], portion=1)[0]
            assert all(math.isfinite(v) for v in whole.logprobs + split.logprobs)
            scores.append((torch.tensor(whole.logprobs), torch.tensor(split.logprobs)))
        for a, b in zip(scores[1:], (0.05, 0.5)):
            for x, y in zip(a, scores[0]):
                assert (x - y).abs().mean() < b, (sizes, float((x - y).abs().mean()))
