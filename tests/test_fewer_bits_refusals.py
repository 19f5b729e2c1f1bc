"""What the operators of serving in fewer bits, and the engine's options for them, refuse before anything runs."""
import pytest
import torch

BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32


@pytest.fixture
def ops():
    from vapi_b200 import ops
    return ops


@pytest.mark.parametrize("offset", [1, 2, 4, 8])
def test_the_c_functions_refuse_codes_off_16_bytes(ops, offset):
    """(with addresses that nothing is read from: the refusal comes before any launch)"""
    lib, at = ops._lib("cache8"), 1 << 20
    for d, dtype in ((64, 1), (64, 0), (48, 1), (256, 0)):
        rcs = (lib.vapi_qk_norm_rope_write8(at, dtype, None, None, 0.0, None, None, 0, at, at + offset, at, at, 3, 4, 2, d, 32, 5, None, None),
               lib.vapi_cache8_read(at + offset, at, at, at, dtype, 3, 2, d, 32, 5, None, None),
               lib.vapi_paged_attention8(at, 4 * d, at + offset, at, dtype, at, 2, at, at, at, 3, 1, 3, 5, 4, 2, d, 32, 5, 0.125, 0, 0, 0, 0, None, None))
        assert rcs == (-1, -1, -1), rcs
        assert b"16-byte" in lib.vapi_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_the_write_refuses_codes_off_16_bytes(ops, dtype):
    memory = torch.zeros(2 * 2 * 2 * 32 * 64 + 16, dtype=torch.uint8, device="cuda")
    exps, slots = torch.zeros(2, 2, 2, 2, dtype=torch.int8, device="cuda"), torch.arange(3, dtype=I32, device="cuda")
    qkv = torch.zeros(3, 512, dtype=dtype, device="cuda")
    for offset in (0, 1, 4, 16):
        cache = ops.Cache8(memory[offset:offset + 2 * 2 * 2 * 32 * 64].view(2, 2, 2, 32, 64).view(torch.float8_e4m3fn), exps)
        call = lambda: ops.qk_norm_rope_write8(qkv, 4, 2, 64, None, None, 0.0, None, None, 0, cache, slots)
        if offset % 16:
            before = ops.launch_count
            with pytest.raises(ops.KernelError, match="16-byte"):
                call()
            assert ops.launch_count == before
        else:
            call()


# ---- a plan that several runners use, one after the other ------------------------------------------------

def _plan_and_tensors(cfg, seed=3):
    from vapi_b200.config.model import resolve_architecture
    from vapi_b200.weights.random import random_tensors
    arch = resolve_architecture(cfg)
    plan = arch.plan(arch.parse(cfg))
    return plan, random_tensors(plan, seed, 0.1, "ones", F32, device="cpu")


def _runner(plan, tensors, **kw):
    from vapi_b200.engine.runner import ModelRunner
    return ModelRunner(plan, tensors, dtype="float32", device="cpu", num_pages=8, max_requests=2, max_batched_tokens=64, page_size=16, **kw)


def _paged(runner):
    return [(g.spec.eight_bit, g.tensor.dtype, g.exps is not None) for g in runner.cache.paged]


def test_a_runner_with_the_plan_of_an_eight_bit_one_keeps_numbers():
    from conftest import TINY_A
    plan, tensors = _plan_and_tensors(TINY_A)
    numbers, codes = [(False, F32, False)], [(True, torch.float8_e4m3fn, True)]
    for kind, want in (("auto", numbers), ("fp8", codes), ("auto", numbers), ("fp8", codes)):
        r = _runner(plan, tensors, kv_cache_dtype=kind)
        assert _paged(r) == want and all(getattr(b.mixer, "cache8", False) == (kind == "fp8") for b in plan.layers if hasattr(b.mixer, "nkv"))


def test_a_refusal_leaves_the_plan_as_it_was():
    from conftest import TINY_A
    plan, tensors = _plan_and_tensors(TINY_A)
    with pytest.raises(ValueError, match="groups of 128"):
        _runner(plan, tensors, kv_cache_dtype="fp8", weight_dtype="int4", weight_group=128)
    assert not any(getattr(b.mixer, "cache8", False) for b in plan.layers)
    last = [b.mixer for b in plan.layers if hasattr(b.mixer, "nkv")][-1]
    last.general = True
    with pytest.raises(ValueError, match="no form with a cache in 8 bits"):
        _runner(plan, tensors, kv_cache_dtype="fp8")
    last.general = False
    assert not any(getattr(b.mixer, "cache8", False) for b in plan.layers) and _paged(_runner(plan, tensors)) == [(False, F32, False)]
