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
