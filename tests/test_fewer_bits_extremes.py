"""Attention over an 8-bit cache at the ends of the activations' range."""
import pytest
import torch

from test_cache8 import _attention_case, _check_attention, _portion_check, _run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("power", [119, 121, 124, 126])
@pytest.mark.parametrize("d,impl", [(64, "tensor_core"), (128, "tensor_core"), (64, "tcgen05"), (128, "tcgen05")])
def test_queries_next_to_the_largest_number(d, impl, power):
    """Queries up to 2^power over keys so small that their scores matter: the same as ordinary numbers."""
    c = _attention_case([70, 33], [5, 33], 4, 2, d, 64, torch.bfloat16, power)
    top = c["q"].float().abs().max()
    c["q"] = (c["q"].float() / top * 2.0 ** 16).bfloat16() * 2.0 ** (power - 16)              # (exact)
    assert torch.isfinite(c["q"]).all() and float(c["q"].abs().max()) >= 2.0 ** (power - 0.01)
    c["exps"][:, 0] = torch.randint(-110, -108, c["exps"][:, 0].shape, generator=torch.Generator().manual_seed(power)).to(torch.int8)
    scale = 2.0 ** (110 - power - 9) * d ** -0.5
    (_check_attention if impl == "tensor_core" else _portion_check)(c, _run_attention(c, scale, impl=impl), scale, **({"window": 0} if impl == "tcgen05" else {}))
