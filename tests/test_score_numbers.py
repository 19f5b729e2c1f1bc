"""What a text's score says where a log probability is no ordinary number."""
import json
import math

import pytest


@pytest.mark.parametrize("logprobs,want", [([-1.0, -3.0], math.exp(2.0)), ([-1.0, -math.inf], math.inf), ([-2000.0], math.inf), ([-1.0, math.nan], math.nan),
                                           ([math.nan, -math.inf], math.nan), ([0.0, 0.0], 1.0), ([], math.nan)])
def test_perplexity(logprobs, want):
    from vapi_b200 import TextScore
    got = TextScore(list(range(len(logprobs) + 1)), logprobs).perplexity
    assert math.isnan(got) if math.isnan(want) else got == pytest.approx(want)
