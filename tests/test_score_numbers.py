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


def test_the_command_prints_json_whatever_the_numbers(tmp_path, capsys, monkeypatch):
    from vapi_b200 import TextScore, api, cli
    from conftest import TINY_A
    scores = [TextScore([1, 2, 3], [math.nan, -math.inf], [math.nan, 0.5], [[(4, math.nan)], [(5, -math.inf), (6, -0.5)]]), TextScore([1])]

    class Model:
        def score(self, prompts, top):
            return scores
    monkeypatch.setattr(api.LLM, "from_config", classmethod(lambda cls, cfg, **kw: Model()))
    path = tmp_path / "cfg.json"
    path.write_text(json.dumps(TINY_A))
    assert cli.main(["--random-weights", "0", "--config-json", str(path), "--prompt-ids", "1,2,3", "--prompt-ids", "1", "--score", "--logprobs", "2"]) == 0

    def refuse(word):
        raise ValueError(word)
    one, two = (json.loads(line, parse_constant=refuse) for line in capsys.readouterr().out.splitlines())
    assert one["logprobs"] == [None, None] and one["entropies"] == [None, 0.5] and one["top"] == [[[4, None]], [[5, None], [6, -0.5]]]
    assert one["perplexity"] is None and two["perplexity"] is None and two["logprobs"] == []
