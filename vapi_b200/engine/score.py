"""What a model says of given texts: the log probability of every token, the entropy it was one of, the alternatives."""
from __future__ import annotations

import math
from dataclasses import dataclass, field
from typing import List, Sequence, Tuple

import torch

from .. import ops
from .runner import ModelRunner
from .step import StepEntry

#: alternatives that are reported at most (as with the ``logprobs`` of a generated token)
MAX_TOP = 20
#: numbers of logits that stand on the device at a time
LOGITS_AT_ONCE = 1 << 27


@dataclass
class TextScore:
    """``logprobs[i]``, ``entropies[i]`` and ``top[i]`` are of token ``i + 1`` given those before it (natural logarithms)."""
    tokens: List[int]
    logprobs: List[float] = field(default_factory=list)
    entropies: List[float] = field(default_factory=list)
    top: List[List[Tuple[int, float]]] = field(default_factory=list)

    @property
    def perplexity(self) -> float:
        """exp of the mean negative log probability (NaN for a text of one token, and where a log probability is NaN; infinity where a
        token had none)."""
        if not self.logprobs:
            return math.nan
        mean = -sum(self.logprobs) / len(self.logprobs)
        return math.inf if mean >= 700 else math.exp(mean)


def score_texts(runner: ModelRunner, texts: Sequence[Sequence[int]], top: int = 0, portion: int = 2048) -> List[TextScore]:
    """Every text through the step function in portions of at most ``portion`` tokens, the logits of all its places wanted; a text
    holds pages and a slot only while it is scored."""
    if not 0 <= int(top) <= MAX_TOP:
        raise ValueError(f"{top} alternatives are outside 0..{MAX_TOP}")
    texts = [[int(t) for t in text] for text in texts]
    for i, text in enumerate(texts):
        if not text:
            raise ValueError(f"text {i} has no tokens")
        if len(text) > runner.max_context:
            raise ValueError(f"text {i} has {len(text)} tokens, the context {runner.max_context}")
        for t in text:
            if not 0 <= t < runner.vocab_size:
                raise ValueError(f"text {i}: token {t} is outside the vocabulary of {runner.vocab_size}")
    portion = max(1, min(int(portion), runner.max_batched_tokens, LOGITS_AT_ONCE // runner.vocab_size))
    top = min(int(top), runner.vocab_size)
    out = []
    for i, text in enumerate(texts):
        score = TextScore(text)
        cache = runner.cache.open(("score", i))
        try:
            for at in range(0, len(text) - 1, portion):
                part = text[at:min(at + portion, len(text) - 1)]         # (the last token predicts nothing that is known)
                if not runner.cache.reserve(cache, at + len(part)):
                    raise RuntimeError(f"text {i}: the cache has no pages for {at + len(part)} tokens")
                logits = runner.step([StepEntry(cache, part, range(len(part)))])
                targets = torch.tensor(text[at + 1:at + 1 + len(part)], dtype=torch.int32).to(logits.device)
                lp = ops.token_logprobs(logits, targets, top)
                logprobs, entropies, ids, tops = (t.tolist() for t in lp)
                runner.check_status()
                score.logprobs += logprobs
                score.entropies += entropies
                score.top += [list(zip(a, b)) for a, b in zip(ids, tops)]
        finally:
            runner.cache.close(cache)
        out.append(score)
    return out
