"""Where drafted tokens come from: any callable that takes a history (a list of token ids) and gives the tokens it expects
next, alone or with its probabilities (float32 [tokens, vocabulary] on the device) for them. Whatever it gives, the tokens
that come out are distributed as the model's own: the drafts only decide how many of them a step yields."""
from __future__ import annotations

import numpy as np

from ..errors import SamplingError


class PromptLookup:
    """Drafts by look-up: the tokens that followed the last occurrence of the history's last ``ngram`` tokens (of fewer, down to one,
    where the longer stretch occurs nowhere before). Certain of its tokens, so without probabilities; good for texts that repeat
    parts of their prompt."""

    def __init__(self, tokens: int = 4, ngram: int = 3):
        if tokens < 1 or ngram < 1:
            raise SamplingError(f"look-up drafts need at least one token and a stretch of one, got {tokens} and {ngram}")
        self.tokens, self.ngram = int(tokens), int(ngram)

    def __call__(self, history: list) -> list:
        h = np.asarray(history, dtype=np.int64)
        n = int(h.size)
        for size in range(min(self.ngram, n - 1), 0, -1):
            same = np.ones(n - size, dtype=bool)                     # by the place the stretch begins at, the last one left out
            for k in range(size):
                same &= h[k:n - size + k] == h[n - size + k]
            found = np.flatnonzero(same)
            if found.size:
                at = int(found[-1]) + size
                return h[at:at + self.tokens].tolist()
        return []
