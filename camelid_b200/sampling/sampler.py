"""The sampler on the device: one call per step for the whole batch.

Greedy is an argmax kernel. Otherwise the logits are adjusted in place (bias, repeat,
presence and frequency penalties over each request's history, prompt included, as
src/main.rs:3714-3733 passes it) and the sampling kernel picks a token per row with the
draw of that row's stream position. Only token ids and an error word come back to the host.
This class is the step-by-step form (the histories' token counts are made on the host every
step); the steps that feed themselves on the device keep those counts on the device
(``engine/graphs.py``).
"""
from __future__ import annotations

import torch

from ..csrc import ops
from ..errors import SamplingError
from .options import SamplingOptions, splitmix64, unit_draw


class Sampler:
    def __init__(self, options: SamplingOptions, vocab_size: int, device):
        self.options = options.validate(vocab_size)
        self.vocab_size = vocab_size
        self.device = torch.device(device)
        self._err = torch.zeros(1, dtype=torch.int32, device=self.device)

    @property
    def native_ok(self) -> bool:
        """Whether the C++ decode loop that samples between graph launches can serve this sampler:
        everything but the adjustments (penalties, bias), which it does not know."""
        return not self.options.adjusts

    @property
    def fed_ok(self) -> bool:
        """Whether steps that pick their own token on the device can serve this sampler: all of
        them; adjustments ride along as token counts kept on the device."""
        return True

    @property
    def error_word(self) -> torch.Tensor:
        return self._err

    def _adjust_entries(self, histories: list):
        o = self.options
        entries, biases = [], []
        penalise = o.presence_penalty != 0.0 or o.frequency_penalty != 0.0 or o.repeat_penalty != 1.0
        for row, hist in enumerate(histories):
            counts: dict = {}
            if penalise:
                for t in hist:
                    if 0 <= t < self.vocab_size:
                        counts[t] = counts.get(t, 0) + 1
            bias: dict = {}
            for tok, b in o.logit_bias:
                bias[tok] = bias.get(tok, 0.0) + b
            for tok in set(counts) | set(bias):
                entries.append((row, tok, counts.get(tok, 0)))
                biases.append(bias.get(tok, 0.0))
        return entries, biases

    def sample(self, logits: torch.Tensor, histories: list) -> torch.Tensor:
        """``logits``: float32 [rows, vocab] on the device (adjusted in place when penalties or
        biases are set); ``histories``: per row the tokens so far, prompt included. Returns
        int32 [rows] on the device."""
        rows = logits.shape[0]
        o = self.options
        out = torch.empty(rows, dtype=torch.int32, device=self.device)
        if o.adjusts:
            entries, biases = self._adjust_entries(histories)
            if entries:
                e = torch.tensor(entries, dtype=torch.int32).to(self.device, non_blocking=True)
                b = torch.tensor(biases, dtype=torch.float32).to(self.device, non_blocking=True)
                ops.adjust_logits(logits, e, b, o.repeat_penalty, o.presence_penalty, o.frequency_penalty)
        if o.greedy:
            ops.argmax_rows(logits, out, self._err)
        else:
            seed = o.seed or 0
            draws = torch.tensor([unit_draw(seed, len(h)) for h in histories], dtype=torch.float32)
            draws = draws.to(self.device, non_blocking=True)
            ops.sample_rows(logits, o.temperature, o.top_k or 0, o.top_p if o.top_p is not None else 1.0,
                            o.min_p or 0.0, draws, out, self._err)
        return out

    def verify(self, logits: torch.Tensor, drafts: list, histories: list, draft_probs: list | None = None, row0: list | None = None) -> tuple:
        """Which drafted tokens stay, and the token behind them. ``logits``: float32 on the device, for every sequence a row for each
        of its ``drafts`` (a list of tokens) and one more, packed or from the rows ``row0`` on (adjusted in place when penalties or
        biases are set: then no row belongs to two); ``histories``: per sequence the tokens before its drafts; ``draft_probs``: per sequence the drafter's probabilities
        (float32 [drafts, vocabulary] on the device), or None where it was certain of its tokens. Returns (accepted drafts,
        next tokens), two lists. The draws come from the sampler's seed and the history's length: the next token's
        from the stream of ``sample``, the acceptances' from one of their own."""
        o = self.options
        n, room = len(drafts), max([len(d) for d in drafts] + [1])
        if row0 is None:
            row0, at = [], 0
            for d in drafts:
                row0.append(at)
                at += len(d) + 1
        rows = logits.shape[0]
        if len(histories) != n or len(row0) != n or any(not 0 <= r <= rows - len(d) - 1 for r, d in zip(row0, drafts)):
            raise SamplingError(f"{n} sequences with {sum(len(d) for d in drafts)} drafts do not fit {rows} rows of logits and "
                                f"{len(histories)} histories")
        if n == 0:
            return [], []
        if o.adjusts:
            # a row's history ends with the drafts before it; rows that no sequence names are left alone
            named = {r + j: list(h) + list(d[:j]) for r, h, d in zip(row0, histories, drafts) for j in range(len(d) + 1)}
            if len(named) < n + sum(len(d) for d in drafts):
                raise SamplingError("two sequences share rows of logits, which penalties and biases would adjust for one of them alone")
            entries, biases = self._adjust_entries(list(named.values()))
            if entries:
                at = list(named)
                e = torch.tensor([(at[r], t, c) for r, t, c in entries], dtype=torch.int32).to(self.device, non_blocking=True)
                b = torch.tensor(biases, dtype=torch.float32).to(self.device, non_blocking=True)
                ops.adjust_logits(logits, e, b, o.repeat_penalty, o.presence_penalty, o.frequency_penalty)
        seed = o.seed or 0
        own = splitmix64(seed ^ 0x5851F42D4C957F2D)                  # the acceptances' stream
        ints = torch.tensor([row0, [len(d) for d in drafts]], dtype=torch.int32).to(self.device, non_blocking=True)
        tokens = torch.tensor([list(d) + [0] * (room - len(d)) for d in drafts], dtype=torch.int32).to(self.device, non_blocking=True)
        accept = torch.tensor([[unit_draw(own, len(h) + j) for j in range(room)] for h in histories], dtype=torch.float32)
        accept = accept.to(self.device, non_blocking=True)
        draws = torch.tensor([unit_draw(seed, len(h)) for h in histories], dtype=torch.float32).to(self.device, non_blocking=True)
        probs = None
        if draft_probs is not None and any(p is not None for p in draft_probs):
            probs = torch.zeros((n, room, self.vocab_size), dtype=torch.float32, device=self.device)
            for i, (p, d) in enumerate(zip(draft_probs, drafts)):
                if p is not None:
                    if tuple(p.shape) != (len(d), self.vocab_size):
                        raise SamplingError(f"sequence {i}: {len(d)} drafts need probabilities [{len(d)}, {self.vocab_size}], got {list(p.shape)}")
                    probs[i, :len(d)] = p
                else:                                                # certain drafts among others with probabilities
                    for j, t in enumerate(d):
                        if 0 <= int(t) < self.vocab_size:            # (a token that is none is rejected and reported by the kernel)
                            probs[i, j, int(t)] = 1.0
        out = torch.empty((n, room + 2), dtype=torch.int32, device=self.device)
        counts, chosen = torch.empty(n, dtype=torch.int32, device=self.device), torch.empty((n, room + 1), dtype=torch.int32, device=self.device)
        scratch = torch.empty(ops.verify_bytes(rows, n, self.vocab_size), dtype=torch.uint8, device=self.device)
        ops.verify_drafts(logits, ints[0], ints[1], tokens, probs, accept, draws, o.temperature, o.top_k or 0,
                          o.top_p if o.top_p is not None else 1.0, o.min_p or 0.0, counts, chosen, self._err, scratch)
        out[:, 0], out[:, 1:] = counts, chosen
        host = out.tolist()
        return [r[0] for r in host], [r[1 + r[0]] for r in host]

    def check(self) -> None:
        """Synchronising read of the error word: non-finite logits are an error
        (src/inference.rs:5890-5907)."""
        code = int(self._err.item())
        if code:
            self._err.zero_()
            raise SamplingError("sampler logits contain a non-finite value" if code & 1
                                else "a drafted token is outside the vocabulary or its probabilities are none" if code & 4 else "sampler softmax produced an invalid normalisation sum")
