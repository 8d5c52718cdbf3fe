"""Sampled speculative decoding: token probabilities and the verification of drafts.

``token_probs`` turns logits into the distribution a request samples from (temperature, top-k,
top-p with the sampling head's meaning of each); ``DraftVerifier`` accepts drafts against it from
given uniform numbers, so that the emitted tokens are samples of the target's distribution.
The arithmetic of the verification is fixed point (csrc/kernels/spec_sampling.cu has the
definition): given the probabilities and the numbers there is one right answer, and every
tensor-parallel rank finds it.
"""

from __future__ import annotations

import torch

from . import _ext

MAX_DRAFTS = 64


def token_probs(logits: torch.Tensor, temperature: torch.Tensor, top_k: torch.Tensor | None = None,
                top_p: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Probabilities [rows, vocab] (f32) of f32 logits with contiguous rows (any row stride).

    ``temperature`` [rows]: softmax(logits / T); T <= 0 puts all mass on the largest logit (the
    lowest id on ties).  ``top_k`` [rows] int32 keeps the k largest (0: off) and ``top_p`` [rows]
    the tokens in descending order while the mass before them is below p; ties with the last
    kept token are kept.  -inf and NaN logits are masked; a row without others gives zeros."""
    if out is None:
        out = torch.empty_like(logits, memory_format=torch.contiguous_format)
    _ext.load().token_probs(logits, temperature, top_k, top_p, out)
    return out


class DraftVerifier:
    """Verification of up to ``k`` drafts of up to ``n`` sequences over ``vocab`` tokens."""

    def __init__(self, n: int, k: int, vocab: int, device="cuda"):
        if n < 1 or not 1 <= k <= MAX_DRAFTS or not 1 <= vocab <= 1 << 24:
            raise ValueError(f"need n >= 1, 1 <= k <= {MAX_DRAFTS} and 1 <= vocab <= 2^24")
        self.C = _ext.load()
        self.n, self.k, self.vocab = n, k, vocab
        self.record = torch.empty(n, k + 2, dtype=torch.int32, device=device)
        self.err = torch.zeros(1, dtype=torch.int32, device=device)

    def verify(self, target: torch.Tensor, drafts: torch.Tensor, uniform: torch.Tensor,
               draft_probs: torch.Tensor | None = None, counts: torch.Tensor | None = None) -> torch.Tensor:
        """``target`` [n, k+1, vocab]: the target's probabilities after the last token and after
        each draft; ``drafts`` [n, k] int32; ``uniform`` [n, k+1] in [0, 1): one number per draft
        and, last, the one that draws the token behind the accepted drafts; ``draft_probs``
        [n, k, vocab]: what the drafts were drawn from (None: they were certain); ``counts`` [n]
        int32: drafts of each sequence (None: k).

        Returns int32 [n, k+2], the verifier's own buffer: 1 + accepted drafts, then those tokens
        and the drawn one, -1 after them (the record of a greedy verify step)."""
        n, k1, vocab = target.shape
        if n > self.n or k1 != self.k + 1 or vocab != self.vocab:
            raise ValueError(f"target [{n}, {k1}, {vocab}] does not fit a verifier of [{self.n}, {self.k + 1}, {self.vocab}]")
        record = self.record[:n]
        self.C.draft_verify(target, draft_probs, drafts, counts, uniform, record, self.err)
        return record

    def check(self) -> None:
        """Raise if a row since the last check had no mass to draw from (reads the error word)."""
        if int(self.err.item()):
            self.err.zero_()
            raise RuntimeError("draft verification: a row without any probability mass")
