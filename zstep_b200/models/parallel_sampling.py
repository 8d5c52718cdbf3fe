"""Many samples of a few prompts, with speculation, on one runner of an attention-only model.

Each prompt is prefilled once; its samples are forks that share the prompt's pages.  A step feeds
every sample its last token and up to K drafts (prompt lookup: what followed the last occurrence
of the newest tokens), reads each prompt's pages once for all of its samples, turns the logits
into the distribution that the samples draw from, accepts drafts against it and takes rejected
rows back.  Finished samples give their pages back and the pool is packed.

    python -m zstep_b200.models.parallel_sampling --prompts 4 --samples 8 --tokens 64

runs it on random weights and prints the tokens per step.
"""

from __future__ import annotations

import argparse
import json

import torch

from ..ops.pages import PagePool
from ..ops.shared_prefix import SharedPrefixPlan
from ..ops.spec_sampling import MAX_DRAFTS, DraftVerifier, token_probs
from .qwen35 import EPI_F32, Qwen35Runner


def prompt_lookup(tokens: list[int], k: int, window: int = 3) -> list[int]:
    """Up to k tokens that followed the latest earlier occurrence of the longest suffix (window..1 tokens)."""
    for n in range(min(window, len(tokens) - 1), 0, -1):
        suffix = tokens[-n:]
        for i in range(len(tokens) - n - 1, -1, -1):
            if tokens[i:i + n] == suffix:
                return tokens[i + n:i + n + k]
    return []


class ParallelSampler:
    """``runner``: one of an attention-only model.  Over a quantised cache (``kv_bits`` 8 or 4) samples share their
    prompt's pages too, but every sample's rows read them for themselves."""

    def __init__(self, runner: Qwen35Runner, num_drafts: int = 3):
        if runner.cfg.gdn_layers:
            raise ValueError("forks copy pages, not recurrent state: the model must have attention layers only")
        if runner.tp != 1:
            raise ValueError("one rank only")
        if not 1 <= num_drafts <= MAX_DRAFTS:
            raise ValueError(f"num_drafts must be at least 1 and at most {MAX_DRAFTS}")
        self.r, self.k = runner, num_drafts
        self.pool = PagePool(runner.paged_caches(), runner.num_slots, runner.max_pages, runner.page_size)
        runner.page_table = self.pool.page_table
        # Padding rows of a step point at the dummy slot, whose table row stays at the padding page.
        self.tokens: dict[int, list[int]] = {}   # sample slot -> prompt and generated tokens
        self.prompt_of: dict[int, int] = {}      # sample slot -> its prompt's slot
        self.prompt_pages: dict[int, int] = {}   # prompt slot -> pages that its samples share
        self.plan = self.verifier = self._plan_key = None   # of the first step on (no plan over a quantised cache)

    def _ints(self, x) -> torch.Tensor:
        return torch.tensor(x, dtype=torch.int32, device=self.r.dev)

    def _current(self) -> None:
        if self.r.page_table is not self.pool.page_table:
            raise RuntimeError("the runner's page table is no longer this sampler's: one sampler at a time")

    def _known(self, tokens: list[list[int]]) -> None:
        vocab = self.r.cfg.vocab_size
        if any(not 0 <= t < vocab for x in tokens for t in x):
            raise ValueError(f"a token outside the vocabulary of {vocab}")

    def start(self, prompts: list[list[int]], samples: int) -> list[int]:
        """Prefill each prompt into a slot and fork it into ``samples`` sample slots; returns those slots.
        Samples of earlier calls go on.  A prompt's slot and pages are kept until the first call
        after its last sample has ended."""
        r, n = self.r, len(prompts)
        self._current()
        living = {self.prompt_of[s] for s in self.tokens}
        taken = living | set(self.tokens)
        free = [s for s in range(r.max_seqs) if s not in taken]
        if n * (samples + 1) > len(free):
            raise ValueError(f"{n} prompts x {samples} samples need {n * (samples + 1)} of {len(free)} slots")
        if any(not p for p in prompts):
            raise ValueError("a prompt needs at least one token")
        if max(map(len, prompts), default=0) > r.max_pages * r.page_size:
            raise ValueError(f"a prompt passes the {r.max_pages * r.page_size} tokens of a sequence")
        if sum(len(p) - 1 for p in prompts) > r.R:
            raise ValueError(f"the prompts pass the {r.R} rows of a step")
        self._known(prompts)
        ended = [p for p in self.prompt_pages if p not in living]
        self.pool.free(self._ints(ended))
        for p in ended:
            del self.prompt_pages[p]
        parents, kids = free[:n], free[n:n * (samples + 1)]
        # The last prompt token is the first step's input: its row comes with the drafts.
        ids = [t for p in prompts for t in p[:-1]]
        pos = [i for p in prompts for i in range(len(p) - 1)]
        slots = [s for s, p in zip(parents, prompts) for _ in p[:-1]]
        self.pool.extend(self._ints(parents), self._ints([len(p) - 1 for p in prompts]))
        self.pool.check()   # short of pages, no slot has grown
        starts = [0]
        for p in prompts:
            starts.append(starts[-1] + len(p) - 1)
        if ids:
            r.stage(ids, pos, slots, seq_start=starts)
            with r.eager_plan(None):
                r._layers(len(ids), decode=False, num_seqs=n)
        parent = [s for s in parents for _ in range(samples)]
        self.pool.fork(self._ints(parent), self._ints(kids))
        try:
            self.pool.check()
        except RuntimeError:
            self.pool.free(self._ints(parents))
            raise
        for s, p in zip(parents, prompts):
            self.prompt_pages[s] = (len(p) - 1) // r.page_size
        for i, (s, p) in enumerate(zip(kids, parent)):
            self.tokens[s] = list(prompts[i // samples])
            self.prompt_of[s] = p
        return kids

    def _plan(self, slots: list[int]) -> SharedPrefixPlan | None:
        """Who shares what: changes only when samples end or start.  None where the cache is quantised."""
        key = tuple((s, self.prompt_of[s], self.prompt_pages[self.prompt_of[s]]) for s in slots)
        if self._plan_key != key:
            if self.r.kv_bits == 16:
                rows = [s for s in slots for _ in range(self.k + 1)]
                groups: dict[int, list[int]] = {}
                for i, s in enumerate(rows):
                    groups.setdefault(self.prompt_of[s], []).append(i)
                prefixes = [(members, self.prompt_pages[p]) for p, members in groups.items()]
                self.plan = SharedPrefixPlan.from_prefixes(rows, prefixes, self.r.hq, self.r.hkv, device=self.r.dev)
            self.verifier = DraftVerifier(len(slots), self.k, self.r.cfg.vocab_size, device=self.r.dev)
            self._plan_key = key
        return self.plan

    def _check_attention(self) -> None:
        parts = [self.plan] if self.plan is not None else [] if self.r.quant is None else [self.r.quant, *self.r.quant_plans.values()]
        for x in parts:
            x.check()

    def logits(self, slots: list[int], drafts: list[list[int]], shared: bool = True) -> torch.Tensor:
        """f32 logits [len(slots), k + 1, vocab] after the newest token of each sample and after each of its
        drafts (missing drafts are padded with token 0).  ``shared`` False: every sample's rows read the prompt's
        pages for themselves."""
        r, k1, n = self.r, self.k + 1, len(slots)
        self._current()
        if len(drafts) != n or any(len(d) > self.k for d in drafts):
            raise ValueError(f"drafts must be one list of up to {self.k} tokens for each sample")
        if n * k1 > r.R:
            raise ValueError(f"{n} samples x {k1} rows pass the {r.R} rows of a step")
        if max((len(self.tokens[s]) for s in slots), default=0) + self.k > r.max_pages * r.page_size:
            raise ValueError(f"a sample and its drafts pass the {r.max_pages * r.page_size} tokens of a sequence")
        self._known(drafts)
        ids, pos, rows = [], [], []
        for s, d in zip(slots, drafts):
            have = len(self.tokens[s]) - 1   # cached tokens
            ids += [self.tokens[s][-1]] + d + [0] * (self.k - len(d))
            pos += list(range(have, have + k1))
            rows += [s] * k1
        plan = self._plan(slots) if shared else None
        self.pool.extend(self._ints(slots), self._ints([len(self.tokens[s]) + self.k for s in slots]))
        self.pool.check()   # short of pages, no slot has grown, and rows would have nowhere to go
        r.stage(ids, pos, rows, seq_start=[i * k1 for i in range(n + 1)])
        with r.eager_plan(plan):
            r._layers(n * k1, decode=False, num_seqs=n)
        out = torch.empty(n * k1, r.vocab_local, dtype=torch.float32, device=r.dev)
        r._gemm(r.lm_head, r.buf["xq"], r.buf["xsf"], n * k1, out, r.vocab_local, EPI_F32)
        return out.view(n, k1, r.vocab_local)

    def step(self, slots: list[int], temperature: float, top_k: int = 0, top_p: float = 1.0,
             generator: torch.Generator | None = None, drafts: list[list[int]] | None = None) -> list[list[int]]:
        """One verify step; appends to and returns the new tokens of each sample.  A step that fails (short
        of pages, past a sequence's end) adds nothing: it can be tried again when samples have ended."""
        n, k1 = len(slots), self.k + 1
        if drafts is None:
            drafts = [prompt_lookup(self.tokens[s], self.k) for s in slots]
        logits = self.logits(slots, drafts)
        rows = n * k1
        dev = self.r.dev
        probs = token_probs(logits.view(rows, -1), torch.full((rows,), temperature, device=dev),
                            torch.full((rows,), top_k, dtype=torch.int32, device=dev) if top_k else None,
                            torch.full((rows,), top_p, device=dev) if top_p < 1.0 else None)
        record = self.verifier.verify(probs.view(n, k1, -1), self._ints([d + [0] * (self.k - len(d)) for d in drafts]),
                                      torch.rand(n, k1, generator=generator, device=dev),
                                      counts=self._ints([len(d) for d in drafts])).tolist()
        self.verifier.check()
        self._check_attention()
        new = [rec[1:1 + rec[0]] for rec in record]
        for s, t in zip(slots, new):
            self.tokens[s] += t
        # Cached: everything but the newest token; the rows of rejected drafts go.
        self.pool.truncate(self._ints(slots), self._ints([len(self.tokens[s]) - 1 for s in slots]))
        return new

    def finish(self, slots: list[int]) -> list[list[int]]:
        """End samples: their pages go back and the live ones move together.  Returns their tokens."""
        if len(set(slots)) != len(slots) or any(s not in self.tokens for s in slots):
            raise ValueError(f"not all of {slots} are samples, each once")
        self._check_attention()
        if self.verifier is not None:
            self.verifier.check()
        self.pool.free(self._ints(slots))
        self.pool.compact()
        self.pool.check()
        for s in slots:
            del self.prompt_of[s]
        return [self.tokens.pop(s) for s in slots]


def main(argv: list[str] | None = None) -> None:
    from ..config import Qwen35Config

    ap = argparse.ArgumentParser()
    ap.add_argument("--prompts", type=int, default=4)
    ap.add_argument("--samples", type=int, default=8)
    ap.add_argument("--prompt-len", type=int, default=1000)
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--drafts", type=int, default=3)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--temperature", type=float, default=0.8)
    ap.add_argument("--top-k", type=int, default=50)
    ap.add_argument("--top-p", type=float, default=0.95)
    a = ap.parse_args(argv)
    if min(a.prompts, a.samples, a.prompt_len, a.tokens, a.drafts, a.layers) < 1:
        ap.error("prompts, samples, prompt-len, tokens, drafts and layers must be at least 1")
    cfg = Qwen35Config(vocab_size=8192, num_hidden_layers=a.layers, layer_types=("full_attention",) * a.layers,
                       num_experts=32, name="attention-only")
    seqs = a.prompts * (a.samples + 1)
    length = a.prompt_len + a.tokens + a.drafts + 1
    runner = Qwen35Runner(cfg, max_seqs=seqs, max_prefill_tokens=max(a.prompts * a.prompt_len, seqs * (a.drafts + 1)),
                          num_pages=a.prompts * (a.prompt_len // 16 + 2) + seqs * ((a.tokens + a.drafts) // 16 + 3) + 1,
                          max_model_len=length)
    gen = torch.Generator(device=runner.dev).manual_seed(0)
    prompts = torch.randint(0, cfg.vocab_size, (a.prompts, a.prompt_len), generator=gen, device=runner.dev).tolist()
    sampler = ParallelSampler(runner, a.drafts)
    slots = sampler.start(prompts, a.samples)
    steps = made = pages = 0
    while slots:
        sampler.step(slots, a.temperature, a.top_k, a.top_p, gen)
        steps += 1
        done = [s for s in slots if len(sampler.tokens[s]) >= a.prompt_len + a.tokens]
        if done:
            pages = max(pages, int((sampler.pool.refcount > 0).sum()))
            made += sum(len(t) - a.prompt_len for t in sampler.finish(done))
            slots = [s for s in slots if s in sampler.tokens]
    print(json.dumps({"samples": a.prompts * a.samples, "steps": steps, "tokens": made, "tokens_per_step": round(made / steps, 2),
                      "pages_in_use": pages, "pages_without_sharing": a.prompts * a.samples * -(-length // 16)}))


if __name__ == "__main__":
    main()
