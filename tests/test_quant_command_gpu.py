"""`zstep run --kv-cache-dtype int8|int4` end to end on a B200 worker."""

import pytest
import torch

from tests.test_e2e_gpu import PROMPTS, model_dir, zstep_run  # noqa: F401
from zstep_b200.config import qwen35_small_gpu
from zstep_b200.models.qwen35 import EPI_F32, Qwen35Runner
from zstep_b200.models.weights import RandomWeights

pytestmark = pytest.mark.gpu


def forced_logits(bits, prompt, tokens):
    """The logits that each token was chosen from, by one prefill of prompt and tokens: [tokens, vocab]."""
    cfg = qwen35_small_gpu()
    r = Qwen35Runner(cfg, weights=RandomWeights(cfg, seed=0), max_seqs=4, max_prefill_tokens=256, num_pages=64, max_model_len=256,
                     kv_bits=bits)
    r.set_pages(0, list(range(1, 17)))
    ids = prompt + tokens[:-1]
    r.stage(ids, list(range(len(ids))), [0] * len(ids), seq_start=[0, len(ids)])
    r._layers(len(ids), decode=False, num_seqs=1)
    out = torch.empty(len(ids), r.vocab_local, dtype=torch.float32, device=r.dev)
    r._gemm(r.lm_head, r.buf["xq"], r.buf["xsf"], len(ids), out, r.vocab_local, EPI_F32)
    assert r.check_error() == 0
    return out[len(prompt) - 1:]


@pytest.mark.parametrize("dtype", ["int8", "int4"])
def test_generation_over_a_quantised_cache(dtype, model_dir):  # noqa: F811
    """Greedy tokens of decode steps, and of verify steps with drafts, are the largest of the same model's logits, or as near
    to it as two ways of computing them may be apart: a logit is a sum over activations in e4m3, each off by up to 2^-4 of
    itself (2^-4 / 3^(1/2) in the root mean square), so by 0.036 of the logits' spread if every rounding falls the other way
    in the other kernel; twice that for the difference of two of them, four times that for the largest of many."""
    bits = {"int8": 8, "int4": 4}[dtype]
    for method in ("none", "mtp"):
        for p in PROMPTS:
            t = zstep_run(model_dir, "--kv-cache-dtype", dtype, "--prompt-ids", ",".join(map(str, p)), "--max-tokens", "16",
                          "--speculative-method", method)["tokens"]
            assert len(t) == 16
            x = forced_logits(bits, list(p), t)
            behind = x.amax(-1) - x.gather(1, torch.tensor(t, device=x.device)[:, None])[:, 0]
            assert bool((behind <= 8 * 0.036 * x.std(-1)).all()), (method, p, behind.tolist())


@pytest.mark.parametrize("dtype", ["int8", "int4"])
def test_mixed_steps_over_a_quantised_cache(dtype, model_dir):  # noqa: F811
    """Requests of a shared prefix that are admitted while others decode, with prefix caching and drafts."""
    rep = zstep_run(model_dir, "--kv-cache-dtype", dtype, "--speculative-method", "mtp", "--bench-tiers", "mtp:4:8:32:16:64:2")
    run0 = rep["tiers"][0]["runs"][0]
    assert run0["output_tok_s"] > 0 and run0["shared_prefix_len"] == 64 and run0["mean_acceptance_length"] >= 1.0
