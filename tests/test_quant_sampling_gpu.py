"""Many samples of shared prompts over a cache in 4 or 8 bits."""

import pytest
import torch

from tests.test_quant_runner_gpu import attention_is
from zstep_b200.config import Qwen35Config
from zstep_b200.models.parallel_sampling import ParallelSampler
from zstep_b200.models.qwen35 import Qwen35Runner
from zstep_b200.models.weights import RandomWeights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", params=[4, 8])
def sampler(request):
    cfg = Qwen35Config(vocab_size=4096, num_hidden_layers=2, layer_types=("full_attention",) * 2, num_experts=16,
                       mtp_num_hidden_layers=0, name="attention-only")
    return ParallelSampler(Qwen35Runner(cfg, weights=RandomWeights(cfg, seed=4), max_seqs=16, max_prefill_tokens=256, num_pages=120,
                                        max_model_len=256, kv_bits=request.param), 3)


def start(s, lens=(70, 33), samples=5):
    g = torch.Generator().manual_seed(9)
    return s.start([torch.randint(0, 4096, (n,), generator=g).tolist() for n in lens], samples)


def test_a_step_attends_over_the_forks(sampler):
    """The last layer's attention of a verify step, called as any runner's, is that of what the pages hold."""
    s = sampler
    slots = start(s)
    g = torch.Generator().manual_seed(1)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for _ in range(3):
        drafts = [torch.randint(0, 4096, (3,), generator=g).tolist() for _ in slots]
        have = [len(s.tokens[x]) for x in slots]
        alone = s.logits(slots, drafts, shared=False)
        assert torch.equal(s.logits(slots, drafts), alone)
        attention_is_of_layer(s.r, 1, [x for x in slots for _ in range(4)], [n + j for n in have for j in range(4)])
        new = s.step(slots, 0.9, top_k=40, top_p=0.9, generator=gen, drafts=drafts)
        assert all(1 <= len(t) <= 4 for t in new) and [len(s.tokens[x]) for x in slots] == [a + len(t) for a, t in zip(have, new)]
        assert s.pool.seq_len[slots].tolist() == [len(s.tokens[x]) - 1 for x in slots]
    assert s.r.check_error() == 0 and s.plan is None
    s.finish(slots)


def attention_is_of_layer(r, layer, slots, lens):
    quant = r.quant

    class Layer:   # what `attention_is` reads, of one layer of several
        num_kv_heads = quant.num_kv_heads

        @staticmethod
        def read(_, *a, **kw):
            return quant.read(layer, *a, **kw)

    r.quant = Layer
    try:
        attention_is(r, len(slots), slots, lens)
    finally:
        r.quant = quant


def test_right_drafts_are_accepted_and_wrong_ones_taken_back(sampler):
    s = sampler
    slots = start(s)
    said = {x: [] for x in slots}
    for _ in range(8):
        for x, t in zip(slots, s.step(slots, 0.0, drafts=[[] for _ in slots])):
            assert len(t) == 1
            said[x] += t
    s.finish(slots)
    slots = start(s)
    assert s.step(slots, 0.0, drafts=[said[x][:3] for x in slots]) == [said[x][:4] for x in slots]
    wrong = [[said[x][4], (said[x][5] + 1) % 4096, said[x][6]] for x in slots]
    assert s.step(slots, 0.0, drafts=wrong) == [said[x][4:6] for x in slots]
    s.finish(slots)
    free = start(s, lens=(20,), samples=1)   # the prompts' pages went back with the next start
    s.finish(free)


def test_a_step_that_fails_adds_nothing(sampler):
    """What the device reports of a step's attention ends the step before a token is added, and is reported once."""
    s = sampler
    slots = start(s, lens=(20,), samples=2)
    before = [list(s.tokens[x]) for x in slots]
    s.step(slots, 0.0)
    mid = [list(s.tokens[x]) for x in slots]
    assert mid != before
    s.r.quant.err.fill_(3)
    with pytest.raises(RuntimeError, match="quantised cache"):
        s.step(slots, 0.0)
    assert [s.tokens[x] for x in slots] == mid
    s.step(slots, 0.0)
    s.finish(slots)
