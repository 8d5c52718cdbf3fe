"""Many samples of shared prompts through the runner: attention of the shared-prefix path against
the per-row path, right drafts accepted and wrong ones taken back, pages returned."""

import json

import pytest
import torch

from zstep_b200.config import Qwen35Config, qwen35_small_gpu
from zstep_b200.ops import mx
from zstep_b200.models.parallel_sampling import ParallelSampler, main, prompt_lookup

PAGE = 16


def test_prompt_lookup():
    assert prompt_lookup([1, 2, 3, 9, 1, 2, 3], 2) == [9, 1]
    assert prompt_lookup([5, 6, 5], 3) == [6, 5]
    assert prompt_lookup([1, 2, 3], 3) == []
    assert prompt_lookup([7], 3) == []


@pytest.fixture(scope="module")
def runner():
    from zstep_b200.models.qwen35 import Qwen35Runner
    from zstep_b200.models.weights import RandomWeights

    cfg = Qwen35Config(vocab_size=4096, num_hidden_layers=2, layer_types=("full_attention",) * 2, num_experts=16,
                       mtp_num_hidden_layers=0, name="attention-only")
    return Qwen35Runner(cfg, weights=RandomWeights(cfg, seed=4), max_seqs=16, max_prefill_tokens=256, num_pages=120,
                        max_model_len=256)


def _start(runner, lens=(70, 33), samples=5, k=3):
    g = torch.Generator().manual_seed(9)
    s = ParallelSampler(runner, k)
    prompts = [torch.randint(0, 4096, (n,), generator=g).tolist() for n in lens]
    return s, s.start(prompts, samples)


def _first_attention(s, slots, drafts, shared):
    """The first layer's attention output as its projection gets it (MXFP8), in 32 bits."""
    r, calls = s.r, []
    real = r._proj_out

    def spy(w, xq, xsf, rows, *a, **kw):
        if not calls:
            calls.append(mx.dequantize(xq[:rows].clone(), mx.codes_from_atoms(xsf.clone(), rows, xq.shape[1])))
        return real(w, xq, xsf, rows, *a, **kw)

    r._proj_out = spy
    try:
        s.logits(slots, drafts, shared)
    finally:
        r._proj_out = real
    return calls[0].double()


def _same_attention(s, slots, drafts):
    """Both paths get the same q, K and V in the first layer.  Each output is within 2^-8 (A + 2 |y|) of
    the true one (bf16 weights and outputs; A <= max |v|, the gate is below 1), then within 2^-4 of itself
    or half the smallest step of e4m3 under its block's scale (2^-10 * 2 amax / 448)."""
    a, b = (_first_attention(s, slots, drafts, x) for x in (True, False))
    vmax = float(s.r.v_cache[0].abs().max())
    amax = b.abs().view(b.shape[0], -1, 32).amax(-1, keepdim=True).expand(-1, -1, 32).reshape(b.shape)
    tol = 2 * (2.0 ** -8 * (vmax + 2 * b.abs()) + 2.0 ** -4 * b.abs() + 2.0 ** -10 * 2 * amax / 448)
    assert b.abs().max() > 0 and ((a - b).abs() <= tol).all()
    # and on the whole far nearer than that
    assert float((a - b).norm() / b.norm()) < 2.0 ** -4


@pytest.mark.gpu
def test_attention_equals_the_unshared_path(runner):
    s, slots = _start(runner)
    g = torch.Generator().manual_seed(1)
    for _ in range(3):
        drafts = [torch.randint(0, 4096, (3,), generator=g).tolist() for _ in slots]
        _same_attention(s, slots, drafts)
        s.step(slots, 0.9, top_k=40, top_p=0.9, drafts=drafts)
    assert runner.check_error() == 0
    s.finish(slots)


@pytest.mark.gpu
def test_right_drafts_are_accepted_and_wrong_ones_taken_back(runner):
    """Greedy: drafting what the model itself said is accepted whole; a wrong draft ends the row there."""
    s, slots = _start(runner)
    said = {x: [] for x in slots}
    for _ in range(8):   # no drafts: one token a step
        for x, t in zip(slots, s.step(slots, 0.0, drafts=[[] for _ in slots])):
            assert len(t) == 1
            said[x] += t
    by_prompt = {}
    for x in slots:      # samples of one prompt say the same
        assert by_prompt.setdefault(s.prompt_of[x], said[x]) == said[x]
    s.finish(slots)
    s, slots = _start(runner)
    new = s.step(slots, 0.0, drafts=[said[x][:3] for x in slots])
    assert new == [said[x][:4] for x in slots]
    wrong = [[said[x][4], (said[x][5] + 1) % 4096, said[x][6]] for x in slots]
    new = s.step(slots, 0.0, drafts=wrong)
    assert new == [said[x][4:6] for x in slots]
    assert s.pool.seq_len[slots].tolist() == [len(s.tokens[x]) - 1 for x in slots]
    s.finish(slots)


@pytest.mark.gpu
def test_ends_free_what_only_they_used(runner):
    s, slots = _start(runner, samples=4)
    gen = torch.Generator(device="cuda").manual_seed(3)
    for _ in range(5):
        s.step(slots, 1.1, generator=gen)
    half = slots[::2]
    left = [x for x in slots if x not in half]
    done = s.finish(half)
    assert all(len(t) >= 33 + 5 for t in done)
    for _ in range(3):   # the others go on over moved pages
        _same_attention(s, left, [[1, 2, 3] for _ in left])
        s.step(left, 1.1, generator=gen)
    s.finish(left)
    live = s.pool.refcount > 0   # packed: what the prompts hold
    assert bool(live[:int(live.sum())].all()) and int(live.sum()) == 1 + 5 + 2
    s.pool.free(torch.tensor([0, 1], dtype=torch.int32, device="cuda"))
    s.pool.check()
    assert s.pool.refcount.tolist() == [1] + [0] * (s.pool.num_pages - 1)


def _prompts(lens, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 4096, (n,), generator=g).tolist() for n in lens]


def _own_pages(s, slots):
    """What every sample writes to next is its own page."""
    table, lens, ref = s.pool.page_table.tolist(), s.pool.seq_len.tolist(), s.pool.refcount.tolist()
    for x in slots:
        assert lens[x] == len(s.tokens[x]) - 1
        if lens[x] % PAGE:
            assert ref[table[x][lens[x] // PAGE]] == 1


@pytest.mark.gpu
def test_a_sampler_starts_again(runner):
    """Shorter, longer and regrouped prompts in the slots of earlier ones say what a new sampler says."""
    s, slots = _start(runner, lens=(150, 40), samples=3)
    s.step(slots, 0.0)
    s.finish(slots)
    for seed, (lens, samples) in enumerate([((60, 40), 3), ((60, 90), 3), ((33, 20, 47), 2)]):
        prompts = _prompts(lens, seed)
        slots = s.start(prompts, samples)
        assert s.pool.seq_len[slots].tolist() == [n - 1 for n in lens for _ in range(samples)]
        drafts = [[1, 2, 3] for _ in slots]
        _same_attention(s, slots, drafts)
        said = {x: [] for x in slots}
        for _ in range(4):
            for x, t in zip(slots, s.step(slots, 0.0)):
                said[x] += t
            _own_pages(s, slots)
        new = ParallelSampler(runner, 3)
        again = new.start(prompts, samples)
        for _ in range(4):
            new.step(again, 0.0)
        assert [said[x] for x in slots] == [new.tokens[x][n:] for x, n in zip(again, (n for n in lens for _ in range(samples)))]
        new.finish(again)
        runner.page_table = s.pool.page_table
        s.finish(slots)
    assert s.start([], 1) == []          # nothing but what ended is given back
    assert s.pool.refcount.tolist() == [1] + [0] * (s.pool.num_pages - 1)


@pytest.mark.gpu
def test_samples_go_on_while_others_start(runner):
    s, first = _start(runner, lens=(70,), samples=4)
    for _ in range(2):
        s.step(first, 0.0)
    second = s.start(_prompts((33, 50), 4), 2)
    assert not set(first) & set(second) and len(set(second)) == 4
    with pytest.raises(ValueError, match="slots"):
        s.start(_prompts((10,), 5), 5)   # 11 of 16 slots are taken
    both = first + second
    _same_attention(s, both, [[4, 5, 6] for _ in both])
    for _ in range(3):
        s.step(both, 0.0)
        _own_pages(s, both)
    assert all(s.tokens[x] == s.tokens[first[0]] for x in first)
    s.finish(first)
    third = s.start(_prompts((20,), 6), 4)
    assert not set(third) & set(second)
    s.step(third + second, 0.0)
    s.finish(third + second)


@pytest.mark.gpu
def test_a_step_that_pages_run_short_for_adds_nothing():
    """39 pages: prompts of 8 each, 12 samples that need a page each with the first step."""
    from zstep_b200.models.qwen35 import Qwen35Runner

    cfg = Qwen35Config(vocab_size=4096, num_hidden_layers=2, layer_types=("full_attention",) * 2, num_experts=16,
                       mtp_num_hidden_layers=0, name="attention-only")
    s = ParallelSampler(Qwen35Runner(cfg, max_seqs=16, max_prefill_tokens=256, num_pages=40, max_model_len=256), 3)
    prompts = _prompts((129, 129), 7)

    def steps(slots, n):
        for _ in range(n):
            s.step(slots, 0.0, drafts=[[] for _ in slots])

    slots = s.start(prompts, 6)
    steps(slots, 6)
    want = [s.tokens[x] for x in slots]
    s.finish(slots)
    slots = s.start(prompts, 6)
    hog = torch.tensor([s.pool.num_slots - 1], dtype=torch.int32, device="cuda")   # no request's slot takes 16 of 23
    s.pool.extend(hog, torch.full_like(hog, 256))
    s.pool.check()
    state = s.pool.state.clone()
    short = pytest.raises(RuntimeError, match="few free pages")
    for _ in range(2):
        with short:
            steps(slots, 1)
        assert [s.tokens[x] for x in slots] == [p for p in prompts for _ in range(6)]
        assert torch.equal(state, s.pool.state)
    for n in (130, 98):   # 9 pages; the last 7, and then a copy of the last one
        with short:
            s.start(_prompts((n,), 8), 1)
        assert torch.equal(state, s.pool.state) and len(s.prompt_pages) == 2
    s.finish(slots[:3] + slots[6:9])
    left = slots[3:6] + slots[9:]
    steps(left, 6)        # six pages: enough for these, as if nothing had been
    assert [s.tokens[x] for x in left] == want[3:6] + want[9:]
    s.finish(left)


@pytest.mark.gpu
def test_a_sample_ends_at_its_table_rows_end(runner):
    s = ParallelSampler(runner, 3)
    slots = s.start(_prompts((252,), 9), 2) + s.start(_prompts((20,), 10), 2)   # 256 tokens a sequence
    for _ in range(2):                   # the second one's last draft row is the last of all
        s.step(slots, 0.0, drafts=[[] for _ in slots])
    table = s.pool.page_table.clone()
    with pytest.raises(ValueError, match="256 tokens"):
        s.step(slots, 0.0, drafts=[[] for _ in slots])
    with pytest.raises(ValueError, match="256 tokens"):
        s.logits(slots[:1], [[]])
    assert torch.equal(table, s.pool.page_table) and len(s.tokens[slots[0]]) == 254
    s.finish(slots[:2])
    s.step(slots[2:], 0.0)
    s.finish(slots[2:])


@pytest.mark.gpu
def test_what_a_step_cannot_take_is_refused(runner):
    s, slots = _start(runner)
    state = s.pool.state.clone()
    for drafts in ([[1]], [[1, 2, 3, 4]] * len(slots), [[4096]] * len(slots), [[-1]] * len(slots)):
        with pytest.raises(ValueError):
            s.step(slots, 0.0, drafts=drafts)
    for prompts in ([[]], [[1, 4096]], [[-1, 2]], [[1] * 257], [[1] * 200, [2] * 200]):
        with pytest.raises(ValueError):
            s.start(prompts, 1)
    with pytest.raises(RuntimeError, match="cannot serve"):   # one sample twice
        s.step(slots[:1] * 2, 0.0)
    assert torch.equal(state, s.pool.state)
    s.step(slots, 0.0)
    s.finish(slots)


@pytest.mark.gpu
def test_steps_that_cannot_be_planned_change_nothing(runner, monkeypatch):
    with pytest.raises(ValueError, match="64"):
        ParallelSampler(runner, 65)
    s, slots = _start(runner, k=64, samples=2)
    assert len(s.step(slots[2:3], 0.0, drafts=[[1] * 64])) == 1   # 64 drafts
    monkeypatch.setattr("zstep_b200.ops.shared_prefix.MAX_SEGS", 2)
    state = s.pool.state.clone()
    with pytest.raises(ValueError, match="at most 2 segments"):
        s.step(slots[:3], 0.0)
    assert torch.equal(state, s.pool.state)
    s.finish(slots)


@pytest.mark.gpu
def test_samples_end_before_any_step(runner):
    s, slots = _start(runner)
    state = s.pool.state.clone()
    for wrong in ([0], [slots[0]] * 2, [slots[0], 15]):   # a prompt's slot, one twice, none
        with pytest.raises(ValueError, match="samples"):
            s.finish(wrong)
    assert torch.equal(state, s.pool.state)
    assert [len(t) for t in s.finish(slots)] == [70] * 5 + [33] * 5
    assert not s.tokens and s.finish([]) == []


@pytest.mark.gpu
def test_a_sampler_whose_runner_has_another_is_refused(runner):
    s, slots = _start(runner)
    new, others = _start(runner)
    for call in (lambda: s.step(slots, 0.0), lambda: s.logits(slots, [[] for _ in slots]), lambda: s.start([[1, 2]], 1)):
        with pytest.raises(RuntimeError, match="one sampler"):
            call()
    new.step(others, 0.0)
    new.finish(others)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,temperature", [(1, 0.8), (3, 0.0), (40, 0.0)])
def test_the_command_ends_every_sample_at_its_length(tokens, temperature, capsys):
    """Fewer tokens than drafts, and greedy samples of which some run ahead by accepted drafts."""
    main(["--prompts", "2", "--samples", "2", "--prompt-len", "40", "--tokens", str(tokens), "--layers", "1",
          "--temperature", str(temperature)])
    said = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert said["samples"] == 4 and 1 <= said["steps"] <= tokens
    assert 4 * tokens <= said["tokens"] <= 4 * (tokens + 3)


def test_the_command_refuses_sizes(capsys):
    for name in ("prompts", "samples", "prompt-len", "tokens", "drafts", "layers"):
        with pytest.raises(SystemExit):
            main([f"--{name}", "0"])


@pytest.mark.gpu
def test_refusals(runner):
    from zstep_b200.models.qwen35 import Qwen35Runner

    hybrid = Qwen35Runner(qwen35_small_gpu(4, 1024, 8), max_seqs=2, max_prefill_tokens=16, num_pages=8, max_model_len=32)
    with pytest.raises(ValueError, match="attention layers"):
        ParallelSampler(hybrid)
    with pytest.raises(ValueError, match="num_drafts"):
        ParallelSampler(runner, 0)
    with pytest.raises(ValueError, match="slots"):
        _start(runner, samples=8)


@pytest.mark.gpu
def test_decode_graph_with_a_prefix_plan():
    """A decode step captured with a plan replays while the sequences grow."""
    from zstep_b200.models.qwen35 import Qwen35Runner
    from zstep_b200.ops.shared_prefix import SharedPrefixPlan

    cfg = qwen35_small_gpu(num_layers=4, vocab=4096, experts=16)
    r = Qwen35Runner(cfg, max_seqs=4, max_prefill_tokens=160, num_pages=64, max_model_len=160)
    prompt = torch.randint(0, 4096, (64,), generator=torch.Generator().manual_seed(2)).tolist()
    for s in range(4):   # the prompt's four pages once, then own pages; every slot runs its own recurrent state
        r.set_pages(s, [1, 2, 3, 4] + list(range(5 + 6 * s, 11 + 6 * s)))
    for s in range(4):
        r.stage(prompt, list(range(64)), [s] * 64, seq_start=[0, 64])
        r.prefill_forward(64, 1)
    k, v, conv, ssm = (t.clone() for t in (r.k_cache, r.v_cache, r.conv_state, r.ssm_state))
    outs = []
    for plan in (None, SharedPrefixPlan.from_prefixes(list(range(4)), [(list(range(4)), 4)], r.hq, r.hkv)):
        for t, c in zip((r.k_cache, r.v_cache, r.conv_state, r.ssm_state), (k, v, conv, ssm)):
            t.copy_(c)
        r.prefix_plan = plan
        r.graphs.clear()
        hidden = []
        for i in range(3):
            r.stage([11 + s + 7 * i for s in range(4)], [64 + i] * 4, list(range(4)))
            r.decode_step(4)
            torch.cuda.synchronize()   # the next step's inputs go through the same pinned block
            hidden.append(r.buf["hidden"][:4].float().clone())
        outs.append(hidden)
    assert r.check_error() == 0
    plan.check()
    for a, b in zip(*outs):
        torch.testing.assert_close(a, b, rtol=5e-2, atol=5e-2)
