"""The runner's prefix plan and page table: what captured graphs hold of them, and whose rows a plan is for."""

from types import SimpleNamespace

import pytest
import torch

from zstep_b200.config import qwen35_small_gpu
from zstep_b200.models.qwen35 import Qwen35Runner
from zstep_b200.ops.shared_prefix import SharedPrefixPlan

gpu = pytest.mark.gpu


class HostRunner(Qwen35Runner):
    """The host side alone."""

    def __init__(self):
        self.dev = torch.device("cpu")
        self.graphs, self.spec, self.coll = {}, SimpleNamespace(g_graphs={}), None
        self.prefix_plan = None
        self.page_table = torch.zeros(3, 2, dtype=torch.int32)
        self.buf = {"err": torch.zeros(1, dtype=torch.int32)}


@pytest.fixture
def host(monkeypatch):
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    return HostRunner()


def plan_of(slots):
    return SimpleNamespace(rows=len(slots), err=torch.zeros(1, dtype=torch.int32), slot_list=list(slots))


def test_graphs_go_where_the_plan_or_the_page_table_changes(host):
    a, b = plan_of([0, 1]), plan_of([1, 0])
    for change in (lambda: setattr(host, "prefix_plan", a), lambda: setattr(host, "prefix_plan", b),
                   lambda: setattr(host, "prefix_plan", None), lambda: setattr(host, "page_table", host.page_table.clone())):
        host.graphs[2] = host.spec.g_graphs[2] = object()
        change()
        assert not host.graphs and not host.spec.g_graphs
    host.prefix_plan = a
    host.graphs[2] = object()
    host.prefix_plan = a                 # the same one
    with host.eager_plan(b):             # steps that replay no graph
        assert host.prefix_plan is b
    assert host.prefix_plan is a and host.graphs


def test_a_failed_plan_shows_in_the_runners_error(host):
    assert host.check_error() == 0
    host.prefix_plan = plan_of([0])
    assert host.check_error() == 0
    host.prefix_plan.err.fill_(3)
    assert host.check_error() == 3
    host.buf["err"].fill_(1)
    assert host.check_error() == 1


def test_rows_that_are_not_the_plans_are_refused(host):
    host.host_inputs, host._staged_rows = torch.zeros(4, 4, dtype=torch.int32), 3
    host.host_inputs[2] = torch.tensor([5, 0, 1, 9])
    host.check_plan_rows(4)
    host.prefix_plan = plan_of([5, 0, 1, 2])
    host.check_plan_rows(4)              # the fourth row is not staged: padding
    host.check_plan_rows(2)
    for slots in ([0, 5, 1, 2], [5, 0], [5, 0, 2, 1]):
        host.prefix_plan = plan_of(slots)
        with pytest.raises(ValueError, match="staged"):
            host.check_plan_rows(4)
    host.host_inputs[2, 2] = 2           # checked with every step
    host.check_plan_rows(4)


@pytest.fixture(scope="module")
def four():
    """Four sequences behind one 64-token prompt, each with its own pages, and their state."""
    r = Qwen35Runner(qwen35_small_gpu(num_layers=4, vocab=4096, experts=16), max_seqs=4, max_prefill_tokens=160, num_pages=64,
                     max_model_len=160)
    prompt = torch.randint(0, 4096, (64,), generator=torch.Generator().manual_seed(5)).tolist()
    for s in range(4):
        r.set_pages(s, [1, 2, 3, 4] + list(range(5 + 6 * s, 11 + 6 * s)))
    for s in range(4):
        r.stage(prompt, list(range(64)), [s] * 64, seq_start=[0, 64])
        r.prefill_forward(64, 1)
    torch.cuda.synchronize()
    return r, [t.clone() for t in (r.k_cache, r.v_cache, r.conv_state, r.ssm_state)]


def decode(four, steps=2):
    """Hidden states of some decode steps behind the prompt, one graph for all of them."""
    r, start = four
    for t, c in zip((r.k_cache, r.v_cache, r.conv_state, r.ssm_state), start):
        t.copy_(c)
    out = []
    for i in range(steps):
        r.stage([11 + s + 7 * i for s in range(4)], [64 + i] * 4, list(range(4)))
        r.decode_step(4)
        torch.cuda.synchronize()
        out.append(r.buf["hidden"][:4].float().clone())
    assert r.check_error() == 0
    return out


@gpu
def test_each_plan_is_the_one_that_runs(four):
    """None, one plan, another, none: no graph is cleared by hand, the plan that is set is the one that works."""
    r = four[0]
    slots = list(range(4))
    plans = [SharedPrefixPlan.from_prefixes(slots, groups, r.hq, r.hkv) for groups in ([(slots, 4)], [([0, 1], 3), ([2, 3], 4)])]
    first = decode(four)
    for plan in (plans[0], plans[1], None, plans[0]):
        for p in plans:
            p._partial.fill_(float("nan"))
        r.prefix_plan = plan
        for a, b in zip(first, decode(four)):
            torch.testing.assert_close(a, b, rtol=5e-2, atol=5e-2)
        assert [bool(p._partial.isnan().all()) for p in plans] == [p is not plan for p in plans]
    r.prefix_plan = None


@gpu
def test_a_batch_in_another_order_is_refused(four):
    """Before a graph of the plan is there, and when it is; the runner goes on with the right order."""
    r = four[0]
    first = decode(four)
    r.prefix_plan = SharedPrefixPlan.from_prefixes(list(range(4)), [([0, 1, 2, 3], 4)], r.hq, r.hkv)
    for _ in range(2):
        r.stage([11, 12, 13, 14], [64] * 4, [1, 0, 2, 3])
        with pytest.raises(ValueError, match="staged"):
            r.decode_step(4)
        for a, b in zip(first, decode(four)):
            torch.testing.assert_close(a, b, rtol=5e-2, atol=5e-2)
    r.stage([1], [66], [1], seq_start=[0, 1])
    with pytest.raises(ValueError, match="staged"):
        r.prefill_forward(1, 1)
    r.prefix_plan = None


@gpu
def test_a_new_page_table_is_the_one_that_is_read(four):
    r = four[0]
    first = decode(four)
    old = r.page_table
    r.page_table = old.clone()
    old.zero_()                          # every page the padding page
    for a, b in zip(first, decode(four)):
        assert torch.equal(a, b)
