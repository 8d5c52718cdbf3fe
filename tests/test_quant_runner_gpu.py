"""The Qwen3.5 runner with its K/V cache in 4 or 8 bits, against its bf16 cache and against the 64-bit attention."""

import numpy as np
import pytest
import torch

from tests.test_quant_cache_gpu import quantised, reference
from zstep_b200.config import qwen35_small_gpu
from zstep_b200.models.qwen35 import Qwen35Runner
from zstep_b200.models.weights import RandomWeights
from zstep_b200.ops import mx
from zstep_b200.ops.kv_layout import unswizzle_pages
from zstep_b200.runtime.runners import GpuRunner

pytestmark = pytest.mark.gpu
LENS = [5, 17, 33]


def runner_of(cfg, bits, **kw):
    r = Qwen35Runner(cfg, weights=RandomWeights(cfg, seed=11), max_seqs=8, max_prefill_tokens=256, num_pages=64, max_model_len=256,
                     kv_bits=bits, **kw)
    for s in range(len(LENS)):
        r.set_pages(s, list(range(1 + 8 * s, 1 + 8 * (s + 1))))
    return r


def prefill(r, cfg):
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist() for n in LENS]
    ids = [t for p in prompts for t in p]
    pos = [i for n in LENS for i in range(n)]
    slots = [s for s, n in enumerate(LENS) for _ in range(n)]
    starts = [0] + list(np.cumsum(LENS))
    r.stage(ids, pos, slots, seq_start=starts)
    first = r.prefill_forward(len(ids), len(LENS)).cpu().tolist()
    assert r.check_error() == 0
    return first, slots, pos


def attention_is(r, rows, slots, lens):
    """The last attention layer's MXFP8 output against the 64-bit attention over what its cache holds."""
    D, hq = r.cfg.head_dim, r.hq
    q, gate = r.buf["q_out"][:rows], r.buf["gate_out"][:rows]
    want, tol = reference(r.quant, r.page_table, q, slots, lens, D ** -0.5, gate)
    # The layer's output projection read `midq`, `midsf`; nothing has written them since (the MoE has buffers of its own).
    got = mx.dequantize(r._mid(hq * D)[:rows], mx.codes_from_atoms(r.buf["midsf"], rows, hq * D)).double().cpu().numpy()
    # e4m3: half a step is 2^-4 of the value, or 2^-10 of the block's scale (at most its largest value) for subnormals.
    block = np.abs(want).reshape(rows, -1, 32).max(-1, keepdims=True).repeat(32, -1).reshape(rows, -1)
    assert np.all(np.abs(got - want) <= tol + 2.0 ** -4 * (np.abs(want) + tol) + 2.0 ** -9 * block)


@pytest.mark.parametrize("bits", [4, 8])
def test_prefill_and_decode(bits):
    cfg = qwen35_small_gpu(num_layers=4, vocab=8192, experts=32)   # layer 3 is the attention layer, and the last
    plain, r = runner_of(cfg, 16), runner_of(cfg, bits)
    assert plain.quant is None and [tuple(t.shape) for t in r.paged_caches()] == [(1, 64, r.quant.page_bytes)]
    _, slots, pos = prefill(plain, cfg)
    toks, _, _ = prefill(r, cfg)
    # Up to the attention layer both runners compute the same numbers: the cache holds those of bf16, quantised.
    idx = [(s, p) for s, p in zip(slots, pos)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    held = r.quant.read(0, r.page_table, i32(slots), i32(pos), dtype=torch.float32)
    for cache, got in zip((plain.k_cache, plain.v_cache), held):
        pages = unswizzle_pages(cache[0])                        # [pages, heads, 16, 256]
        raw = torch.stack([pages[int(plain.page_table[s, p // 16]), :, p % 16] for s, p in idx])
        want = quantised(raw, bits)[0]
        assert np.all(np.abs(got.double().cpu().numpy() - want) <= 2.0 ** -24 * np.abs(want))
    attention_is(r, len(slots), slots, [p + 1 for p in pos])
    # Decode steps: the graph's tokens are the eager step's, and the attention is that of the cache.
    for step in range(3):
        at = [n + step for n in LENS]
        state = (r.ssm_state.clone(), r.conv_state.clone())
        r.stage(toks, at, [0, 1, 2])
        eager = r.decode_forward(3).cpu().tolist()
        attention_is(r, 3, [0, 1, 2], [p + 1 for p in at])
        r.ssm_state.copy_(state[0])
        r.conv_state.copy_(state[1])
        r.stage(toks, at, [0, 1, 2])
        assert r.decode_step(3).cpu().tolist() == eager
        assert r.check_error() == 0
        toks = eager


def test_verify_rows_and_recorded_errors():
    """A verify-sized varlen step (its plan is the one of K + 1 rows) attends as rows one by one would."""
    cfg = qwen35_small_gpu(num_layers=4, vocab=8192, experts=32)
    r = runner_of(cfg, 4, num_spec_tokens=3)
    assert sorted(r.quant_plans) == [1, 4, 256]
    toks, _, _ = prefill(r, cfg)
    rows = [t + j for t in range(3) for j in range(4)]
    slots = [s for s in range(3) for _ in range(4)]
    pos = [n + j for n in LENS for j in range(4)]
    r.stage(rows, pos, slots, seq_start=[0, 4, 8, 12])
    r._layers(12, decode=False, num_seqs=3, max_seq_rows=4)
    attention_is(r, 12, slots, [p + 1 for p in pos])
    with pytest.raises(ValueError, match="sequence boundaries"):
        r._layers(12, decode=False)
    assert r.check_error() == 0
    r.stage([1], [10000], [0])   # a position that no page-table row reaches
    r.decode_forward(1)
    assert r.check_error() != 0


def test_what_reads_bf16_refuses():
    cfg = qwen35_small_gpu(num_layers=4, vocab=1024, experts=8)
    r = runner_of(cfg, 8)
    with pytest.raises(ValueError, match="bf16 cache"):
        r.prefix_plan = object()
    with pytest.raises(ValueError, match="bf16 cache"):
        with r.eager_plan(object()):
            pass
    with pytest.raises(ValueError, match="kv_bits"):
        Qwen35Runner(cfg, max_seqs=2, max_prefill_tokens=16, num_pages=8, max_model_len=32, kv_bits=5)
    GpuRunner.wrap(r)
