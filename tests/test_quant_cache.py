"""What the quantised K/V cache refuses before anything reaches a GPU."""

import os
import subprocess

import pytest
import torch

from tests.test_tokenizer import build_hf_tokenizer
from zstep_b200.ops.quant_cache import QuantAttention, QuantCache

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("change,word", [(dict(bits=5), "bits"), (dict(bits=16), "bits"), (dict(head_dim=96), "head_dim"),
                                         (dict(page_size=24), "page_size"), (dict(page_size=8), "page_size"), (dict(layers=0), "positive"),
                                         (dict(num_pages=0), "positive"), (dict(num_kv_heads=0), "positive")])
def test_cache_forms(change, word):
    args = dict(layers=1, num_pages=4, num_kv_heads=2, head_dim=64, device="cpu")
    with pytest.raises(ValueError, match=word):
        QuantCache(**{**args, **change})


def test_bytes_of_a_value():
    """16 tokens of a head: the numbers, and 32 bits for 64 of them, of K and of V."""
    for dim in (64, 128, 256):
        for bits in (4, 8):
            for page in (16, 64):
                c = QuantCache(2, 3, 5, dim, bits=bits, page_size=page, device="cpu")
                assert c.page_bytes == 5 * page * 2 * (dim * bits // 8 + dim // 64 * 4)
                assert tuple(c.data.shape) == (2, 3, c.page_bytes)


@pytest.mark.parametrize("heads,rows,seqs,per", [(3, 1, 1, 1), (0, 1, 1, 1), (2, 0, 1, 1), (2, 1, 0, 1), (2, 1, 1, 0),
                                                 (2, 1 << 28, 1, 1), (2, 1, 1 << 24, 1), (2, 1 << 62, 1, 1)])
def test_plan_forms(heads, rows, seqs, per):
    with pytest.raises(ValueError):
        QuantAttention(QuantCache(1, 4, 2, 64, device="cpu"), heads, max_rows=rows, max_seqs=seqs, max_seq_rows=per)


def test_a_cache_on_the_cpu_is_not_run():
    cache = QuantCache(1, 4, 2, 64, device="cpu")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    table = torch.zeros(1, 2, dtype=torch.int32)
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA device"):
        cache.write(0, x, x, table, i32(0), i32(0))
    with pytest.raises(RuntimeError, match="CUDA device"):
        cache.read(0, table, i32(0), i32(0))
    with pytest.raises(ValueError, match="layer"):
        cache.write(1, x, x, table, i32(0), i32(0))
    plan = QuantAttention(cache, 2, 1)
    with pytest.raises(RuntimeError, match="CUDA device"):
        plan.update(i32(0), i32(1))
    with pytest.raises(RuntimeError, match="CUDA device"):
        plan.attend(0, x, table, 1.0)


@pytest.mark.parametrize("value,device", [("fp8", "cuda"), ("int2", "cuda"), ("int4", "cpu"), ("int8", "cpu")])
def test_command_line(value, device, tmp_path):
    build_hf_tokenizer(str(tmp_path))
    r = subprocess.run([os.path.join(ROOT, "zstep_b200", "bin", "zstep"), "run", "--mock", "--model-dir", str(tmp_path), "--device", device,
                        "--prompt-ids", "1", "--kv-cache-dtype", value], capture_output=True, text=True, timeout=60)
    assert r.returncode == 2 and "kv-cache-dtype" in r.stderr
