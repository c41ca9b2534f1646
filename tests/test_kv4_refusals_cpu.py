"""More refusals of the 4-bit KV cache's entry points that need no device."""
import subprocess
import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

import ecq_b200 as ecq  # noqa: E402


def i32(*s):
    return torch.zeros(*s, dtype=torch.int32)


@pytest.mark.parametrize("n", [-1, 2 ** 31, 2 ** 32 + 1])
def test_counts_that_are_no_32_bit_integers(n):
    # ctypes takes 2^32 + 1 for 1
    rows, pages = torch.zeros(1, 1, 64, dtype=torch.float16), ecq.kv4_pages(2, 1, 64, page_size=16, group_size=32, device="cpu")
    calls = [lambda: ecq.kv4_extend(i32(1), i32(1), i32(1, 1), i32(1), i32(1), 16, n),
             lambda: ecq.kv4_extend(i32(1), i32(1), i32(1, 1), i32(1), i32(1), n, 1),
             lambda: ecq.kv4_release(torch.ones(1, dtype=torch.bool), i32(1), i32(1, 1), i32(1), i32(1), n),
             lambda: ecq.kv4_attention(rows, pages, i32(1, 1), i32(1), i32(2), n, group_size=32)]
    if n > 0:
        many = rows.expand(n, 1, 64)
        calls.append(lambda: ecq.kv4_append(many, many, pages, i32(1), group_size=32))
    for call in calls:
        with pytest.raises(ValueError, match="2\\^31"):
            call()


def test_import_with_a_torch_without_cuda():
    code = ("import torch\n"
            "for name in ('_cuda_getCurrentRawStream', '_cuda_getDevice'):\n"
            "    delattr(torch._C, name)\n"
            "import ecq_b200.model, ecq_b200 as ecq\n"
            "assert ecq.kv4_pages(1, 1, 64, device='cpu').numel()\n")
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=Path(__file__).resolve().parents[1])
    assert run.returncode == 0, run.stderr


@pytest.mark.parametrize("attention", ["ecq", "sdpa"])
def test_the_decoder_with_a_4bit_cache_has_no_choice_of_attention(attention):
    from ecq_b200.model import Llama7BConfig, Llama7BDecoder

    cfg = Llama7BConfig(layers=1, hidden=512, heads=4, head_dim=128, mlp=1024, vocab=1000, kv_len=16)
    with pytest.raises(ValueError, match="int4"):
        Llama7BDecoder(cfg, device="cpu", kv_cache="int4", attention=attention)
