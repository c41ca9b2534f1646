"""More refusals of the 4-bit KV cache's entry points that need no device."""
import subprocess
import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

import ecq_b200 as ecq  # noqa: E402
from ecq_b200 import _lib  # noqa: E402


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


# the C ABI's pointers are looked at but not dereferenced before a call is refused
AT = dict(lens=0x10000, new=0x20000, lens_out=0x30000, table=0x40000, free=0x50000, count=0x60000, count_out=0x70000, starts=0x80000,
          slots=0x90000, positions=0xa0000, done=0xb0000)


@pytest.mark.parametrize("out,what,shift", [
    ("lens_out", "new", 0), ("lens_out", "new", 76), ("lens_out", "new", -76), ("lens_out", "lens", 4), ("lens_out", "lens", -4),
    ("lens_out", "table", 0), ("lens_out", "table", 4 * 100 - 4), ("lens_out", "free", 4 * 49), ("lens_out", "count", -76), ("lens_out", "starts", 80),
    ("lens_out", "slots", 0), ("lens_out", "positions", 16), ("lens_out", "count_out", 0), ("count_out", "lens", 40), ("count_out", "new", 76),
    ("count_out", "table", 8), ("count_out", "free", 4 * 49), ("count_out", "starts", 80), ("count_out", "slots", 4), ("count_out", "count", 2)])
def test_lengths_and_count_that_share_memory_with_something_else(out, what, shift):
    # 20 requests with 5 columns, a stack of 50, 7 tokens
    a = dict(AT)
    a[out] = a[what] + shift
    L = _lib.lib()
    extend = L.ecq_kv4_extend(a["lens"], a["new"], a["lens_out"], a["table"], 5, 5, 20, 16, a["free"], 50, a["count"], a["count_out"],
                              a["starts"], a["slots"], a["positions"], 7, None, None)
    assert extend == -1
    if what in ("lens", "table", "free", "count", "count_out"):
        assert L.ecq_kv4_release(a["done"], a["lens"], a["lens_out"], a["table"], 5, 5, 20, 16, a["free"], 50, a["count"], a["count_out"],
                                 None, None) == -1


@pytest.mark.skipif(torch.cuda.is_available(), reason="the calls would run")
@pytest.mark.parametrize("out,what,shift", [("lens_out", "lens", 0), ("lens_out", "new", 80), ("lens_out", "new", -80), ("lens_out", "table", 400),
                                            ("count_out", "count", 0), ("count_out", "slots", 28), ("count_out", "free", -4)])
def test_lengths_and_count_beside_other_memory_are_not_refused(out, what, shift):
    a = dict(AT)
    a[out] = a[what] + shift
    assert _lib.lib().ecq_kv4_extend(a["lens"], a["new"], a["lens_out"], a["table"], 5, 5, 20, 16, a["free"], 50, a["count"], a["count_out"],
                                     a["starts"], a["slots"], a["positions"], 7, None, None) != -1
