"""Calls of the 4-bit KV cache's functions as a torch program makes them."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import ecq_b200 as ecq  # noqa: E402
from test_gpu_kv4 import fill, i32  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def test_a_gradient_that_attention_does_not_have_is_said():
    pages, table = fill([40, 17], 2, 64, 32, 16, 1)
    q = torch.randn(2, 4, 64, device="cuda").half()
    want = ecq.kv4_attention(q, pages, table, i32([40, 17]), group_size=32)
    w = torch.ones(64, device="cuda", dtype=torch.float16, requires_grad=True)
    got = ecq.kv4_attention(q * w, pages, table, i32([40, 17]), group_size=32)
    assert torch.equal(got, want) and got.requires_grad
    with pytest.raises(RuntimeError, match="no backward"):
        got.float().sum().backward()
    assert w.grad is None
    with torch.no_grad():
        assert not ecq.kv4_attention(q * w, pages, table, i32([40, 17]), group_size=32).requires_grad
    # a buffer that is used again stays a buffer
    buf = torch.zeros(5, 4, 64, dtype=torch.float16, device="cuda")
    with torch.no_grad():
        view = buf[1:3]
    for out in (buf[:2], view, buf[3:]):
        got = ecq.kv4_attention(q * w, pages, table, i32([40, 17]), group_size=32, out=out)
        assert torch.equal(got, want) and torch.equal(out, want) and not got.requires_grad and not buf.requires_grad


@pytest.mark.parametrize("odd", [1, 4, 68])
@pytest.mark.parametrize("dim", [64, 128])
def test_strides_of_dimensions_with_one_entry_do_not_matter(odd, dim):
    # one token out of a fused projection whose width is no multiple of 8, and one head of one
    pages, table = fill([40], 2, dim, 32, 16, 1)
    x = torch.randn(8 * dim, device="cuda").half()
    q = x[:4 * dim].view(1, 4, dim)
    k, v = x[4 * dim:6 * dim].view(1, 2, dim), x[6 * dim:].view(1, 2, dim)
    want = ecq.kv4_attention(q, pages, table, i32([40]), group_size=32)
    as_odd = lambda t, at: x.as_strided(t.shape, (8 * dim + odd, dim, 1), at)  # noqa: E731
    out = torch.zeros(9 * dim, device="cuda", dtype=torch.float16).as_strided(q.shape, (8 * dim + odd, dim, 1))
    got = ecq.kv4_attention(as_odd(q, 0), pages, table, i32([40]), group_size=32, out=out)
    assert torch.equal(got, want) and torch.equal(out, want)
    a, b = pages.clone(), pages.clone()
    ecq.kv4_append(k, v, a, i32([5]), group_size=32)
    ecq.kv4_append(as_odd(k, 4 * dim), as_odd(v, 6 * dim), b, i32([5]), group_size=32)
    assert torch.equal(a, b)
    pool = ecq.kv4_pages(1, 1, dim, 16, 32)
    ecq.kv4_append(x.as_strided((3, 1, dim), (2 * dim, odd, 1)), x.as_strided((3, 1, dim), (2 * dim, odd, 1), dim), pool, i32([0, 1, 2]), group_size=32)
    want = ecq.kv4_attention(x.view(4, 2, dim)[:3, :1].contiguous(), pool, i32([[0], [0], [0]]), i32([3, 3, 3]), group_size=32)
    got = ecq.kv4_attention(x.as_strided((3, 1, dim), (2 * dim, odd, 1)), pool, i32([[0], [0], [0]]), i32([3, 3, 3]), group_size=32,
                            out=torch.zeros(6 * dim, device="cuda", dtype=torch.float16).as_strided((3, 1, dim), (2 * dim, odd, 1)))
    assert torch.equal(got, want)


def test_an_output_whose_rows_share_memory_is_refused():
    pages, table = fill([40, 17], 2, 64, 32, 16, 1)
    q = torch.randn(2, 4, 64, device="cuda").half()
    for out in (torch.zeros(1, 4, 64, device="cuda").half().expand(2, 4, 64), torch.zeros(2, 1, 64, device="cuda").half().expand(2, 4, 64),
                torch.zeros(1000, device="cuda").half().as_strided((2, 4, 64), (32, 128, 1))):
        with pytest.raises(ValueError, match="share memory"):
            ecq.kv4_attention(q, pages, table, i32([40, 17]), group_size=32, out=out)


@pytest.mark.parametrize("tp", [2, 4])
def test_the_decoders_ranks_hold_their_heads_of_the_4bit_cache(tp):
    from ecq_b200.model import Llama7BConfig, Llama7BDecoder

    cfg = Llama7BConfig(layers=2, hidden=2048, heads=16, head_dim=128, mlp=2048, vocab=1000, kv_len=100)
    whole = Llama7BDecoder(cfg, tp=1, seed=5, kv_cache="int4").cache
    for rank in range(tp):
        mine = Llama7BDecoder(cfg, tp=tp, rank=rank, seed=5, exchange="nccl", kv_cache="int4").cache
        assert torch.equal(mine.block_table, whole.block_table) and torch.equal(mine.seq_lens, whole.seq_lens)
        n = cfg.heads // tp
        q = torch.randn(1, cfg.heads, 128, device="cuda").half()
        for layer in range(cfg.layers):
            assert torch.equal(mine.pages[layer], whole.pages[layer][:, rank * n:(rank + 1) * n])
            mine.attention(layer, q[:, rank * n:(rank + 1) * n])
        mine.check()
