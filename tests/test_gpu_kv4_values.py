"""Attention over the 4-bit KV cache where values, scores or lengths are at the
ends of their ranges."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import ecq_b200 as ecq  # noqa: E402
from test_gpu_kv4 import DTYPES, LAYOUTS, check_attention, decode, i32, reference  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def store(k, v, page, g):
    """Rows [n, heads, dim] of one request in a pool of their own, and its table."""
    n, heads, dim = k.shape
    pages = ecq.kv4_pages(-(-n // page), heads, dim, page, g)
    pages.fill_(255)
    ecq.kv4_append(k, v, pages, torch.arange(n, dtype=torch.int32, device="cuda"), group_size=g)
    return pages, torch.arange(pages.shape[0], dtype=torch.int32, device="cuda")[None]


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


# -- stored values past fp16's end ------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,g", LAYOUTS)
@pytest.mark.parametrize("heads,share,new", [(1, 4, 1), (64, 2, 100)])  # streamed; the prompt kernel
@pytest.mark.parametrize("big", ["k", "v"])
def test_groups_whose_largest_value_is_past_the_end_of_fp16(dtype, dim, g, heads, share, new, big):
    # a fifth of such groups has a scale that was rounded up so far that code 15 stands for 65520 or more
    n, page = 200, 16
    end = torch.finfo(dtype).max if dtype == torch.float16 else 65280.0  # the largest of the type below fp16's end
    x = randn(2, n, heads, dim, seed=dim + g)
    x[int(big == "v")] *= 30000
    x = x.clamp(-end, end).to(dtype)
    pages, table = store(x[0], x[1], page, g)
    value = decode(pages, dim, g)[int(big == "v")][1]
    assert (abs(value[:n]) >= 65520).any() or dtype == torch.bfloat16
    q = (randn(new, heads * share, dim, seed=1) * (1e-4 if big == "k" else 1.0)).to(dtype)
    got = ecq.kv4_attention(q, pages, table, i32([n]), i32([0, new]), new, group_size=g)
    assert bool(got.isfinite().all())
    check_attention(got, *reference(q, pages, table, [n], [0, new], page, dim, g), dtype, new > 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,g", LAYOUTS)
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_one_value_at_the_end_of_fp16_stays_with_the_rows_that_see_it(dtype, dim, g, which, sign):
    n, new, heads, share, at = 150, 110, 64, 2, 100
    x = randn(2, n, heads, dim, seed=3).abs().to(dtype)       # groups without a negative value: zero is about 0
    clean, table = store(x[0], x[1], 16, g)
    x[which, at, :, 5] = sign * float("inf")                  # clamped to 65504
    x[which, at, 1, 5] = sign * 65504.0                       # in bf16 65536, clamped too
    pages, _ = store(x[0], x[1], 16, g)
    q = (randn(new, heads * share, dim, seed=4) * (1e-4 if which == 0 else 1.0)).to(dtype)
    got, want = (ecq.kv4_attention(q, p, table, i32([n]), i32([0, new]), new, group_size=g) for p in (pages, clean))
    first = at - (n - new)
    assert torch.equal(got[:first], want[:first])
    assert bool(got.isfinite().all())
    check_attention(got, *reference(q, pages, table, [n], [0, new], 16, dim, g), dtype, True)


def test_bytes_far_past_the_end_of_fp16_stay_with_the_rows_that_see_them():
    # what kv4_append never writes: scales of 60000, so values up to 900000 (finite; fp16 has none near them)
    n, new, heads, share, at, dim, g = 100, 80, 64, 2, 60, 64, 32
    x = randn(2, n, heads, dim, seed=5).half()
    clean, table = store(x[0], x[1], 16, g)
    q = randn(new, heads * share, dim, seed=6).bfloat16()
    want = ecq.kv4_attention(q, clean, table, i32([n]), i32([0, new]), new, group_size=g)
    for v in (0, 1):
        pages = clean.clone()
        par = pages.view(-1, heads, 16 * 64 + 256)[at // 16, :, 1024 + 128 * v:1152 + 128 * v].view(torch.float16).view(heads, 16, 2, 2)
        par[:, at % 16, 0, 0] = 60000.0
        got = ecq.kv4_attention(q, pages, table, i32([n]), i32([0, new]), new, group_size=g)
        first = at - (n - new)
        assert torch.equal(got[:first], want[:first])
        if v:
            assert bool(got[first:, :, :32].isnan().all()) and torch.equal(got[first:, :, 32:], want[first:, :, 32:])
