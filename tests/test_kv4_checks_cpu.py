"""The bound that the GPU tests hold attention outputs to, on the CPU: outputs
with K, V and weights in fp16 are within it, those with a key too many or too few
are not."""
import pytest

torch = pytest.importorskip("torch")

from kv4_checks import within  # noqa: E402


def attention(q, k, v, keep, rounded):
    """q [rows, dim], k and v [keys, dim], keep [rows, keys]."""
    h = (lambda x: x.half().double()) if rounded else (lambda x: x)
    s = (q @ h(k).t() * q.shape[1] ** -0.5).masked_fill(~keep, -float("inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return h(p) @ h(v) / p.sum(-1, keepdim=True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("keys,rows,dim", [(1500, 130, 64), (300, 128, 128), (700, 40, 128)])
def test_the_bound_tells_one_key(dtype, keys, rows, dim):
    gen = torch.Generator().manual_seed(keys)
    q, k, v = (torch.randn(n, dim, generator=gen, dtype=torch.float64) for n in (rows, keys, keys))
    q = q.to(dtype).double()
    at = keys - rows + torch.arange(rows)[:, None]
    j = torch.arange(keys)
    want = attention(q, k, v, j <= at, False)[:, None]

    def good(keep):
        return within(attention(q, k, v, keep, True).to(dtype)[:, None], want, 1, dtype)

    assert good(j <= at)
    for gone in (0, 64, keys - rows - 1):                # a key that no row sees any more
        assert not good((j <= at) & (j != gone))
    assert not good(j < at) and not good(j <= at + 1)    # the causal limit off by one
    border = ((at + 1) % 64 == 0).long()                 # for the rows only that end with a step of 64 keys
    if bool(border.any()):
        assert not good(j <= at - border)
