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


@pytest.mark.parametrize("given", [False, True])
def test_a_gradient_that_attention_does_not_have_is_said(given):
    pages, table = fill([40, 17], 2, 64, 32, 16, 1)
    q = torch.randn(2, 4, 64, device="cuda").half()
    want = ecq.kv4_attention(q, pages, table, i32([40, 17]), group_size=32)
    w = torch.ones(64, device="cuda", dtype=torch.float16, requires_grad=True)
    out = torch.full_like(q, 7.0) if given else None
    got = ecq.kv4_attention(q * w, pages, table, i32([40, 17]), group_size=32, out=out)
    assert torch.equal(got, want) and got.requires_grad and (not given or got.data_ptr() == out.data_ptr())
    with pytest.raises(RuntimeError, match="no backward"):
        got.float().sum().backward()
    assert w.grad is None
    with torch.no_grad():
        assert not ecq.kv4_attention(q * w, pages, table, i32([40, 17]), group_size=32).requires_grad
