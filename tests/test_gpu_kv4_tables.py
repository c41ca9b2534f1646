"""The 4-bit KV cache's bookkeeping at the ends of its ranges."""
import random

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import ecq_b200 as ecq  # noqa: E402
from test_gpu_kv4 import BADARG, i32  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def need(gigabytes):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gigabytes << 30:
        pytest.skip(f"needs {gigabytes} GB")


MOST = 2 ** 31 - 1


@pytest.mark.parametrize("refused", [False, True])
def test_extend_with_the_most_tokens(refused):
    need(24)
    table, status = torch.full((2, 4), -1, dtype=torch.int32, device="cuda"), i32([0])
    st = ecq.kv4_extend(i32([3, 0]), i32([9, -1 if refused else 20]), table, i32([7, 6, 5, 4]), i32([4]), 16, MOST, status=status)
    assert status.item() == (BADARG if refused else 0)
    n = 0 if refused else 29
    assert st.q_starts.tolist() == ([0, 0, 0] if refused else [0, 9, 29]) and st.slots.shape[0] == MOST
    for x in (st.slots, st.positions):
        assert x[n:].amax().item() == -1 and x[n:].amin().item() == -1
    if not refused:
        assert st.positions[:29].tolist() == list(range(3, 12)) + list(range(20))
        assert st.slots[9:29].tolist() == [4 * 16 + i for i in range(16)] + [5 * 16 + i for i in range(4)]


def test_append_of_the_most_tokens():
    need(16)
    pages, status = ecq.kv4_pages(2, 1, 64, 16, 64), i32([0])
    slots = torch.full((MOST,), -1, dtype=torch.int32, device="cuda")
    slots[-1], slots[5] = 20, 3
    k = torch.arange(64, device="cuda").half().view(1, 1, 64).expand(MOST, 1, 64)
    ecq.kv4_append(k, (-k[:1]).expand(MOST, 1, 64), pages, slots, status=status)
    got, neg = ecq.kv4_gather(pages, i32([20, 3, 4]), 64)
    assert status.item() == 0 and bool(got[0].any()) and torch.equal(got[0], got[1]) and torch.equal(neg[0], neg[1]) and not bool(got[2].any())
