"""The 4-bit KV cache's bookkeeping at the ends of its ranges."""
import random

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import ecq_b200 as ecq  # noqa: E402
from test_gpu_kv4 import BADARG, Model, i32  # noqa: E402


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
    table[0, 0] = 9
    st = ecq.kv4_extend(i32([3, 0]), i32([9, -1 if refused else 20]), table, i32([7, 6, 5, 4]), i32([4]), 16, MOST, status=status)
    assert status.item() == (BADARG if refused else 0)
    n = 0 if refused else 29
    assert st.q_starts.tolist() == ([0, 0, 0] if refused else [0, 9, 29]) and st.slots.shape[0] == MOST
    for x in (st.slots, st.positions):
        assert x[n:].amax().item() == -1 and x[n:].amin().item() == -1
    if not refused:
        assert st.positions[:29].tolist() == list(range(3, 12)) + list(range(20))
        assert st.slots[:9].tolist() == [9 * 16 + i for i in range(3, 12)]
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


TOO_LARGE = 2 ** 31 // 16  # the first page of 16 tokens whose slots are no int32


@pytest.mark.parametrize("page", [-1, -2 ** 31, TOO_LARGE, 2 ** 31 - 1])
@pytest.mark.parametrize("batch,in_place", [(3, False), (3, True), (700, False), (700, True)])
@pytest.mark.parametrize("where", ["held", "first popped", "last popped"])
def test_extend_refuses_bad_pages(page, batch, in_place, where):
    cols, each = 6, 3
    lens = [5] + [16] * (batch - 1)              # request 0 goes on in its first page, the others start new ones
    new = [2] + [16 * each] * (batch - 1)
    table = torch.arange(batch * cols, dtype=torch.int32, device="cuda").view(batch, cols).contiguous()
    pops = each * (batch - 1)
    free = torch.arange(pops + 4, dtype=torch.int32, device="cuda")
    status, ln, ct = i32([0]), i32(lens), i32([pops + 4])
    kw = dict(status=status, seq_lens_out=ln, free_count_out=ct) if in_place else dict(status=status)
    pad = sum(new) + 3
    ok = table.clone()
    if where == "held":
        table[0, 0] = page
    else:
        free[-1 if where == "first popped" else 4] = page
    free[:4] = -1                                # not popped: not looked at
    table[1:, 0] = -1                            # full: not looked at either
    keep, stack = table.clone(), free.clone()
    st = ecq.kv4_extend(ln, i32(new), table, free, ct, 16, pad, **kw)
    assert status.item() == BADARG
    assert st.seq_lens.tolist() == lens and st.free_count.item() == pops + 4 and torch.equal(table, keep) and torch.equal(free, stack)
    assert not bool(st.q_starts.any()) and bool((st.slots == -1).all()) and bool((st.positions == -1).all())
    # the same with a good page
    status.zero_()
    table[0, 0] = ok[0, 0]
    free[4:] = torch.arange(4, pops + 4, dtype=torch.int32, device="cuda")
    st = ecq.kv4_extend(ln, i32(new), table, free, ct, 16, pad, **kw)
    assert status.item() == 0 and st.free_count.item() == 4
    assert st.slots[:2].tolist() == [5, 6] and bool((st.slots[:-3] >= 0).all())
    assert st.seq_lens.tolist() == [a + b for a, b in zip(lens, new)]


@pytest.mark.parametrize("count", [-1, -2 ** 31, 101, 2 ** 31 - 1])
@pytest.mark.parametrize("in_place", [False, True])
def test_a_count_that_the_stack_cannot_have(count, in_place):
    # more pages asked for than the first ones that are looked at: nothing behind the stack is read
    batch, cols = 700, 5
    table = torch.arange(batch * cols, dtype=torch.int32, device="cuda").view(batch, cols).contiguous()
    keep, status, ln, ct = table.clone(), i32([0]), i32([0] * batch), i32([count])
    kw = dict(status=status, seq_lens_out=ln, free_count_out=ct) if in_place else dict(status=status)
    st = ecq.kv4_extend(ln, i32([80] * batch), table, torch.arange(100, dtype=torch.int32, device="cuda"), ct, 16, 80 * batch, **kw)
    assert status.item() == BADARG and torch.equal(table, keep) and st.free_count.item() == count
    assert not bool(st.seq_lens.any()) and not bool(st.q_starts.any()) and bool((st.slots == -1).all())
    status.zero_()
    _, got = ecq.kv4_release(torch.ones(batch, dtype=torch.bool, device="cuda"), i32([80] * batch), table,
                             torch.arange(100, dtype=torch.int32, device="cuda"), i32([count]), 16, status=status)
    assert status.item() == BADARG and got.item() == count


@pytest.mark.parametrize("page", [-1, -2 ** 31, TOO_LARGE])
@pytest.mark.parametrize("batch,cols", [(3, 6), (700, 6), (40, 700)])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("last", [False, True])
def test_release_refuses_bad_pages(page, batch, cols, in_place, last):
    lens = [16 * cols - 3 - b % 5 for b in range(batch)]
    done = [b % 2 == 0 for b in range(batch)]
    who = max(b for b in range(batch) if done[b]) if last else 0
    table = torch.arange(batch * cols, dtype=torch.int32, device="cuda").view(batch, cols).contiguous()
    table[1] = -1                                    # not done: not looked at
    good = int(table[who, cols - 1 if last else 0])
    table[who, cols - 1 if last else 0] = page
    room = batch * cols + 2
    free = torch.full((room,), -5, dtype=torch.int32, device="cuda")
    status, ln, ct, flags = i32([0]), i32(lens), i32([2]), torch.tensor(done, device="cuda")
    kw = dict(status=status, seq_lens_out=ln, free_count_out=ct) if in_place else dict(status=status)
    got = ecq.kv4_release(flags, ln, table, free, ct, 16, **kw)
    assert status.item() == BADARG and got[0].tolist() == lens and got[1].item() == 2 and bool((free[:2] == -5).all())  # behind the stack's end anything may be
    status.zero_()
    table[who, cols - 1 if last else 0] = good
    got = ecq.kv4_release(flags, ln, table, free, ct, 16, **kw)
    pages = [p for b in range(batch) if done[b] for p in range(b * cols, (b + 1) * cols)]
    assert status.item() == 0 and got[1].item() == 2 + len(pages) and free[2:2 + len(pages)].tolist() == pages
    assert got[0].tolist() == [0 if d else n for n, d in zip(lens, done)]


@pytest.mark.parametrize("batch,page,most", [(1, 16, 1), (1, 64, 5000), (17, 16, 40), (512, 32, 70), (513, 16, 3), (1100, 256, 30),
                                             (700, 16, 400), (8192, 16, 2)])
def test_extend_and_release_in_place_over_many_steps(batch, page, most):
    """As a cache calls them: lengths and count in place, on a cluster of CTAs where there is much to write."""
    rng = random.Random(batch + page)
    cols = -(-3 * most // page) + 1
    n_pages = batch * cols
    m = Model(batch, cols, page, n_pages)
    lens, count, free, status = i32([0] * batch), i32([n_pages]), i32(m.free), i32([0])
    table = torch.full((batch, cols), -1, dtype=torch.int32, device="cuda")
    for step in range(6):
        new = [rng.choice([0, 1, rng.randint(0, most)]) if n + most <= cols * page else 0 for n in m.lens]
        if step == 0:
            new[-1] = most
        pad = sum(new) + rng.randint(0, 5)
        starts, slots, pos = m.extend(new)
        st = ecq.kv4_extend(lens, i32(new), table, free, count, page, pad, status=status, seq_lens_out=lens, free_count_out=count)
        assert st.seq_lens is lens and lens.tolist() == m.lens and st.q_starts.tolist() == starts
        assert st.slots.tolist() == slots + [-1] * (pad - len(slots)) and st.positions.tolist() == pos + [-1] * (pad - len(pos))
        assert count.item() == len(m.free)
        got = table.cpu().numpy()
        for b, row in enumerate(m.rows):
            assert got[b, :len(row)].tolist() == row
        done = [rng.random() < 0.4 for _ in range(batch)]
        m.release(done)
        ecq.kv4_release(torch.tensor(done, device="cuda"), lens, table, free, count, page, status=status, seq_lens_out=lens,
                        free_count_out=count)
        assert lens.tolist() == m.lens and count.item() == len(m.free) and free[:len(m.free)].tolist() == m.free
    assert sorted([p for r in m.rows for p in r] + m.free) == list(range(n_pages)) and status.item() == 0
