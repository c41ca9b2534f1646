"""The 4-bit KV cache on the GPU: bookkeeping against a Python model, storage
against the quantiser's definition, attention against float64 over the values
that the pool's bytes stand for, and the calls together as a server makes them."""
import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import ecq_b200 as ecq  # noqa: E402
from ecq_b200._lib import EcqError  # noqa: E402

DTYPES = [torch.float16, torch.bfloat16]
NO_PAGES, BADARG = 8, 4


@pytest.fixture(scope="module", autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# -- bookkeeping ------------------------------------------------------------------

class Model:
    """The tables of a server in plain Python."""

    def __init__(self, batch, cols, page, n_pages):
        self.page, self.cols = page, cols
        self.lens, self.rows = [0] * batch, [[] for _ in range(batch)]
        self.free = list(range(n_pages - 1, -1, -1))

    def extend(self, new):
        slots, pos, starts = [], [], [0]
        for b, n in enumerate(new):
            while len(self.rows[b]) * self.page < self.lens[b] + n:
                self.rows[b].append(self.free.pop())
            for p in range(self.lens[b], self.lens[b] + n):
                pos.append(p)
                slots.append(self.rows[b][p // self.page] * self.page + p % self.page)
            self.lens[b] += n
            starts.append(starts[-1] + n)
        return starts, slots, pos

    def release(self, done):
        for b, d in enumerate(done):
            if d:
                self.free += self.rows[b]
                self.lens[b], self.rows[b] = 0, []


@pytest.mark.parametrize("batch,page,most", [(1, 16, 1), (1, 64, 5000), (17, 16, 40), (512, 32, 70), (513, 16, 3), (1100, 256, 30),
                                             (8192, 16, 2)])
def test_extend_and_release_over_many_steps(batch, page, most):
    rng = random.Random(batch * page)
    cols = -(-3 * most // page) + 1
    n_pages = batch * cols
    m = Model(batch, cols, page, n_pages)
    lens, count = i32([0] * batch), i32([n_pages])
    free, table = i32(m.free), torch.full((batch, cols + 3), -7, dtype=torch.int32, device="cuda")[:, :cols]
    status = i32([0])
    for step in range(6):
        new = [rng.choice([0, 1, rng.randint(0, most)]) if n + most <= cols * page else 0 for n in m.lens]
        if step == 0:
            new[-1] = most
        pad = sum(new) + rng.randint(0, 5)
        starts, slots, pos = m.extend(new)
        st = ecq.kv4_extend(lens, i32(new), table, free, count, page, pad, status=status)
        torch.cuda.synchronize()
        assert st.seq_lens.tolist() == m.lens and st.q_starts.tolist() == starts
        assert st.slots.tolist() == slots + [-1] * (pad - len(slots))
        assert st.positions.tolist() == pos + [-1] * (pad - len(pos))
        assert st.free_count.item() == len(m.free)
        got = table.cpu().numpy()
        for b, row in enumerate(m.rows):
            assert got[b, :len(row)].tolist() == row
        lens, count = st.seq_lens, st.free_count
        done = [rng.random() < 0.4 for _ in range(batch)]
        m.release(done)
        lens, count = ecq.kv4_release(torch.tensor(done, device="cuda"), lens, table, free, count, page, status=status)
        assert lens.tolist() == m.lens and count.item() == len(m.free)
        assert free[:len(m.free)].tolist() == m.free
    held = [p for r in m.rows for p in r] + m.free
    assert sorted(held) == list(range(n_pages))
    assert status.item() == 0


@pytest.mark.parametrize("batch", [3, 1500])
@pytest.mark.parametrize("what", ["pages", "pages and tokens", "tokens", "negative", "negative length", "row"])
def test_extend_is_all_or_nothing(batch, what):
    lens, new = [5] * batch, [1] * batch
    free_n, pad = 4 * batch, 4 * batch
    bit = BADARG
    if what == "pages":
        new[1], free_n, bit, pad = 40, 1, NO_PAGES, 5 * batch + 40  # 45 tokens: two more pages of 16
    elif what == "pages and tokens":
        new[1], free_n, pad = 40, 1, batch  # more tokens than there is room for: that is said first
    elif what == "tokens":
        pad = batch - 1
    elif what == "negative":
        new[-1] = -1
    elif what == "negative length":
        lens[0] = -3
    else:
        new[0] = 4 * 16 - 4  # 5 + 60 tokens in a row of 4 pages of 16
    table = torch.arange(batch * 4, dtype=torch.int32, device="cuda").view(batch, 4)
    keep, free, status = table.clone(), torch.arange(free_n, dtype=torch.int32, device="cuda"), i32([0])
    for in_place in (False, True):
        ln, ct = i32(lens), i32([free_n])
        st = ecq.kv4_extend(ln, i32(new), table, free, ct, 16, pad, status=status, seq_lens_out=ln if in_place else None,
                            free_count_out=ct if in_place else None)
        assert status.item() == bit
        status.zero_()
        assert st.seq_lens.tolist() == lens and st.free_count.item() == free_n
        assert torch.equal(table, keep) and st.q_starts.tolist() == [0] * (batch + 1)
        assert st.slots.tolist() == [-1] * pad and st.positions.tolist() == [-1] * pad


def test_release_without_room_changes_nothing():
    table, free, status = torch.zeros(2, 4, dtype=torch.int32, device="cuda"), i32([7, 8, 9]), i32([0])
    lens, count = ecq.kv4_release(torch.tensor([True, True], device="cuda"), i32([17, 40]), table, free, i32([1]), 16, status=status)
    assert status.item() == NO_PAGES and lens.tolist() == [17, 40] and count.item() == 1 and free.tolist() == [7, 8, 9]
    status.zero_()
    lens, count = ecq.kv4_release(torch.tensor([True, False], device="cuda"), i32([65, 40]), table, free, i32([1]), 16, status=status)
    assert status.item() == BADARG and lens.tolist() == [65, 40]  # 65 tokens are more than a row of 4 pages holds


# -- storage ----------------------------------------------------------------------

def decode(pages, dim, g):
    """Codes [slots, heads, D] and float64 values of a pool's bytes, K and V, from
    the layout's definition."""
    n, heads, per = pages.shape
    G = dim // g
    blk = 16 * dim + 128 * G
    b = pages.cpu().numpy().reshape(n, heads, per // blk, blk)
    d = np.arange(dim)
    nib = (((d % 32) // 8) * (dim // 4) + (d // 32) * 8 + d % 8, (d % 8) * (dim // 8) + d // 8)
    out = []
    for v in (0, 1):
        rows = b[..., 8 * dim * v:8 * dim * (v + 1)].reshape(n, heads, -1, 16, dim // 2)
        code = rows[..., nib[v] // 2] >> (4 * (nib[v] % 2)).astype(np.uint8) & 15
        par = np.ascontiguousarray(b[..., 16 * dim + 64 * G * v:16 * dim + 64 * G * (v + 1)]).view(np.float16)
        par = par.reshape(n, heads, -1, 16, G, 2).astype(np.float64)
        val = code * np.repeat(par[..., 0], g, -1) + np.repeat(par[..., 1], g, -1)
        order = lambda x: x.transpose(0, 2, 3, 1, 4).reshape(-1, heads, dim)  # noqa: E731
        out.append((order(code), order(val)))
    return out


def quantise(x, g):
    """The definition, in float32 as the kernel computes it."""
    x = x.float().cpu().numpy().clip(-65504, 65504)
    xg = x.reshape(*x.shape[:-1], -1, g)
    lo, hi = xg.min(-1, keepdims=True), xg.max(-1, keepdims=True)
    zero = lo.astype(np.float16).astype(np.float32)
    scale = ((hi - lo) / np.float32(15)).astype(np.float16).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        code = np.where(scale == 0, 0, np.rint((xg - zero) / scale).clip(0, 15))
    return code.reshape(x.shape), (code.astype(np.float64) * scale + zero).reshape(x.shape)


LAYOUTS = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,g", LAYOUTS)
@pytest.mark.parametrize("heads,page,tokens", [(1, 16, 1), (3, 16, 37), (8, 64, 200), (5, 256, 300)])
def test_append_and_gather(dtype, dim, g, heads, page, tokens):
    gen = torch.Generator(device="cuda").manual_seed(dim + g + tokens)
    n_pages = -(-tokens // page) + 2
    pages = ecq.kv4_pages(n_pages, heads, dim, page, g)
    pages.fill_(0xA5)
    before = pages.clone()
    qkv = torch.randn(tokens, 3, heads, dim, generator=gen, device="cuda").to(dtype)  # k and v as views of one projection
    qkv[0, 1, 0, :g] = 3.25                      # a constant group
    qkv[-1, 2, -1, :g] *= 2.0 ** -20             # a group whose scale is subnormal
    slots = torch.randperm(n_pages * page, generator=gen, device="cuda")[:tokens].to(torch.int32)
    if tokens > 2:
        slots[1] = -1
    ecq.kv4_append(qkv[:, 1], qkv[:, 2], pages, slots, group_size=g)
    kept = slots >= 0
    at = slots[kept].long().cpu().numpy()
    parts = decode(pages, dim, g)
    for (code, val), x in zip(parts, (qkv[:, 1], qkv[:, 2])):
        want_code, want = quantise(x[kept], g)
        assert np.array_equal(code[at], want_code)
        assert np.array_equal(val[at], want)
    # other slots keep every byte
    with np.errstate(invalid="ignore"):
        for (code, val), (code0, val0) in zip(parts, decode(before, dim, g)):
            rest = np.setdiff1d(np.arange(n_pages * page), at)
            assert np.array_equal(code[rest], code0[rest]) and np.array_equal(val[rest], val0[rest], equal_nan=True)
    k, v = ecq.kv4_gather(pages, slots, dim, group_size=g, dtype=dtype)
    assert k.shape == v.shape == (tokens, heads, dim) and k.dtype == dtype
    for got, (_, val) in zip((k, v), parts):
        want = torch.zeros(tokens, heads, dim, dtype=torch.float64)
        want[kept.cpu()] = torch.from_numpy(val[at])
        # fp32 sum of an exact product, then one rounding: half a step of each
        tol = want.abs() * (torch.finfo(dtype).eps / 2 + 2.0 ** -24) + 2.0 ** -25
        assert bool(((got.cpu().double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_of_values_without_a_code(dtype):
    x = torch.randn(4, 1, 64, device="cuda").to(dtype)
    x[0, 0, 3], x[1, 0, 5], x[2, 0, 40] = float("nan"), float("inf"), float("-inf")
    pages = ecq.kv4_pages(1, 1, 64, 16, 32)
    ecq.kv4_append(x, x, pages, i32([0, 1, 2, 3]), group_size=32)
    for got in ecq.kv4_gather(pages, i32([0, 1, 2, 3]), 64, group_size=32, dtype=torch.float16):
        got = got[:, 0].float()
        assert bool(got[0, :32].isnan().all()) and not bool(got[0, 32:].isnan().any())  # a NaN stays in its group
        assert got[1, 5] >= 65000 and bool(got[1].isfinite().all())                      # infinities are clamped
        assert got[2, 40] <= -65000 and bool(got[2].isfinite().all())
        assert bool(got[3].isfinite().all())


def test_slots_beyond_the_pool_are_reported_and_not_written():
    pages, status = ecq.kv4_pages(2, 2, 64, 16, 64), i32([0])
    x = torch.ones(3, 2, 64, dtype=torch.float16, device="cuda")
    ecq.kv4_append(x, x, pages, i32([32, -5, 2 ** 31 - 1]), group_size=64, status=status)
    assert status.item() == BADARG and not bool(pages.any())
    status.zero_()
    k, v = ecq.kv4_gather(pages + 1, i32([32, 0]), 64, group_size=64, status=status)
    assert status.item() == BADARG and not bool(k[0].any()) and bool(k[1].any())


# -- attention --------------------------------------------------------------------

def fill(lens, heads, dim, g, page, seed, dtype=torch.float16, spare=3, strong=0.0):
    """A pool with random rows for requests of `lens` tokens, everything else 255
    (NaN as a scale), and its table; rows are stored by kv4_append."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cols = max(1, -(-max(lens) // page))
    held = [-(-n // page) for n in lens]
    pages = ecq.kv4_pages(sum(held) + spare, heads, dim, page, g)
    pages.fill_(255)
    ids = torch.randperm(pages.shape[0], generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), cols), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, (n, m) in enumerate(zip(lens, held)):
        table[b, :m] = ids[at:at + m]
        at += m
        if n:
            p = torch.arange(n, device="cuda")
            slots = (table[b, p // page] * page + p % page).to(torch.int32)
            k, v = (torch.randn(n, heads, dim, generator=gen, device="cuda") for _ in range(2))
            k = k + strong * torch.randn(heads, dim, generator=gen, device="cuda")
            ecq.kv4_append(k.to(dtype), v.to(dtype), pages, slots, group_size=g)
    return pages, table


def reference(q, pages, table, lens, starts, page, dim, g, scale=None):
    """float64 attention over the values in the pool, and what the rounding of a
    row's inputs can come to: sum |q||k| scale over its keys (the largest) and
    the largest |v|."""
    (_, k), (_, v) = decode(pages, dim, g)
    k, v = torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda()
    heads, share = k.shape[1], q.shape[1] // k.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    out, s_abs, v_abs = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), *torch.zeros(2, *q.shape[:2], 1, device="cuda")
    tb = table.long()
    for b, n in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        if n == 0 or lo == hi:
            continue
        p = torch.arange(n, device="cuda")
        rows = tb[b, p // page] * page + p % page
        for h in range(heads):
            x, kk, vv = q[lo:hi, h * share:(h + 1) * share].double(), k[rows, h], v[rows, h]
            seen = p <= (n - (hi - lo) + torch.arange(hi - lo, device="cuda"))[:, None]
            s = torch.einsum("isd,jd->isj", x, kk) * scale
            w = torch.softmax(s.masked_fill(~seen[:, None], -float("inf")), -1).nan_to_num()
            out[lo:hi, h * share:(h + 1) * share] = torch.einsum("isj,jd->isd", w, vv)
            a = torch.einsum("isd,jd->isj", x.abs(), kk.abs()) * abs(scale)
            s_abs[lo:hi, h * share:(h + 1) * share] = a.masked_fill(~seen[:, None], 0).amax(-1, keepdim=True).float()
            v_abs[lo:hi, h * share:(h + 1) * share] = vv.abs().max().float()
    return out, s_abs.double(), v_abs.double()


def check_attention(got, want, s_abs, v_abs, dtype, rounded=False):
    """Scores are sums of at most 256 products in fp32 (each step 2^-24 of what is
    summed: 2^-16 of sum |q||k|); an error e of a score is a factor 1 +- e of its
    weight, and of the sum: 2 e of the largest |v|. Weights (2^-20: two fp16 parts,
    exp2) and their fp32 sums add 2^-16 of it. Then one rounding to the type.
    ``rounded``: the prompt kernel's K, V and weights are fp16, 2^-11 of each: 2^-11
    of sum |q||k| in a score, and 2^-11 of the largest |v| twice. For bf16 the other
    kernel's weights, and weights times scale, are fp16: 2^-11 each, of codes times
    scales (at most twice the largest |v|, as are the zeros)."""
    k, v = (2.0 ** -11, 2 * 2.0 ** -11) if rounded else (0.0, 4 * 2.0 ** -11 if dtype == torch.bfloat16 else 0.0)
    tol = (torch.finfo(dtype).eps / 2) * want.abs() + (2 * (2.0 ** -16 + k) * s_abs + 2 * 2.0 ** -16 + v) * v_abs + 2.0 ** -24
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


def stream_rows(batch, heads):
    """Requests with more rows (queries times heads that share a cache head) go to
    the prompt kernel."""
    return max(32, 4500 // (batch * heads))


def attend_case(lens, new, heads, share, dim, g, page, dtype, seed=1, q_scale=1.0, **kw):
    pages, table = fill(lens, heads, dim, g, page, seed, strong=2.0)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = (q_scale * torch.randn(starts[-1], heads * share, dim, generator=gen, device="cuda")).to(dtype)
    one = all(n == 1 for n in new)
    status = i32([0])
    got = ecq.kv4_attention(q, pages, table, i32(lens), None if one else i32(starts), max(new + [1]), group_size=g, status=status, **kw)
    torch.cuda.synchronize()
    assert status.item() == 0
    want, s_abs, v_abs = reference(q, pages, table, lens, starts, page, dim, g, kw.get("scale"))
    for b, n in enumerate(new):
        at = slice(starts[b], starts[b + 1])
        check_attention(got[at], want[at], s_abs[at], v_abs[at], dtype, n * share > stream_rows(len(lens), heads))
    return q, pages, table, starts, got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,g", LAYOUTS)
@pytest.mark.parametrize("lens,page", [([1], 16), ([0, 15, 16, 17], 16), ([64, 65, 63, 0, 130], 64), ([700, 3, 299], 32), ([513], 256)])
def test_attention_of_single_tokens(dtype, dim, g, lens, page):
    attend_case(lens, [1] * len(lens), 2, 2, dim, g, page, dtype, seed=len(lens))


@pytest.mark.parametrize("heads,share", [(1, 1), (3, 1), (1, 3), (2, 4), (1, 5), (2, 7), (1, 8), (1, 9), (1, 16), (1, 17), (1, 33), (1, 64)])
def test_attention_head_layouts(heads, share):
    attend_case([100, 33], [1, 1], heads, share, 128, 64, 16, torch.float16, seed=share)
    attend_case([100, 33], [3, 2], heads, share, 64, 32, 16, torch.bfloat16, seed=share + 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,g", [(64, 32), (128, 128)])
@pytest.mark.parametrize("lens,new", [([5], [5]), ([1, 40, 40, 0, 200], [1, 2, 0, 0, 7]), ([33, 47], [33, 17]), ([90, 300], [64, 1])])
def test_attention_of_several_tokens_is_causal(dtype, dim, g, lens, new):
    attend_case(lens, new, 2, 3, dim, g, 16, dtype, seed=sum(new))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,g", LAYOUTS)
@pytest.mark.parametrize("lens,new,page", [([65], [65], 16), ([64, 200], [64, 129], 16), ([300, 5, 64], [257, 1, 64], 64)])
def test_attention_of_prompts(dtype, dim, g, lens, new, page):
    attend_case(lens, new, 64, 2, dim, g, page, dtype, seed=sum(new))  # 64 heads: the prompt kernel from 32 rows on


@pytest.mark.parametrize("share,new,lens", [
    (1, [65, 128, 129, 600], [65, 1000, 129, 700]), (4, [17, 32, 33, 64, 65, 1, 0], [17, 500, 33, 64, 129, 77, 30]),
    (8, [130], [1500]), (7, [40, 9, 10], [41, 400, 10]), (64, [2, 1, 5], [100, 64, 5]), (3, [300], [300])])
def test_attention_of_prompts_head_layouts(share, new, lens):
    attend_case(lens, new, 48, share, 128, 64, 32, torch.float16, seed=share)
    attend_case(lens, new, 80, share, 64, 32, 128, torch.bfloat16, seed=share + 1, scale=-0.2)


def test_attention_of_prompts_longer_than_the_request_and_scales():
    # more queries than tokens: the first ones see nothing
    lens, new = [50, 0], [70, 80]
    pages, table = fill(lens, 64, 64, 32, 16, 3)
    q = torch.randn(150, 128, 64, device="cuda").half()
    got = ecq.kv4_attention(q, pages, table, i32(lens), i32([0, 70, 150]), 80, group_size=32)
    want, s_abs, v_abs = reference(q, pages, table, lens, [0, 70, 150], 16, 64, 32)
    check_attention(got, want, s_abs, v_abs, torch.float16, True)
    assert not bool(got[:20].any()) and not bool(got[70:].any()) and bool(got[20:70].any())
    for kw in (dict(scale=0.0), dict(q_scale=30.0), dict(q_scale=1e-6, scale=3e5)):
        attend_case([400], [150], 128, 2, 128, 64, 64, torch.bfloat16, **kw)


def test_tokens_that_are_not_numbers_reach_only_rows_that_see_them():
    # a row of NaN at position 45 of a 70-token prompt: earlier queries are as without it
    for n, share in ((70, 2), (9, 2), (1, 1)):
        x = torch.randn(2, 70, 128, 64, device="cuda").half()
        pages, clean = ecq.kv4_pages(5, 128, 64, 16, 32), ecq.kv4_pages(5, 128, 64, 16, 32)
        slots, table = torch.arange(70, dtype=torch.int32, device="cuda"), torch.arange(5, dtype=torch.int32, device="cuda")[None]
        q = torch.randn(n, 128 * share, 64, device="cuda").half()
        ecq.kv4_append(x[0], x[1], clean, slots, group_size=32)
        for which in (0, 1):
            y = x.clone()
            y[which, 66, 0, 3] = float("nan")  # in one of the heads
            ecq.kv4_append(y[0], y[1], pages, slots, group_size=32)
            starts = i32([0, n])
            got, want = (ecq.kv4_attention(q, p, table, i32([70]), starts, n, group_size=32) for p in (pages, clean))
            first = max(0, 66 - (70 - n))  # the first query that sees token 66
            assert torch.equal(got[:first], want[:first])
            assert torch.equal(got[:, share:], want[:, share:])
            seen, want = got[first:, :share], want[:, :share]
            if which == 0:
                assert bool(seen.isnan().all())
            else:  # the value's group of channels
                assert bool(seen[..., :32].isnan().all()) and torch.equal(seen[..., 32:], want[first:, :, 32:])


def test_a_scale_that_is_infinite_ends_and_stays_with_the_rows_that_see_it():
    # bytes that kv4_append never writes: token 40's V scales are infinite
    for lens, new, heads in (([100, 60], [1, 1], 2), ([100, 60], [60, 50], 64)):
        q, pages, table, starts, want = attend_case(lens, new, heads, 2, 64, 32, 16, torch.float16)
        broken, at = pages.clone(), int(table[0, 2]) * 16 + 8
        par = broken.view(-1, heads, 16 * 64 + 256)[at // 16, :, 16 * 64 + 128:].view(torch.float16).view(heads, 16, 2, 2)
        par[:, at % 16, :, 0] = float("inf")
        got = ecq.kv4_attention(q, broken, table, i32(lens), None if new[0] == 1 else i32(starts), max(new), group_size=32)
        first = max(0, 40 - (100 - new[0]))  # the first query of request 0 that sees token 40
        assert torch.equal(got[:first], want[:first]) and torch.equal(got[starts[1]:], want[starts[1]:])
        assert not bool(got[first:starts[1]].isfinite().any())


def test_more_queries_than_max_q_are_reported():
    for new, heads, said in ((9, 2, 1), (200, 64, 40)):
        pages, table = fill([300], heads, 64, 32, 16, 3)
        q, status = torch.randn(new, 2 * heads, 64, device="cuda").half(), i32([0])
        ecq.kv4_attention(q, pages, table, i32([300]), i32([0, new]), said, group_size=32, status=status)
        assert status.item() == BADARG


def test_prompts_with_bad_pages_leave_their_keys_out():
    lens, new, dim, g, page = [200, 130], [100, 100], 64, 32, 16
    q, pages, table, starts, want = attend_case(lens, new, 100, 2, dim, g, page, torch.float16)
    bad, status = table.clone(), i32([0])
    bad[1, 8] = 2 ** 31 - 1  # tokens 128 and 129 of request 1: its last two queries lose them
    got = ecq.kv4_attention(q, pages, bad, i32(lens), i32(starts), 100, group_size=g, status=status)
    assert status.item() == BADARG
    assert torch.equal(got[:198], want[:198])
    short, s_abs, v_abs = reference(q, pages, table, [200, 128], [0, 100, 198], page, dim, g)
    check_attention(got[:198], short[:198], s_abs[:198], v_abs[:198], torch.float16, True)
    k = reference(q[198:], pages, table[1:], [128], [0, 1], page, dim, g)
    check_attention(got[198:199], k[0][:1], k[1][:1], k[2][:1], torch.float16, True)


def test_attention_of_long_contexts():
    attend_case([20011], [1], 2, 4, 128, 64, 64, torch.float16)
    attend_case([4099, 17, 9000], [2, 1, 4], 1, 8, 64, 64, 128, torch.bfloat16)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,g", LAYOUTS)
@pytest.mark.parametrize("lens,new,share", [([1, 300, 0, 77], [1, 1, 1, 1], 4), ([500, 33, 640], [4, 1, 3], 5), ([2000], [1], 1)])
def test_attention_with_room_for_long_requests(dtype, dim, g, lens, new, share):
    # tables with room for far more than the requests have: the work is cut into ranges, and cut pairs are joined
    q, pages, table, starts, got = attend_case(lens, new, 3, share, dim, g, 16, dtype, seed=sum(lens))
    wide = torch.full((len(lens), 20000), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    again = ecq.kv4_attention(q, pages, wide, i32(lens), i32(starts), max(new), group_size=g)
    want, s_abs, v_abs = reference(q, pages, table, lens, starts, 16, dim, g)
    check_attention(again, want, s_abs, v_abs, dtype)
    for _ in range(2):
        assert torch.equal(again, ecq.kv4_attention(q, pages, wide, i32(lens), i32(starts), max(new), group_size=g))


def test_attention_of_many_requests():
    # more than the threads of a CTA look at in one round
    rng = random.Random(3)
    lens = [rng.choice([0, 1, 15, 16, 17, 40]) for _ in range(300)]
    attend_case(lens, [1] * 300, 2, 2, 64, 32, 16, torch.float16)


def test_attention_with_peaked_and_flat_scores():
    attend_case([1000], [1], 2, 4, 128, 64, 16, torch.float16, q_scale=30.0)      # one key takes all
    attend_case([1000], [1], 2, 4, 128, 64, 16, torch.float16, q_scale=0.0)       # the mean of all values
    attend_case([300], [1], 1, 2, 64, 32, 16, torch.float16, scale=-0.7)
    attend_case([300], [1], 1, 2, 64, 32, 16, torch.float16, scale=0.0)
    attend_case([300], [1], 1, 2, 128, 32, 16, torch.bfloat16, q_scale=1e-6, scale=3e5)
    attend_case([300], [1], 1, 2, 128, 32, 16, torch.bfloat16, q_scale=1e6, scale=3e-7)


def test_attention_when_late_keys_dominate():
    # scores rise with the position: the running maximum moves all the way
    n, dim = 2000, 128
    pages = ecq.kv4_pages(-(-n // 16), 1, dim, 16, 64)
    k = torch.zeros(n, 1, dim, device="cuda")
    k[:, 0, 0] = torch.linspace(-40, 40, n, device="cuda")
    v = torch.randn(n, 1, dim, device="cuda")
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    ecq.kv4_append(k.half(), v.half(), pages, slots, group_size=64)
    table = torch.arange(pages.shape[0], dtype=torch.int32, device="cuda")[None]
    q = torch.ones(1, 2, dim, dtype=torch.float16, device="cuda")
    got = ecq.kv4_attention(q, pages, table, i32([n]), group_size=64, scale=1.0)
    check_attention(got, *reference(q, pages, table, [n], [0, 1], 16, dim, 64, 1.0), torch.float16)


def test_attention_of_extreme_values():
    n, dim = 200, 64
    pages = ecq.kv4_pages(-(-n // 16), 1, dim, 16, 32)
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    v = torch.randn(n, 1, dim, device="cuda") * 30000
    ecq.kv4_append(torch.randn(n, 1, dim, device="cuda").half(), v.clamp(-65504, 65504).half(), pages, slots, group_size=32)
    table = torch.arange(pages.shape[0], dtype=torch.int32, device="cuda")[None]
    q = torch.randn(1, 4, dim, device="cuda").half()
    got = ecq.kv4_attention(q, pages, table, i32([n]), group_size=32)
    assert bool(got.isfinite().all())
    check_attention(got, *reference(q, pages, table, [n], [0, 1], 16, dim, 32), torch.float16)


def test_attention_strides_and_rows_behind_the_last():
    lens, new, dim, g, page = [40, 70], [2, 3], 64, 32, 16
    q, pages, table, starts, want = attend_case(lens, new, 2, 2, dim, g, page, torch.float16)
    # q and out as parts of larger tensors, padded behind the last token; a wider table
    wide = torch.full((9, 3, 4, dim), 7.0, dtype=torch.float16, device="cuda")
    wide[:5, 1] = q
    out = torch.full((9, 4, dim + 8), -3.0, dtype=torch.float16, device="cuda")
    big = torch.full((2, 50), 2 ** 30, dtype=torch.int32, device="cuda")
    big[:, :table.shape[1]] = table
    got = ecq.kv4_attention(wide[:, 1], pages, big, i32(lens), i32(starts), 3, group_size=g, out=out[..., :dim])
    assert got.data_ptr() == out.data_ptr()
    assert float((out[:5, :, :dim].float() - want.float()).abs().max()) <= 2e-3 * float(want.abs().max())
    assert bool((out[5:] == -3.0).all()) and bool((out[..., dim:] == -3.0).all())


def test_attention_reports_bad_pages_and_lengths():
    lens, dim, g, page = [40, 40, 40], 64, 32, 16
    q, pages, table, _, want = attend_case(lens, [1, 1, 1], 1, 2, dim, g, page, torch.float16)
    status = i32([0])
    bad = table.clone()
    bad[1, 2] = pages.shape[0]        # the last 8 keys of request 1 are left out
    got = ecq.kv4_attention(q, pages, bad, i32(lens), group_size=g, status=status)
    assert status.item() == BADARG
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    short, s_abs, v_abs = reference(q, pages, table, [40, 32, 40], [0, 1, 2, 3], page, dim, g)
    check_attention(got, short, s_abs, v_abs, torch.float16)
    status.zero_()
    got = ecq.kv4_attention(q, pages, table, i32([40, 2 ** 31 - 1, 40]), group_size=g, status=status)
    assert status.item() == BADARG and torch.equal(got[0], want[0])
    status.zero_()
    got = ecq.kv4_attention(q, pages, table, i32([40, -9, 0]), group_size=g, status=status)
    assert torch.equal(got[0], want[0]) and not bool(got[1:].any())


def test_attention_gives_the_same_bits_again():
    a = attend_case([3000, 1, 800], [1, 1, 1], 2, 4, 128, 64, 64, torch.float16)
    for _ in range(3):
        again = ecq.kv4_attention(a[0], a[1], a[2], i32([3000, 1, 800]), group_size=64)
        assert torch.equal(again, a[4])


def test_python_refuses():
    pages, table = ecq.kv4_pages(4, 2, 64, 16, 32), torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    q, lens = torch.zeros(1, 4, 64, dtype=torch.float16, device="cuda"), i32([1])
    ok = dict(group_size=32)
    ecq.kv4_attention(q, pages, table, lens, **ok)
    for args, kw in [((q[:, :3], pages, table, lens), ok), ((q, pages, table, i32([1, 1])), ok), ((q.float(), pages, table, lens), ok),
                     ((q.transpose(1, 2), pages, table, lens), ok), ((q, pages, table.long(), lens), ok),
                     ((q, pages[..., :-16], table, lens), ok), ((q, pages, table, lens, i32([0])), ok),
                     ((q, pages, table, lens, None, 2), ok), ((q, pages, table, lens), dict(group_size=32, out=q[:, :2])),
                     ((q, pages, table, lens), dict(group_size=64)), ((q, pages, table, lens.cpu()), ok),
                     ((q[:0], pages, table, lens), ok)]:
        with pytest.raises((ValueError, EcqError)):
            ecq.kv4_attention(*args, **kw)
    k = torch.zeros(2, 2, 64, dtype=torch.float16, device="cuda")
    for args in [(k, k[:1], pages, i32([0, 1])), (k, k, pages, i32([0])), (k, k.bfloat16(), pages, i32([0, 1])),
                 (k[:, :1], k[:, :1], pages, i32([0, 1])), (k, k, pages, torch.tensor([0, 1], device="cuda")), (k[..., 1:], k[..., 1:], pages, i32([0, 1]))]:
        with pytest.raises((ValueError, EcqError)):
            ecq.kv4_append(*args, group_size=32)
    with pytest.raises(ValueError):
        ecq.kv4_gather(pages, i32([0]), 64, group_size=32, dtype=torch.float32)
    with pytest.raises(ValueError):
        ecq.kv4_extend(lens, i32([1, 2]), table, i32([0]), i32([1]), 16, 4)
    with pytest.raises(EcqError):
        ecq.kv4_extend(lens, lens, table, i32([0]), i32([1]), 20, 4)
    with pytest.raises(ValueError):
        ecq.kv4_release(lens, lens, table, i32([0]), i32([1]), 16)


# -- together ---------------------------------------------------------------------

def plain_attention(q, k, v, n_new):
    """float64 attention of the last n_new of k's tokens."""
    share = q.shape[1] // k.shape[1]
    kk, vv = k.double().repeat_interleave(share, 1), v.double().repeat_interleave(share, 1)
    s = torch.einsum("ihd,jhd->hij", q.double(), kk) * q.shape[2] ** -0.5
    seen = torch.arange(len(k), device="cuda") <= (len(k) - n_new + torch.arange(n_new, device="cuda"))[:, None]
    return torch.einsum("hij,jhd->ihd", torch.softmax(s.masked_fill(~seen, -float("inf")), -1), vv)


def test_a_server_run():
    """Prompts, steps, guesses, ends and new prompts through one cache of two
    layers: the rows that each request reads are its own, in order."""
    batch, heads, share, dim, layers = 5, 2, 2, 64, 2
    c = ecq.KV4Cache(layers, 40, heads, dim, batch, 200, page_size=16, group_size=32)
    rng, gen = random.Random(4), torch.Generator(device="cuda").manual_seed(4)
    hist = [[[] for _ in range(batch)] for _ in range(layers)]
    pad = 100  # 5 requests of at most 20 new tokens
    for step in range(8):
        new = [rng.randint(5, 20) if not len(hist[0][b]) else rng.choice([0, 1, 1, 3]) for b in range(batch)]
        st = c.extend(i32(new), pad)
        starts = st.q_starts.tolist()
        for layer in range(layers):
            qkv = torch.randn(pad, heads * (share + 2), dim, generator=gen, device="cuda").half()
            q, k, v = qkv[:, :heads * share], qkv[:, heads * share:-heads], qkv[:, -heads:]
            c.append(layer, k, v, st.slots)
            o = c.attention(layer, q, st.q_starts, 20, out=torch.zeros(pad, heads * share, dim, dtype=torch.float16, device="cuda"))
            kq, vq = (torch.from_numpy(quantise(x, 32)[1]).cuda() for x in (k, v))
            for b, n in enumerate(new):
                hist[layer][b] += [(kq[t], vq[t]) for t in range(starts[b], starts[b + 1])]
                if n:
                    kk, vv = (torch.stack(x) for x in zip(*hist[layer][b]))
                    want = plain_attention(q[starts[b]:starts[b + 1]], kk, vv, n)
                    assert float((o[starts[b]:starts[b + 1]].double() - want).abs().max()) <= 2.0 ** -11 * 4 + 2e-4
                    gk, gv = c.gather(layer, st.slots[starts[b]:starts[b + 1]].clone())
                    assert float((gk.double() - kk[-n:]).abs().max()) <= 2.0 ** -11 * 8
            assert not bool(o[starts[-1]:].any())
        done = [rng.random() < 0.3 for _ in range(batch)]
        c.release(torch.tensor(done, device="cuda"))
        for b in range(batch):
            if done[b]:
                for layer in range(layers):
                    hist[layer][b] = []
        c.check()
    assert c.seq_lens.tolist() == [len(h) for h in hist[0]]


def test_running_out_of_pages_raises_and_the_cache_stays_usable():
    c = ecq.KV4Cache(1, 2, 1, 64, 2, 64, page_size=16, group_size=32)
    c.extend(i32([20, 0]), 32)
    c.check()
    st = c.extend(i32([0, 1]), 32)  # both pages are taken
    assert st.q_starts.tolist() == [0, 0, 0]
    k = torch.ones(32, 1, 64, dtype=torch.float16, device="cuda")
    before = c.pages[0].clone()
    c.append(0, k, k, st.slots)     # stores nothing
    assert torch.equal(before, c.pages[0])
    with pytest.raises(EcqError, match="pages"):
        c.check()
    assert c.seq_lens.tolist() == [20, 0]
    c.release(torch.tensor([True, False], device="cuda"))
    c.extend(i32([0, 1]), 32)
    c.check()
    assert c.seq_lens.tolist() == [0, 1]


def test_a_captured_step_replays_with_other_requests():
    batch, heads, dim = 4, 2, 128
    def fresh():
        c = ecq.KV4Cache(1, 64, heads, dim, batch, 256, page_size=16, group_size=64)
        p = torch.randn(90, heads, dim, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").half()
        st = c.extend(i32([30, 0, 41, 19]), 90)
        c.append(0, p, p.flip(0), st.slots)
        return c

    def step(c, new, q, k, v, out):
        st = c.extend(new, 2 * batch)
        c.append(0, k, v, st.slots)
        return c.attention(0, q, st.q_starts, 2, out=out)

    a, b = fresh(), fresh()
    new = i32([1, 0, 2, 1])
    q, k, v = (torch.zeros(2 * batch, h, dim, dtype=torch.float16, device="cuda") for h in (2 * heads, heads, heads))
    out = torch.zeros_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(fresh(), new, q, k, v, out)  # warm up on a cache of its own
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step(a, new, q, k, v, out)
    torch.cuda.current_stream().wait_stream(side)
    gen = torch.Generator(device="cuda").manual_seed(9)
    for i in range(20):
        new.copy_(i32([[1, 0, 2, 1], [0, 2, 1, 1], [2, 2, 2, 2]][i % 3]))
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=gen, device="cuda"))
        out.zero_()
        graph.replay()
        eager = step(b, new, q, k, v, torch.zeros_like(out))
        assert torch.equal(out, eager)
        assert torch.equal(a.seq_lens, b.seq_lens) and torch.equal(a.block_table, b.block_table)
    a.check()
    b.check()


def test_two_streams_at_once():
    cases = [attend_case([2500, 900], [1, 1], 2, 4, 128, 64, 64, torch.float16, seed=s) for s in (1, 2)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (s, c) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                got[i].append(ecq.kv4_attention(c[0], c[1], c[2], i32([2500, 900]), group_size=64))
    torch.cuda.synchronize()
    for g, c in zip(got, cases):
        assert all(torch.equal(x, c[4]) for x in g)


# -- the decoder ------------------------------------------------------------------

def test_decoder_with_a_4bit_cache_matches_plain_attention_over_its_values():
    from ecq_b200.model import Llama7BConfig, Llama7BDecoder

    cfg = Llama7BConfig(layers=2, hidden=512, heads=4, head_dim=128, mlp=1024, vocab=1000, kv_len=100)
    a = Llama7BDecoder(cfg, tp=1, seed=5, kv_cache="int4")
    fp16 = Llama7BDecoder(cfg, tp=1, seed=5)
    tok = torch.tensor([17], device="cuda")
    got = a.step_logits(tok).float()
    a.check()
    cache, n = a.cache, cfg.kv_len + 1
    assert cache.seq_lens.tolist() == [n]
    pos = torch.arange(n, device="cuda")
    slots = (cache.block_table[0, pos // 64] * 64 + pos % 64).to(torch.int32)
    for li in range(cfg.layers):  # the rows are those of the fp16 cache, in 4 bits: half a step of the largest group
        for half, rows in enumerate(cache.gather(li, slots)):
            want = fp16.kv[li, half, :, :cfg.kv_len].transpose(0, 1).float()
            step = (want.amax() - want.amin()) / 15
            assert float((rows[:-1].float() - want).abs().max()) <= 0.5 * float(step) + 2.0 ** -8

    def plain(layer, q):
        k, v = cache.gather(layer, slots)
        return plain_attention(q, k, v, 1).half()

    cache.attention = plain
    want = a.step_logits(tok).float()
    assert float((got - want).abs().max() / want.abs().max()) <= 1e-2
    assert int(torch.argmax(got)) == int(torch.argmax(want))


def test_decoder_with_a_4bit_cache_in_a_graph():
    from ecq_b200.model import Llama7BConfig, Llama7BDecoder

    cfg = Llama7BConfig(layers=2, hidden=512, heads=4, head_dim=128, mlp=1024, vocab=1000, kv_len=64)
    dec = Llama7BDecoder(cfg, tp=1, seed=6, kv_cache="int4")
    tok = torch.tensor([3], device="cuda")
    eager = dec.step(tok)
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        dec.step(tok)
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            out = dec.step(tok)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    dec.check()
    assert int(out) == int(eager)
    with pytest.raises(ValueError):
        Llama7BDecoder(cfg, kv_cache="int8")
