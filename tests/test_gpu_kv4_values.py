"""Attention over the 4-bit KV cache where values, scores or lengths are at the
ends of their ranges, and with a bound on the error that one key too many or too
few does not pass."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import ecq_b200 as ecq  # noqa: E402
from kv4_checks import bounds, errors, within  # noqa: E402
from test_gpu_kv4 import BADARG, DTYPES, LAYOUTS, check_attention, decode, fill, i32, reference  # noqa: E402


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
    # what kv4_append never writes: scales of 60000, so values up to 900000. They count as fp16's end.
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
        assert bool(got.isfinite().all())
        if v:
            assert torch.equal(got[first:, :, 32:], want[first:, :, 32:])
            kk, vv = (torch.from_numpy(x[1][:n]).cuda().clamp(-65504, 65504).repeat_interleave(share, 1) for x in decode(pages, dim, g))
            seen = torch.arange(n, device="cuda") <= n - new + torch.arange(new, device="cuda")[:, None]
            s = torch.einsum("ihd,jhd->hij", q.double(), kk) * dim ** -0.5
            exact = torch.einsum("hij,jhd->ihd", torch.softmax(s.masked_fill(~seen, -float("inf")), -1), vv)
            # the token's weight: off by 2^-11 and twice what K's rounding, 2^-11 of |q| |k| <= 16, makes of a score
            tol = exact.abs() * (torch.finfo(torch.bfloat16).eps / 2 + 34 * 2.0 ** -11) + 34 * 2.0 ** -11 * 8
            assert bool(((got.double() - exact).abs() <= tol)[first:, :, :32].all())


# -- weights times scales past fp16's end ---------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,g", LAYOUTS)
@pytest.mark.parametrize("share", [1, 4, 9])
@pytest.mark.parametrize("score", [1.0, 2.0 ** 20, 2.0 ** 25])
def test_large_values_after_small_ones(dtype, dim, g, share, score):
    """One key for all tokens, so the mean of the values, of which every other
    256 tokens' are large: a warp's sums of small ones meet weights that their
    scales carry out of fp16, at references of which 10 is less than a step."""
    heads, n, page = 32, 2500, 64
    k = torch.ones(n, heads, dim, device="cuda")
    big = (torch.arange(n, device="cuda") // 256 % 2 == 1)[:, None, None]
    v = torch.where(big, 20000.0, 2000.0) * randn(n, heads, dim, seed=dim)
    if dtype == torch.float16:
        k *= max(1.0, score / 1024)
    pages, table = store(k.to(dtype), v.clamp(-60000, 60000).to(dtype), page, g)
    wide = torch.full((1, 2000), -1, dtype=torch.int32, device="cuda")  # room for far more: ranges
    wide[:, :table.shape[1]] = table
    q = torch.full((1, heads * share, dim), (score if dtype == torch.bfloat16 else min(score, 1024.0)) * 1.3125 / dim ** 0.5, device="cuda").to(dtype)
    value = torch.from_numpy(decode(pages, dim, g)[1][1]).cuda()[:n]
    want = value.mean(0).repeat_interleave(share, 0)[None]
    # equal weights stay equal. A weight's product with a scale is rounded to fp16, once for bf16: 2^-11 of what it adds,
    # evenly and independently: codes times scales of at most twice the largest value, over n tokens (six times the root mean
    # square). fp32 sums of n such terms: 2^-24 sqrt(n) of the largest
    tol = want.abs() * torch.finfo(dtype).eps / 2 + (6 * 2.0 ** -11 / 3 ** 0.5 * n ** -0.5 + 2.0 ** -24 * n ** 0.5) * 2 * value.abs().max()
    for tb in (wide, table):
        got = ecq.kv4_attention(q, pages, tb, i32([n]), group_size=g)
        assert bool(((got.double() - want).abs() <= tol).all()), float(((got.double() - want).abs() / tol).max())


# -- scores of any size -------------------------------------------------------------

FORMS = [(1, 4, 1, 1), (1, 4, 1, 5000), (2, 9, 3, 1), (64, 2, 60, 1)]  # heads, share, queries, room in the table: streamed (clusters, ranges, two tiles), prompt


def one_hot(heads, share, new, room, dtype, dim, exponents, sign, seed):
    """Queries of one direction and many sizes, keys of which token 5 is the
    best by far: each output is that token's value."""
    n, g, page = 100, 32, 16
    way = torch.randint(1, 9, (dim,), generator=torch.Generator().manual_seed(seed)).cuda().float()
    k, v = randn(n, heads, dim, seed=seed).abs() + 1, randn(n, heads, dim, seed=seed + 1)
    k[5] = 8.0 if sign > 0 else 0.125
    pages, table = store(k.to(dtype), v.to(dtype), page, g)
    wide = torch.full((1, max(room, table.shape[1])), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    rows = new * heads * share
    size = sign * 2.0 ** torch.tensor([exponents[i % len(exponents)] for i in range(rows)], dtype=torch.float64, device="cuda")
    q = (size[:, None] * way.double()).view(new, heads * share, dim).to(dtype)
    assert bool(q.isfinite().all())
    got = ecq.kv4_attention(q, pages, wide, i32([n]), i32([0, new]), new, group_size=g)
    want = torch.from_numpy(decode(pages, dim, g)[1][1]).cuda()[5].repeat_interleave(share, 0).expand(new, -1, -1)
    # the other keys' weights are 0 in float64 too. V and the weight are rounded to fp16 at most, or the weight times V's
    # scale, which a code of up to 15 makes 2^-11 of the group's range, twice the largest value; then the output.
    err = (got.double() - want).abs()
    assert bool((err <= want.abs() * torch.finfo(dtype).eps / 2 + 3 * 2.0 ** -11 * want.abs().max()).all()), float(err.max())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype,exponents", [(torch.float16, (6, 9, 12)), (torch.bfloat16, (16, 18, 20, 21)), (torch.bfloat16, (30, 60, 80, 90)), (torch.bfloat16, (96, 99, 102))])
def test_scores_that_fp32_cannot_tell_from_their_neighbours(dim, form, dtype, exponents):
    one_hot(*form, dtype, dim, exponents, 1.0, 7)
    one_hot(*form, dtype, dim, exponents, -1.0, 9)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("exponent", range(0, 29, 2))
def test_large_scores_that_are_equal(form, dtype, exponent):
    """One key for all tokens: the mean of the values that a query sees, however
    large the score (2^exponent times 16 to 30) is."""
    heads, share, new, room = form
    n, dim, g, page = 90, 64, 32, 16
    k = torch.ones(n, heads, dim, device="cuda")
    if dtype == torch.float16:
        k *= 2.0 ** max(0, exponent - 13)
        exponent = min(exponent, 13)
    pages, table = store(k.to(dtype), randn(n, heads, dim, seed=exponent).to(dtype), page, g)
    wide = torch.full((1, max(room, table.shape[1])), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    # odd multiples, so that the products with log2(e) are none that fp32 holds exactly
    q = (2.0 ** exponent * (16 + torch.arange(new * heads * share, device="cuda") % 15)[:, None].expand(-1, dim) / 8).view(new, heads * share, dim).to(dtype)
    got = ecq.kv4_attention(q, pages, wide, i32([n]), i32([0, new]), new, group_size=g)
    v = torch.from_numpy(decode(pages, dim, g)[1][1]).cuda()[:n]
    mean = v.cumsum(0)[n - new:] / torch.arange(n - new + 1, n + 1, device="cuda")[:, None, None]
    want = mean.repeat_interleave(share, 1)
    # equal weights in fp16 are equal; V (and V's scale times a weight) is off by 2^-11 of the largest, and the output is rounded
    tol = want.abs() * torch.finfo(dtype).eps / 2 + 3 * 2.0 ** -11 * v.abs().max()
    assert bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("first", [0, 70])
def test_moderate_scores_beside_huge_negative_ones(form, dtype, first):
    # tokens from `first` on, 20 of them, are out of reach; the others' softmax is as without them
    heads, share, new, room = form
    n, dim, g, page = 150, 64, 32, 16
    k, v = randn(n, heads, dim, seed=1), randn(n, heads, dim, seed=2)
    k[:, :, 0] = 0.0
    k[first:first + 20, :, 0] = -60000.0
    pages, table = store(k.to(dtype), v.to(dtype), page, g)
    wide = torch.full((1, max(room, table.shape[1])), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    q = randn(new, heads * share, dim, seed=3)
    q[..., 0] = 2000.0
    q = q.to(dtype)
    got = ecq.kv4_attention(q, pages, wide, i32([n]), i32([0, new]), new, group_size=g)
    (_, kk), (_, vv) = decode(pages, dim, g)
    seen = torch.arange(n, device="cuda") <= n - new + torch.arange(new, device="cuda")[:, None]
    seen &= (torch.arange(n, device="cuda") < first) | (torch.arange(n, device="cuda") >= first + 20)
    kk, vv = (torch.from_numpy(x[:n]).cuda().repeat_interleave(share, 1) for x in (kk, vv))
    s = torch.einsum("ihd,jhd->hij", q.double(), kk) * dim ** -0.5
    want = torch.einsum("hij,jhd->ihd", torch.softmax(s.masked_fill(~seen, -float("inf")), -1), vv)
    # The other channels' |q| |k| come to under 128, over 8: with K off by 2^-11 of itself a score is off by 16 2^-11 and an
    # output by twice that of |v|; V and weights (codes times scales: twice the largest |v|) are off by 2^-11 each.
    tol = want.abs() * torch.finfo(dtype).eps / 2 + (2 * 16 + 4) * 2.0 ** -11 * vv.abs().max()
    assert bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_queries_of_any_size(dim, form, sign):
    one_hot(*form, torch.bfloat16, dim, [124, 122, 119, 116, 114, 110, 104, 100, 95, 60, 20], sign, 7)


# -- what only the device sees --------------------------------------------------------

@pytest.mark.parametrize("heads,new,room", [(1, 1, 1), (1, 1, 5000), (2, 9, 1), (64, 60, 1)])
@pytest.mark.parametrize("page,entry", [(16, -1), (64, -1), (16, -2 ** 31), (16, -2 ** 31 + 1), (64, -2 ** 31 + 1), (256, -2 ** 31)])
def test_negative_page_numbers_are_reported_and_left_out(heads, new, room, page, entry):
    # the last page of the table is bad: the answer is that of a request without its keys
    share, dim, g = 2, 64, 32
    n = 4 * page + 9
    pages, table = store(randn(n, heads, dim, seed=1).half(), randn(n, heads, dim, seed=2).half(), page, g)
    wide = torch.full((1, max(room, table.shape[1])), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    q, status = randn(new, heads * share, dim, seed=3).half(), i32([0])
    bad = wide.clone()
    bad[0, 4] = entry
    got = ecq.kv4_attention(q, pages, bad, i32([n]), i32([0, new]), new, group_size=g, status=status)
    assert status.item() == BADARG
    for i in range(new):
        last = min(n - new + i + 1, 4 * page)
        want = reference(q[i:i + 1], pages, table, [last], [0, 1], page, dim, g)
        check_attention(got[i:i + 1], *want, torch.float16, new * share > 70)


@pytest.mark.parametrize("heads,new,room", [(1, 1, 1), (1, 1, 5000), (64, 60, 1)])
@pytest.mark.parametrize("length", [-1, -2 ** 31])
def test_negative_lengths_are_reported_and_their_rows_zero(heads, new, room, length):
    dim, g, n = 64, 32, 70
    pages, table = store(randn(n, heads, dim, seed=1).half(), randn(n, heads, dim, seed=2).half(), 16, g)
    wide = torch.full((2, max(room, table.shape[1])), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    q, status = randn(2 * new, 2 * heads, dim, seed=3).half(), i32([0])
    starts = i32([0, new, 2 * new])
    want = ecq.kv4_attention(q, pages, wide, i32([n, 0]), starts, new, group_size=g, status=status)
    assert status.item() == 0
    got = ecq.kv4_attention(q, pages, wide, i32([n, length]), starts, new, group_size=g, status=status)
    assert status.item() == BADARG and torch.equal(got, want) and not bool(got[new:].any())


# -- one key too many or too few ------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,g", LAYOUTS)
@pytest.mark.parametrize("lens,new,heads,share,page", [
    ([1500], [130], 80, 8, 64), ([300, 5, 64], [257, 1, 64], 64, 2, 16), ([128, 129, 191, 192, 193], [128, 65, 100, 64, 193], 64, 1, 32),
    ([2500, 700], [300, 400], 8, 4, 256)])                                # prompts
def test_prompts_see_all_their_keys_and_no_others(dtype, dim, g, lens, new, heads, share, page):
    exactly(lens, new, heads, share, dim, g, page, dtype, 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,g", LAYOUTS)
@pytest.mark.parametrize("lens,new,heads,share,page,room", [
    ([2049], [1], 8, 1, 64, 1), ([700, 64, 65, 999], [1, 1, 1, 1], 2, 7, 16, 1), ([6000, 129], [1, 1], 2, 4, 64, 2000),
    ([1500, 400, 64], [6, 3, 5], 8, 4, 32, 1), ([1500, 400, 640], [6, 3, 5], 2, 4, 32, 4000)])
def test_steps_see_all_their_keys_and_no_others(dtype, dim, g, lens, new, heads, share, page, room):
    exactly(lens, new, heads, share, dim, g, page, dtype, room)


def exactly(lens, new, heads, share, dim, g, page, dtype, room):
    pages, table = fill(lens, heads, dim, g, page, sum(lens), dtype)       # keys and values without a common part
    wide = torch.full((len(lens), max(room, table.shape[1])), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = randn(starts[-1], heads * share, dim, seed=7).to(dtype)
    got = ecq.kv4_attention(q, pages, wide, i32(lens), i32(starts), max(new), group_size=g)
    want = reference(q, pages, table, lens, starts, page, dim, g)[0]
    for b in range(len(lens)):
        at = slice(starts[b], starts[b + 1])
        assert within(got[at], want[at], heads, dtype), (b, errors(got[at], want[at], heads), bounds(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("share", [1, 4, 9])
def test_the_largest_scales_at_large_scores(dtype, share):
    """Bytes that kv4_append never writes: scales near fp16's end, codes of 1, at
    references whose step is 8, so that weights are up to 2^14."""
    heads, n, dim, g = 2, 64, 64, 32
    k = torch.full((n, heads, dim), 1024.0, device="cuda").to(dtype)
    pages, table = store(k, randn(n, heads, dim, seed=1).to(dtype), 16, g)
    blocks = pages.view(-1, heads, 16 * 64 + 256)
    blocks[:, :, 512:1024] = 0x11                                                 # V codes
    par = blocks[:, :, 1152:].contiguous().view(torch.float16).view(-1, heads, 16, 2, 2)
    par[..., 0], par[..., 1] = 60000.0, -60000.0 + 32 * torch.arange(16, device="cuda")[:, None]
    blocks[:, :, 1152:] = par.view(torch.uint8).view(-1, heads, 128)
    value = torch.from_numpy(decode(pages, dim, g)[1][1]).cuda()
    # scores whose products lie 3.4 and more above a multiple of 8: with the reference 10 below, rounded, weights are 2^13.4 to 2^14
    for size in (5792.0, 6208.0, 7040.0, 8704.0, 10240.0):
        q = torch.full((1, heads * share, dim), size, device="cuda").to(dtype)
        got = ecq.kv4_attention(q, pages, table, i32([n]), group_size=g)
        want = value.mean(0).repeat_interleave(share, 0)[None]
        # a weight times a scale: rounded to fp16 once for bf16; else its rest too, of 2^-12 times 2^-15 2^13, to 2^-25: 2^-23 of
        # the weight, and that product to 2^-11 of itself: under 2^-20 together, of 60000
        tol = want.abs() * torch.finfo(dtype).eps / 2 + 60000 * (2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -20)
        assert bool(((got.double() - want).abs() <= tol).all()), (size, float((got.double() - want).abs().max()))
