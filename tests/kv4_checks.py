"""Bounds on the root-mean-square error of attention outputs, for tests that
shall see one key too many or too few.

They hold for scores of unit spread (q, k normal, scale 1 / sqrt(dim)) and values
without a common part. K, V and weights in fp16 are off by at most 2^-11 of
themselves, evenly: a root mean square of 2^-11 / sqrt(3) each, K's as that of a
score of size one. The errors of different keys are as independent as the values,
so the sum is off by as much of its own size: sqrt(3) 2^-11 / sqrt(3) = 2^-11 at
most over many rows, and the output's rounding adds eps / 2 / sqrt(3); twice that
is the bound of a head. In one row a single key may have most of the weight, with
its full roundings: 2^-11 for V and P each, and for its score four times the root
mean square, under 2.4 2^-11; then eps / 2."""
import torch


def bounds(dtype: torch.dtype) -> tuple[float, float]:
    """Of a head, of a row."""
    half = torch.finfo(dtype).eps / 2
    return 2 * (2.0 ** -11 + half / 3 ** 0.5), 4.4 * 2.0 ** -11 + half


def errors(got: torch.Tensor, want: torch.Tensor, heads: int) -> tuple[float, float]:
    """The error's root mean square over that of `want` [rows, heads * share, dim]:
    the largest of a cache head, and of one row of a query head. Rows of `want`
    that are 0 are left out."""
    err, size = ((x.double().square().sum(-1)) for x in (got.double() - want.double(), want))
    by_head = [x.unflatten(1, (heads, -1)).sum((0, 2)) for x in (err, size)]
    some = size > 0
    return float((by_head[0] / by_head[1]).max() ** 0.5), float((err[some] / size[some]).max() ** 0.5)


def within(got: torch.Tensor, want: torch.Tensor, heads: int, dtype: torch.dtype) -> bool:
    return all(e <= b for e, b in zip(errors(got, want, heads), bounds(dtype)))
