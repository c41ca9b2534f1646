"""A paged KV cache held in 4 bits, for serving many requests: block tables and
slot maps built on the GPU, K and V rows stored and read back, and attention
over the cache (include/ecq_kv4.h has the pool's layout).

One serving step of a layer stack::

    step = cache.extend(new_lens, max_tokens)      # once: pages, slots, positions
    for layer in ...:                              # k, v, q of the step's tokens
        cache.append(layer, k, v, step.slots)
        o = cache.attention(layer, q, step.q_starts, max_q)
    cache.release(done)                            # pages of finished requests

``KV4Cache`` holds the tensors; the ``kv4_*`` functions under it take plain
tensors. Calls run on the current stream of the tensors' device, allocate only
their results and workspaces (from torch's allocator, so they can be captured
into CUDA graphs) and do not synchronise. Bad values that only the device sees
set bits of the ``status`` word.

The calls are for inference: the cache's bytes carry no gradient to k and v, and
a backward pass through a result of ``kv4_attention`` to its q raises. What is
written into a tensor that the caller gives (``out``) carries none either.
"""
from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple

import torch

from . import _lib
from ._lib import EcqError, check, lib

_DTYPES = {torch.float16: 0, torch.bfloat16: 1}
_I32 = torch.int32
_U8 = torch.uint8
# the current stream's handle and the current device, without objects for them (a torch without CUDA has neither, and no
# tensor that would get here)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", None)


class KV4Step(NamedTuple):
    """What ``kv4_extend`` returns (int32 tensors)."""

    seq_lens: torch.Tensor    # [batch] lengths with the new tokens
    q_starts: torch.Tensor    # [batch + 1] first new token of each request, then their number
    slots: torch.Tensor       # [max_tokens] slot of each new token, -1 behind the last
    positions: torch.Tensor   # [max_tokens] position of each new token in its request, -1 behind the last
    free_count: torch.Tensor  # [1] pages left on the free stack


# A step of a small model is a few microseconds of GPU time per call, so the
# checks are written to cost little: plain comparisons, device numbers instead
# of device objects, sizes from a cache.

def _device(first: torch.Tensor, names: str, *others) -> int:
    """The device number that all tensors share."""
    d = first.get_device()
    if d < 0:
        raise ValueError("the 4-bit KV cache runs on CUDA tensors only")
    for i, t in enumerate(others):
        if t is not None and t.get_device() != d:
            raise ValueError(f"{names.split()[i]} is on {t.device}, not on {first.device}")
    return d


def _on(device: int, fn, *args) -> int:
    """fn(*args, stream) with `device` current (a launch needs that)."""
    if _current_device() == device:
        return fn(*args, _raw_stream(device))
    with torch.cuda.device(device):
        return fn(*args, _raw_stream(device))


def _fits(name: str, n: int, least: int = 0) -> None:
    """Counts are 32-bit integers in the library, and ctypes cuts larger ones off."""
    if not least <= n < 1 << 31:
        raise ValueError(f"{name} must be at least {least} and below 2^31, not {n}")


def _int32(name: str, t: torch.Tensor, n: int | None = None) -> None:
    if t.dtype != _I32 or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 with one dimension")
    if n is not None and t.shape[0] != n:
        raise ValueError(f"{name} must have {n} entries, not {t.shape[0]}")


def _table(block_table: torch.Tensor, batch: int) -> tuple[int, int]:
    """Row stride and columns."""
    if block_table.dtype != _I32 or block_table.dim() != 2 or block_table.shape[0] != batch:
        raise ValueError(f"block_table must be int32 [{batch}, pages per request]")
    cols = block_table.shape[1]
    stride, last = block_table.stride()
    if batch == 1 and stride < cols:  # a single row's stride says nothing
        stride = cols
    if cols < 1 or (last != 1 and cols > 1) or stride < cols:
        raise ValueError("block_table needs contiguous rows of at least one page")
    return stride, cols


def _status(status) -> int | None:
    if status is None:
        return None
    if status.dtype != _I32 or status.numel() < 1:
        raise ValueError("status must be int32 [1]")
    return status.data_ptr()


@lru_cache(maxsize=256)
def _tokens_per_page(page_bytes: int, head_dim: int, group_size: int) -> int:
    block = check(lib().ecq_kv4_page_bytes(head_dim, 16, group_size), f"head_dim {head_dim}, group_size {group_size}")
    size, rest = divmod(page_bytes, block)
    if rest or size not in (1, 2, 4, 8, 16):
        raise ValueError(f"pages of {page_bytes} bytes do not hold 16, 32, 64, 128 or 256 tokens of {block // 16} bytes")
    return 16 * size


def _page_size(pages: torch.Tensor, head_dim: int, group_size: int) -> int:
    """The tokens per page of a pool, from its shape."""
    if pages.dtype != _U8 or pages.dim() != 3 or not pages.is_contiguous():
        raise ValueError("pages must be contiguous uint8 [pages, kv_heads, page bytes]")
    return _tokens_per_page(pages.shape[2], head_dim, group_size)


@lru_cache(maxsize=256)
def _workspace_bytes(batch: int, heads: int, kv_heads: int, head_dim: int, max_q: int, max_pages: int, page_size: int,
                     device: int) -> int:
    return check(lib().ecq_kv4_attention_workspace_bytes(batch, heads, kv_heads, head_dim, max_q, max_pages, page_size),
                 "kv4_attention")


def _rows(name: str, t: torch.Tensor) -> tuple[int, int, int]:
    """Dtype code and the strides of tokens and heads."""
    code = _DTYPES.get(t.dtype)
    if t.dim() != 3 or code is None:
        raise ValueError(f"{name} must be float16 or bfloat16 [tokens, heads, head_dim]")
    token, head, last = t.stride()
    if t.shape[0] == 1:  # a dimension of one entry has no stride to speak of
        token = 0
    if t.shape[1] == 1:
        head = 0
    if t.numel() and (last != 1 or token % 8 or head % 8 or t.data_ptr() % 16):
        raise ValueError(f"{name}: head_dim must be contiguous, rows 16-byte aligned")
    return code, token, head


def kv4_pages(n_pages: int, kv_heads: int, head_dim: int, page_size: int = 64, group_size: int = 64,
              device="cuda") -> torch.Tensor:
    """An empty pool: uint8 [n_pages, kv_heads, page bytes]."""
    per = check(lib().ecq_kv4_page_bytes(head_dim, page_size, group_size),
                f"head_dim {head_dim}, page_size {page_size}, group_size {group_size}")
    if n_pages < 1 or kv_heads < 1 or n_pages * page_size >= 1 << 31:
        raise ValueError("a pool has at least one page and head, and fewer than 2^31 slots")
    return torch.zeros(n_pages, kv_heads, per, dtype=torch.uint8, device=device)


def kv4_extend(seq_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
               free_count: torch.Tensor, page_size: int, max_tokens: int, *, seq_lens_out: torch.Tensor | None = None,
               free_count_out: torch.Tensor | None = None, status: torch.Tensor | None = None) -> KV4Step:
    """The bookkeeping of a step on the GPU: request b grows from seq_lens[b]
    by new_lens[b] tokens (int32 [batch]). Pages that it did not have yet are
    popped off the end of free_pages[:free_count] into its row of block_table
    (in place); lengths and count come back as new tensors, or in
    ``seq_lens_out`` / ``free_count_out``, which may be seq_lens / free_count
    themselves and share memory with nothing else. At most
    ``max_tokens`` new tokens: ``slots`` and ``positions`` have that length,
    filled with -1 behind the last, so a captured step keeps its shapes. All
    or nothing: if pages, room or lengths do not suffice, or a page that a request
    goes on in or would get has no slots in int32, nothing changes, every slot is
    -1 and ``status`` says so."""
    _fits("max_tokens", max_tokens)
    _fits("page_size", page_size)
    device = _device(seq_lens, "new_lens block_table free_pages free_count seq_lens_out free_count_out status", new_lens,
                     block_table, free_pages, free_count, seq_lens_out, free_count_out, status)
    batch = seq_lens.shape[0] if seq_lens.dim() else 0
    _int32("seq_lens", seq_lens, batch)
    _int32("new_lens", new_lens, batch)
    _int32("free_pages", free_pages)
    _int32("free_count", free_count, 1)
    stride, cols = _table(block_table, batch)
    out = torch.empty(2 * batch + 2 + 2 * max_tokens, dtype=_I32, device=seq_lens.device)
    starts, slots, positions, lens_out, count_out = out.split_with_sizes((batch + 1, max_tokens, max_tokens, batch, 1))
    if seq_lens_out is not None:
        _int32("seq_lens_out", seq_lens_out, batch)
        lens_out = seq_lens_out
    if free_count_out is not None:
        _int32("free_count_out", free_count_out, 1)
        count_out = free_count_out
    at = out.data_ptr()
    check(_on(device, lib().ecq_kv4_extend, seq_lens.data_ptr(), new_lens.data_ptr(), lens_out.data_ptr(),
              block_table.data_ptr(), stride, cols, batch, page_size, free_pages.data_ptr(), free_pages.shape[0],
              free_count.data_ptr(), count_out.data_ptr(), at, at + 4 * (batch + 1), at + 4 * (batch + 1 + max_tokens),
              max_tokens, _status(status)), "kv4_extend")
    return KV4Step(lens_out, starts, slots, positions, count_out)


def kv4_release(done: torch.Tensor, seq_lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                free_count: torch.Tensor, page_size: int, *, seq_lens_out: torch.Tensor | None = None,
                free_count_out: torch.Tensor | None = None,
                status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Push the pages of the requests where ``done`` (bool [batch]) on
    free_pages (in place) and set their lengths to 0. Returns the lengths and
    the count of free pages, as new tensors or in the ``_out`` ones. All or
    nothing, as ``kv4_extend``; what lies behind the stack's end may change."""
    _fits("page_size", page_size)
    device = _device(seq_lens, "done block_table free_pages free_count seq_lens_out free_count_out status", done,
                     block_table, free_pages, free_count, seq_lens_out, free_count_out, status)
    batch = seq_lens.shape[0] if seq_lens.dim() else 0
    _int32("seq_lens", seq_lens, batch)
    if done.dtype not in (torch.bool, _U8) or done.dim() != 1 or done.shape[0] != batch or not done.is_contiguous():
        raise ValueError(f"done must be contiguous bool [{batch}]")
    _int32("free_pages", free_pages)
    _int32("free_count", free_count, 1)
    stride, cols = _table(block_table, batch)
    lens_out, count_out = seq_lens_out, free_count_out
    if lens_out is None and count_out is None:
        lens_out, count_out = torch.empty(batch + 1, dtype=_I32, device=seq_lens.device).split_with_sizes((batch, 1))
    elif lens_out is None:
        lens_out = torch.empty_like(seq_lens)
    elif count_out is None:
        count_out = torch.empty_like(free_count)
    if seq_lens_out is not None:
        _int32("seq_lens_out", lens_out, batch)
    if free_count_out is not None:
        _int32("free_count_out", count_out, 1)
    check(_on(device, lib().ecq_kv4_release, done.data_ptr(), seq_lens.data_ptr(), lens_out.data_ptr(),
              block_table.data_ptr(), stride, cols, batch, page_size, free_pages.data_ptr(), free_pages.shape[0],
              free_count.data_ptr(), count_out.data_ptr(), _status(status)), "kv4_release")
    return lens_out, count_out


def kv4_append(k: torch.Tensor, v: torch.Tensor, pages: torch.Tensor, slots: torch.Tensor, *, group_size: int = 64,
               status: torch.Tensor | None = None) -> None:
    """Store rows k, v [tokens, kv_heads, head_dim] (float16 or bfloat16, any
    strides with contiguous 16-byte aligned rows) in 4 bits at slots [tokens]
    (int32, distinct; negative: not stored). slots may be longer than k, as a
    padded step's are: the rest is not looked at."""
    code, k_token, k_head = _rows("k", k)
    _, v_token, v_head = _rows("v", v)
    if k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError("k and v must have one shape and type")
    _fits("the number of tokens", k.shape[0])
    device = _device(k, "v pages slots status", v, pages, slots, status)
    tokens, heads, dim = k.shape
    page_size = _page_size(pages, dim, group_size)
    if pages.shape[1] != heads:
        raise ValueError(f"k has {heads} heads, the pool {pages.shape[1]}")
    _int32("slots", slots)
    if slots.shape[0] < tokens:
        raise ValueError(f"slots must have at least {tokens} entries")
    check(_on(device, lib().ecq_kv4_append, k.data_ptr(), k_token, k_head, v.data_ptr(), v_token, v_head, code,
              pages.data_ptr(), pages.shape[0], heads, dim, page_size, group_size, slots.data_ptr(), tokens,
              _status(status)), "kv4_append")


def kv4_gather(pages: torch.Tensor, slots: torch.Tensor, head_dim: int, *, group_size: int = 64,
               dtype: torch.dtype = torch.float16,
               status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The rows at slots [n] (int32) as k, v [n, kv_heads, head_dim] of dtype:
    code * scale + zero, rounded once; zeros for negative slots."""
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError("dtype must be float16 or bfloat16")
    device = _device(pages, "slots status", slots, status)
    page_size = _page_size(pages, head_dim, group_size)
    _int32("slots", slots)
    n, heads = slots.shape[0], pages.shape[1]
    k, v = torch.empty((2, n, heads, head_dim), dtype=dtype, device=pages.device).unbind()
    check(_on(device, lib().ecq_kv4_gather, k.data_ptr(), v.data_ptr(), code, pages.data_ptr(), pages.shape[0], heads,
              head_dim, page_size, group_size, slots.data_ptr(), n, _status(status)), "kv4_gather")
    return k, v


class _NoBackward(torch.autograd.Function):
    """kv4_attention of a q that requires a gradient: the same output, which says so when one is asked for."""

    @staticmethod
    def forward(ctx, q, call):
        return call(q)

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError("kv4_attention has no backward pass: call it under torch.no_grad() or with q.detach()")


def kv4_attention(q: torch.Tensor, pages: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                  q_starts: torch.Tensor | None = None, max_q: int = 1, *, group_size: int = 64,
                  scale: float | None = None, out: torch.Tensor | None = None,
                  status: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(q . k * scale) v over the cache, for new tokens whose rows are in
    it already (``kv4_append`` before it).

    q [tokens, heads, head_dim] (float16 or bfloat16; heads a multiple of the
    pool's), seq_lens int32 [batch] with the new tokens counted, block_table
    int32 [batch, pages]. q_starts int32 [batch + 1] says which tokens are
    whose, at most max_q for one request; None: one each. They are the last of
    their request, each sees the tokens up to its own. scale: 1 / sqrt(head_dim)
    by default. Rows that see nothing (length 0) are 0; rows at or behind
    q_starts[-1] are left as they were in ``out``, whose rows must not share
    memory."""
    if q.requires_grad and out is None and torch.is_grad_enabled():
        return _NoBackward.apply(q, lambda q: kv4_attention(
            q, pages, block_table, seq_lens, q_starts, max_q, group_size=group_size, scale=scale, status=status))
    code, q_token, q_head = _rows("q", q)
    _fits("max_q", max_q, 1)
    device = _device(q, "pages block_table seq_lens q_starts out status", pages, block_table, seq_lens, q_starts, out, status)
    tokens, heads, dim = q.shape
    page_size = _page_size(pages, dim, group_size)
    n_pages, kv_heads, _ = pages.shape
    if heads % kv_heads or heads < kv_heads:
        raise ValueError(f"{heads} query heads do not share {kv_heads} cache heads evenly")
    _int32("seq_lens", seq_lens)
    batch = seq_lens.shape[0]
    stride, cols = _table(block_table, batch)
    if q_starts is not None:
        _int32("q_starts", q_starts, batch + 1)
    elif tokens != batch or max_q != 1:
        raise ValueError("without q_starts every request has one query")
    if out is None:
        if q.is_contiguous():
            out = torch.empty_like(q)
        else:
            out = torch.empty((tokens, heads, dim), dtype=q.dtype, device=q.device)
        o_token, o_head = heads * dim, dim
    else:
        if out.shape != q.shape or out.dtype != q.dtype:
            raise ValueError("out must have q's shape and type")
        o_token, o_head, last = out.stride()
        if tokens == 1:
            o_token = 0
        if heads == 1:
            o_head = 0
        if out.numel() and (last != 1 or o_token % 4 or o_head % 4 or out.data_ptr() % 8):
            raise ValueError("out: head_dim must be contiguous, rows 8-byte aligned")
        if (tokens > 1 and o_token < dim) or (heads > 1 and o_head < dim):
            raise ValueError("out: rows share memory")
    need = _workspace_bytes(batch, heads, kv_heads, dim, max_q, cols, page_size, device)
    ws = torch.empty(need, dtype=_U8, device=q.device) if need else None
    check(_on(device, lib().ecq_kv4_attention, q.data_ptr(), q_token, q_head, out.data_ptr(), o_token, o_head, code,
              pages.data_ptr(), n_pages, heads, kv_heads, dim, page_size, group_size, block_table.data_ptr(), stride, cols,
              seq_lens.data_ptr(), None if q_starts is None else q_starts.data_ptr(), batch, tokens, max_q,
              dim ** -0.5 if scale is None else scale, None if ws is None else ws.data_ptr(), need, _status(status)),
          "kv4_attention")
    return out


class KV4Cache:
    """The 4-bit KV cache of a layer stack: one pool per layer, and one block
    table, length vector and free stack for all of them."""

    def __init__(self, layers: int, n_pages: int, kv_heads: int, head_dim: int, max_batch: int, max_len: int,
                 page_size: int = 64, group_size: int = 64, device="cuda"):
        self.head_dim, self.page_size, self.group_size = head_dim, page_size, group_size
        self.pages = [kv4_pages(n_pages, kv_heads, head_dim, page_size, group_size, device) for _ in range(layers)]
        dev = self.pages[0].device
        if not 1 <= max_batch <= 8192 or max_len < 1:
            raise ValueError("a cache holds 1 to 8192 requests of at least one token")
        self.max_len = max_len
        self.seq_lens = torch.zeros(max_batch, dtype=torch.int32, device=dev)
        self.block_table = torch.full((max_batch, -(-max_len // page_size)), -1, dtype=torch.int32, device=dev)
        # popped from the end: page 0 goes first
        self.free_pages = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=dev)
        self.free_count = torch.full((1,), n_pages, dtype=torch.int32, device=dev)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)

    @property
    def nbytes(self) -> int:
        """Bytes of all layers' pools."""
        return sum(p.numel() for p in self.pages)

    def extend(self, new_lens: torch.Tensor, max_tokens: int) -> KV4Step:
        """``kv4_extend`` of the cache's requests, lengths and count in place."""
        return kv4_extend(self.seq_lens, new_lens, self.block_table, self.free_pages, self.free_count, self.page_size,
                          max_tokens, seq_lens_out=self.seq_lens, free_count_out=self.free_count, status=self.status)

    def release(self, done: torch.Tensor) -> None:
        """``kv4_release`` of the requests where ``done`` (bool [max_batch])."""
        kv4_release(done, self.seq_lens, self.block_table, self.free_pages, self.free_count, self.page_size,
                    seq_lens_out=self.seq_lens, free_count_out=self.free_count, status=self.status)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """``kv4_append`` into a layer's pool."""
        kv4_append(k, v, self.pages[layer], slots, group_size=self.group_size, status=self.status)

    def gather(self, layer: int, slots: torch.Tensor,
               dtype: torch.dtype = torch.float16) -> tuple[torch.Tensor, torch.Tensor]:
        """``kv4_gather`` from a layer's pool."""
        return kv4_gather(self.pages[layer], slots, self.head_dim, group_size=self.group_size, dtype=dtype,
                          status=self.status)

    def attention(self, layer: int, q: torch.Tensor, q_starts: torch.Tensor | None = None, max_q: int = 1,
                  scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """``kv4_attention`` over a layer's pool."""
        return kv4_attention(q, self.pages[layer], self.block_table, self.seq_lens, q_starts, max_q,
                             group_size=self.group_size, scale=scale, out=out, status=self.status)

    def check(self) -> None:
        """Synchronise and raise if a call found bad values or too few pages."""
        s = int(self.status.item())
        if s:
            self.status.zero_()
            what = [w for bit, w in ((_lib.STATUS_NO_PAGES, "the free pages did not suffice"),
                                     (_lib.STATUS_BADARG, "a length, slot or page number is out of range"),
                                     (_lib.STATUS_TIMEOUT, "a bounded wait gave up")) if s & bit]
            raise EcqError("4-bit KV cache: " + ", ".join(what or [f"status {s}"]))


__all__ = ["KV4Cache", "KV4Step", "kv4_pages", "kv4_extend", "kv4_release", "kv4_append", "kv4_gather", "kv4_attention"]
