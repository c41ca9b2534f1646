"""Refusals of the 4-bit KV cache's entry points that need no device: argument
checks of the C ABI (returned before anything is launched; the pointers are
never dereferenced) and of the Python functions."""
import pytest

from ecq_b200 import _lib

ARG, UNSUPPORTED, WORKSPACE = -1, -8, -9


def test_page_bytes():
    L = _lib.lib()
    assert L.ecq_kv4_page_bytes(128, 16, 64) == 16 * 128 + 128 * 2
    assert L.ecq_kv4_page_bytes(64, 256, 32) == 16 * (16 * 64 + 128 * 2)
    for dim, page, g in ((96, 16, 32), (128, 24, 64), (128, 512, 64), (128, 8, 64), (64, 16, 128), (128, 16, 16), (128, 0, 64)):
        assert L.ecq_kv4_page_bytes(dim, page, g) == UNSUPPORTED


def _extend(**kw):
    a = dict(lens=16, new=16, out=16, table=16, stride=4, cols=4, batch=2, page=16, free=16, cap=8, count=16, count_out=16,
             starts=16, slots=16, pos=16, tokens=3)
    a.update(kw)
    return _lib.lib().ecq_kv4_extend(*a.values(), None, None)


@pytest.mark.parametrize("kw,rc", [
    (dict(lens=None), ARG), (dict(new=None), ARG), (dict(out=None), ARG), (dict(table=None), ARG), (dict(count=None), ARG),
    (dict(count_out=None), ARG), (dict(starts=None), ARG), (dict(slots=None), ARG), (dict(pos=None), ARG),
    (dict(free=None), ARG), (dict(cap=-1), ARG), (dict(batch=0), ARG), (dict(tokens=-1), ARG), (dict(cols=0), ARG),
    (dict(stride=3), ARG), (dict(page=17), ARG), (dict(page=8), ARG), (dict(page=512), ARG),
    (dict(cols=1 << 27, stride=1 << 27), ARG), (dict(batch=8193), UNSUPPORTED)])
def test_extend_refuses(kw, rc):
    assert _extend(**kw) == rc


def _release(**kw):
    a = dict(done=16, lens=16, out=16, table=16, stride=4, cols=4, batch=2, page=16, free=16, cap=8, count=16, count_out=16)
    a.update(kw)
    return _lib.lib().ecq_kv4_release(*a.values(), None, None)


@pytest.mark.parametrize("kw,rc", [
    (dict(done=None), ARG), (dict(lens=None), ARG), (dict(out=None), ARG), (dict(table=None), ARG), (dict(free=None), ARG),
    (dict(count=None), ARG), (dict(count_out=None), ARG), (dict(batch=0), ARG), (dict(stride=3), ARG), (dict(page=40), ARG),
    (dict(batch=8193), UNSUPPORTED)])
def test_release_refuses(kw, rc):
    assert _release(**kw) == rc


def _append(**kw):
    a = dict(k=16, kt=1024, kh=128, v=16, vt=1024, vh=128, dtype=0, pages=16, n=4, heads=8, dim=128, page=16, g=64, slots=16, tokens=1)
    a.update(kw)
    return _lib.lib().ecq_kv4_append(*a.values(), None, None)


@pytest.mark.parametrize("kw,rc", [
    (dict(k=None), ARG), (dict(v=None), ARG), (dict(slots=None), ARG), (dict(pages=None), ARG), (dict(k=8), ARG),
    (dict(v=24), ARG), (dict(pages=8), ARG), (dict(kt=1028), ARG), (dict(vh=4), ARG), (dict(n=0), ARG), (dict(heads=0), ARG),
    (dict(tokens=-1), ARG), (dict(n=1 << 27), ARG), (dict(dim=80), UNSUPPORTED), (dict(g=48), UNSUPPORTED),
    (dict(page=48), UNSUPPORTED), (dict(dtype=2), UNSUPPORTED)])
def test_append_refuses(kw, rc):
    assert _append(**kw) == rc


def test_nothing_to_do_is_no_error():
    assert _append(tokens=0, k=None, v=None, slots=None) == 0
    assert _attention(total=0, q=None, out=None, starts=16) == 0


def _attention(**kw):
    a = dict(q=16, qt=1024, qh=128, out=16, ot=1024, oh=128, dtype=0, pages=16, n=4, heads=8, kv_heads=8, dim=128, page=16, g=64,
             table=16, stride=4, cols=4, lens=16, starts=None, batch=2, total=2, max_q=1, scale=1.0, ws=16, ws_bytes=1 << 40)
    a.update(kw)
    return _lib.lib().ecq_kv4_attention(*a.values(), None, None)


@pytest.mark.parametrize("kw,rc", [
    (dict(q=None), ARG), (dict(out=None), ARG), (dict(pages=None), ARG), (dict(table=None), ARG), (dict(lens=None), ARG),
    (dict(q=8), ARG), (dict(out=4), ARG), (dict(qt=1020), ARG), (dict(oh=2), ARG), (dict(heads=12), ARG), (dict(heads=4), ARG),
    (dict(batch=0), ARG), (dict(total=3), ARG), (dict(max_q=2), ARG), (dict(max_q=0, starts=16), ARG), (dict(stride=3), ARG),
    (dict(cols=0), ARG), (dict(total=-1), ARG), (dict(n=0), ARG), (dict(heads=65, kv_heads=1), UNSUPPORTED),
    (dict(dim=256), UNSUPPORTED), (dict(g=256), UNSUPPORTED), (dict(page=20), UNSUPPORTED), (dict(dtype=-1), UNSUPPORTED)])
def test_attention_refuses(kw, rc):
    assert _attention(**kw) == rc


def test_attention_workspace_size_is_host_only():
    size = _lib.lib().ecq_kv4_attention_workspace_bytes
    assert size(1, 32, 8, 128, 1, 4096, 64) >= 0
    assert size(0, 32, 8, 128, 1, 4096, 64) == ARG and size(1, 32, 0, 128, 1, 4096, 64) == ARG
    assert size(1, 32, 8, 72, 1, 4096, 64) == UNSUPPORTED
    need = size(1, 32, 8, 128, 1, 4096, 64)
    if need:
        assert _attention(heads=32, kv_heads=8, batch=1, total=1, cols=4096, stride=4096, page=64, ws_bytes=need - 1) == WORKSPACE
        assert _attention(heads=32, kv_heads=8, batch=1, total=1, cols=4096, stride=4096, page=64, ws=None) == WORKSPACE


def test_python_refuses_cpu_tensors_and_sizes():
    torch = pytest.importorskip("torch")
    import ecq_b200 as ecq

    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    pages = ecq.kv4_pages(2, 1, 64, page_size=16, group_size=32, device="cpu")
    assert tuple(pages.shape) == (2, 1, 16 * 64 + 256)
    rows = torch.zeros(1, 1, 64, dtype=torch.float16)
    for call in (lambda: ecq.kv4_extend(i32(1), i32(1), i32(1, 1), i32(1), i32(1), 16, 1),
                 lambda: ecq.kv4_release(torch.ones(1, dtype=torch.bool), i32(1), i32(1, 1), i32(1), i32(1), 16),
                 lambda: ecq.kv4_append(rows, rows, pages, i32(1), group_size=32),
                 lambda: ecq.kv4_gather(pages, i32(1), 64, group_size=32),
                 lambda: ecq.kv4_attention(rows, pages, i32(1, 1), i32(1), group_size=32)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(_lib.EcqError):
        ecq.kv4_pages(2, 1, 96, device="cpu")
    with pytest.raises(ValueError):
        ecq.kv4_pages(1 << 26, 1, 64, page_size=64, device="cpu")
