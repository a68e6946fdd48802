"""Streams around a paged cache's own scratch (needs a B200): handles made on one stream and
used on another, and dropped while a stream still works on them."""
from __future__ import annotations

from ctypes import byref, c_void_p

import pytest

torch = pytest.importorskip("torch")

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]

from moe_sm100 import _lib  # noqa: E402
from moe_sm100.paged import PagedKVCache  # noqa: E402


def _tensors(pages: int = 40, seqs: int = 3) -> tuple:
    i32 = dict(dtype=torch.int32, device="cuda")
    k, v = (torch.zeros((1, pages, 2, 16, 64), dtype=torch.float16, device="cuda") for _ in range(2))
    return (k, v, torch.full((seqs, 8), -1, **i32), torch.zeros(seqs, **i32), torch.zeros(pages, **i32))


def _busy(a, times: int = 40) -> None:
    """Some tens of milliseconds of work on the current stream."""
    for _ in range(times):
        torch.matmul(a, a)


def test_a_handle_made_on_a_busy_stream_is_ready_for_others() -> None:
    a = torch.zeros((8192, 8192), device="cuda").half()
    tensors = _tensors()
    words = PagedKVCache(*tensors)._scratch.numel()
    torch.cuda.synchronize()
    maker, user = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(maker):
        stale = torch.full((words,), 13, dtype=torch.int32, device="cuda")
        maker.synchronize()
        del stale                     # the next scratch may lie there
        _busy(a)
        cache = PagedKVCache(*tensors)
    cache.status(stream=user)
    cache.reserve([1, 2], [20, 33], stream=user)
    cache.status(stream=user)
    cache.reserve([0, 0], [1, 1], stream=user)
    with pytest.raises(ValueError):
        cache.status(stream=user)
    assert cache.lengths.tolist() == [0, 20, 33]
    assert cache.block_table[1].tolist() == [0, 1] + [-1] * 6
    assert cache.block_table[2].tolist() == [2, 3, 4] + [-1] * 5


@pytest.mark.parametrize("current", [False, True])
def test_a_handle_dropped_while_a_stream_works_on_it(current: bool) -> None:
    """The scratch is not given to others before the stream is done with it."""
    a = torch.zeros((8192, 8192), device="cuda").half()
    tensors = _tensors()
    seqs, counts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([1, 2], [20, 33]))
    cache = PagedKVCache(*tensors)
    words = cache._scratch.numel()
    user = torch.cuda.Stream()
    user.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(user):
        _busy(a)
        if current:
            cache.reserve(seqs, counts)
    if not current:
        cache.reserve(seqs, counts, stream=user)
    del cache
    others = [torch.full((words,), 13, dtype=torch.int32, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    assert all((x == 13).all() for x in others)
    assert tensors[3].tolist() == [0, 20, 33]


def test_a_stream_made_elsewhere_may_be_gone_when_the_cache_is() -> None:
    tensors = _tensors()
    seqs, counts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([1, 2], [20, 33]))
    cache = PagedKVCache(*tensors)
    handle = c_void_p()
    _lib.check(_lib.lib().moe_rt_stream_create(byref(handle)))
    torch.cuda.synchronize()
    cache.reserve(seqs, counts, stream=handle.value)
    cache.status(stream=handle.value)
    _lib.check(_lib.lib().moe_rt_stream_destroy(handle))
    lengths = tensors[3].tolist()
    del cache, tensors
    torch.zeros(1 << 20, device="cuda")
    torch.cuda.synchronize()
    assert lengths == [0, 20, 33]


def test_torch_streams_are_told_from_others() -> None:
    """What the cache goes by: torch's own streams have odd numbers, the default one 0."""
    assert torch.cuda.default_stream().stream_id == 0
    assert all(torch.cuda.Stream(priority=p).stream_id & 1 for p in (0, -1) for _ in range(40))
    handle = c_void_p()
    _lib.check(_lib.lib().moe_rt_stream_create(byref(handle)))
    other = torch.cuda.ExternalStream(handle.value)
    with torch.cuda.stream(other):
        number = torch.cuda.current_stream().stream_id
    assert number != 0 and not number & 1
    _lib.check(_lib.lib().moe_rt_stream_destroy(handle))


def test_a_cache_over_memory_that_is_not_torchs() -> None:
    lib = _lib.lib()
    ptr = c_void_p()
    shape = (1, 40, 2, 16, 64)
    _lib.check(lib.moe_rt_malloc(40 * 2 * 16 * 64 * 2, byref(ptr)))

    class Pool:
        __cuda_array_interface__ = dict(shape=shape, typestr="<f2", data=(ptr.value, False), version=3)

    k = torch.as_tensor(Pool(), device="cuda")
    assert k.data_ptr() == ptr.value
    k.zero_()
    cache = PagedKVCache(k, *_tensors()[1:])
    side = torch.cuda.Stream()
    row = torch.ones((3, 2, 64), dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    cache.reserve([1], [3], stream=side)
    cache.append(row, row, [1], [0, 3], stream=side)
    cache.status(stream=side)
    assert k.sum().item() == 3 * 2 * 64
    cache.close()
    del cache, k
    torch.cuda.synchronize()
    _lib.check(lib.moe_rt_free(ptr))
