"""Compaction of a paged cache: calls that must not touch it (needs a B200)."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]

from test_gpu_paged import _pair, _same_tables  # noqa: E402


def test_compact_into_a_closed_cache_is_refused() -> None:
    cache, o = _pair(1, 10, 16, 1, 64, 4, 6)
    for c in (cache, o):
        c.reserve([0, 1, 2], [20, 33, 5])
        c.truncate([0], [0])
    into, _ = _pair(1, 10, 16, 1, 64, 4, 6)
    into.close()
    with pytest.raises(ValueError):
        cache.compact(into=into)
    cache.status()
    _same_tables(cache, o)                   # not compacted in place instead
    cache.close()
    with pytest.raises(ValueError):
        cache.compact()
