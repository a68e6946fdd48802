"""Compaction of a paged cache in states and calls at its edge (needs a B200)."""
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


@pytest.mark.parametrize("other", [False, True])
def test_a_page_that_nobody_holds_has_no_place_after_compaction(other: bool) -> None:
    """A block table that names a page without references: compaction drops it, in place and
    into another pool alike, whatever the calls before left in the scratch."""
    cache, o = _pair(1, 40, 16, 1, 64, 4, 6)
    for c in (cache, o):
        c.reserve([0, 1, 2, 3], [90, 50, 96, 10])
        c.truncate([0, 2], [0, 20])
    cache.copy_pages([6, 6], [30, 31])       # other numbers in the scratch
    o.table[0][:3] = [30, 31, 2]             # pages that are free
    cache.block_table[0, :3] = torch.tensor([30, 31, 2], dtype=torch.int32, device="cuda")
    if other:
        into, oi = _pair(1, 20, 16, 1, 64, 4, 6)
        cache.compact(into=into)
        o.compact(oi)
        cache.status()
        _same_tables(into, oi)
    else:
        cache.compact()
        o.compact()
        cache.status()
        _same_tables(cache, o)
