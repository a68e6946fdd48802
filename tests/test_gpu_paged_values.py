"""Values that attention over the paged cache has to keep apart (needs a B200): what a page
holds past a sequence's end, NaN and infinities, maxima that grow along the keys."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]

from moe_sm100.paged import PagedKVCache  # noqa: E402
from oracle.paged_oracle import attend_chunk  # noqa: E402
from test_gpu_paged import DTYPES, _attend_case, _check_rows, _filled  # noqa: E402


# ------------------------------------------------------------------ past the end
@pytest.mark.parametrize("dtype,dim", [("f16", 128), ("bf16", 64)])
@pytest.mark.parametrize("heads,kv_heads", [(8, 8), (24, 2)])
@pytest.mark.parametrize("page", [16, 256])
def test_many_more_new_rows_than_tokens(dtype: str, dim: int, heads: int, kv_heads: int, page: int) -> None:
    """Rows without a token and rows with a few, in units of every size, next to long chunks
    (so that the shares hold whole units); the pages hold NaN past the tokens."""
    _attend_case(dtype, heads, kv_heads, dim, page,
                 [(10, 300), (5, 320), (1, 70), (64, 500), (65, 130), (2000, 1000), (0, 200)], seed=page + heads)


# ------------------------------------------------------------------ NaN and infinities
def _batch(dtype, heads, kv_heads, dim, page, work, seed):
    cache, o = _filled(dtype, page, kv_heads, dim, [n for n, _ in work], seed=seed)
    starts = [0] + np.cumsum([m for _, m in work]).tolist()
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = (1.5 * torch.randn((starts[-1], heads, dim), generator=g, device="cuda")).to(DTYPES[dtype])
    return cache, o, q, starts


def _key(cache, o, s: int, j: int) -> tuple[int, int]:
    return o.table[s][j // o.page], j % o.page


def _attend(cache, q, n, starts):
    out = torch.full_like(q, 3.0)
    lse = torch.full(q.shape[:2], 7.0, device="cuda")
    cache.attend(q, list(range(n)), starts, out=out, lse=lse)
    cache.status()
    return out.double().cpu().numpy(), lse.double().cpu().numpy()


# one batch that holds every size of unit whole, and lone sequences that every share cuts
NAN_WORK = [[(40, 1), (300, 1), (3, 3), (500, 20), (400, 70), (700, 100), (900, 300), (33, 33), (256, 256)],
            [(20011, 1)], [(9001, 20)], [(9001, 40)], [(6001, 100)], [(5000, 300)]]


@pytest.mark.parametrize("dtype,dim", [("f16", 128), ("bf16", 64)])
@pytest.mark.parametrize("work", NAN_WORK, ids=lambda w: f"{len(w)}x{w[-1][1]}")
def test_a_nan_query_gives_nan_in_its_own_row(dtype: str, dim: int, work: list) -> None:
    heads = 4
    cache, o, q, starts = _batch(dtype, heads, 2, dim, 16, work, seed=31)
    clean = q.double().cpu().numpy()
    bad = np.zeros(q.shape[:2], dtype=bool)
    for i in range(len(work)):
        for row, h in ((starts[i], 0), (starts[i + 1] - 1, heads - 1), ((starts[i] + starts[i + 1]) // 2, 1)):
            q[row, h, (7 * row) % dim] = float("nan")
            bad[row, h] = True
    got, lse = _attend(cache, q, len(work), starts)
    assert np.isnan(got[bad]).all() and np.isnan(lse[bad]).all()
    for i, s in enumerate(range(len(work))):  # the other rows as if nothing had happened
        a, b = starts[i], starts[i + 1]
        ref, ref_lse, _ = attend_chunk(clean[a:b], *o.cached(0, s), 1 / np.sqrt(dim))
        got[a:b][bad[a:b]], lse[a:b][bad[a:b]] = ref[bad[a:b]], ref_lse[bad[a:b]]
    _check_rows(got, lse, clean, o, list(range(len(work))), starts, 0, 1 / np.sqrt(dim), dtype)


@pytest.mark.parametrize("dtype,dim", [("f16", 128), ("bf16", 64)])
@pytest.mark.parametrize("work", NAN_WORK, ids=lambda w: f"{len(w)}x{w[-1][1]}")
@pytest.mark.parametrize("every", [False, True])
def test_a_nan_key_gives_nan_to_the_rows_that_see_it(dtype: str, dim: int, work: list, every: bool) -> None:
    """One NaN among a sequence's keys (one of its new tokens, so that some rows do not see
    it), or in all of them."""
    heads, scale = 4, 1 / np.sqrt(dim)
    cache, o, q, starts = _batch(dtype, heads, 2, dim, 16, work, seed=32)
    for s, (n, m) in enumerate(work):
        for j in range(n) if every else [n - 1 - m // 2]:
            page, slot = _key(cache, o, s, j)
            cache.k[0, page, 1, slot, 5] = float("nan")
            o.k[0, page, 1, slot, 5] = float("nan")
    got, lse = _attend(cache, q, len(work), starts)
    qq = q.double().cpu().numpy()
    for s in range(len(work)):
        a, b = starts[s], starts[s + 1]
        with np.errstate(invalid="ignore"):
            ref, ref_lse, _ = attend_chunk(qq[a:b], *o.cached(0, s), scale)
        gone = np.isnan(ref).any(axis=2)
        assert gone[-1, heads // 2:].all() and not gone[:, :heads // 2].any()
        assert np.isnan(got[a:b][gone]).all() and np.isnan(lse[a:b][gone]).all()
        assert np.isfinite(got[a:b][~gone]).all()
        # sizes and roundings as _check_rows derives them, of the rows that are left
        k = np.nan_to_num(o.cached(0, s)[0])
        size = max(scale * (np.abs(qq[a:b, h]) @ np.abs(k[:, h // 2]).T).max() for h in range(heads))
        e = dim * 2.0 ** -23 * size + 2.0 ** -21 * (1 + size) + len(k) * 2.0 ** -24
        u = torch.finfo(DTYPES[dtype]).eps / 2
        with np.errstate(invalid="ignore"):
            mag = attend_chunk(qq[a:b], k, o.cached(0, s)[1], scale)[2]
        tol = u * (mag + np.abs(ref)) * 1.01 + 2 * e * mag + torch.finfo(DTYPES[dtype]).tiny
        assert (np.abs(got[a:b] - ref) <= tol)[~gone].all()


@pytest.mark.parametrize("work", NAN_WORK, ids=lambda w: f"{len(w)}x{w[-1][1]}")
@pytest.mark.parametrize("value", [float("inf"), float("-inf")])
def test_infinite_scores(work: list, value: float) -> None:
    """exp(s - max) is NaN where the maximum is infinite: with keys of both signs scores of
    +inf, with keys of one sign nothing but -inf.  Other rows keep their results."""
    cache, o, q, starts = _batch("bf16", 4, 2, 64, 16, work, seed=33)
    cache.k[..., 3] = torch.where(cache.k[..., 3] == 0, 1, cache.k[..., 3]).abs()
    cache.k[:, :, 0, ::2, 3] *= -1           # kv head 0: both signs, kv head 1: one
    o.k[:] = cache.k.double().cpu().numpy()
    clean = q.double().cpu().numpy()
    for i in range(len(work)):
        q[starts[i + 1] - 1, 1:3, 3] = value
    got, lse = _attend(cache, q, len(work), starts)
    for i in range(len(work)):
        a, b = starts[i], starts[i + 1]
        seen_both = work[i][0] > 1
        if seen_both or value > 0:
            assert np.isnan(got[b - 1, 1]).all()
        assert np.isnan(got[b - 1, 2]).all()
        ref, ref_lse, _ = attend_chunk(clean[a:b], *o.cached(0, i), 0.125)
        got[b - 1, 1:3], lse[b - 1, 1:3] = ref[-1, 1:3], ref_lse[-1, 1:3]
    _check_rows(got, lse, clean, o, list(range(len(work))), starts, 0, 0.125, "bf16")


# ------------------------------------------------------------------ growing maxima
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("work", [[(1000, 100), (1300, 300), (300, 300), (1000, 5), (64, 64), (900, 129)],
                                  [(4000, 100)], [(4000, 300)], [(6000, 3)]],
                         ids=lambda w: f"{len(w)}x{w[-1][1]}")
def test_maxima_that_grow_along_the_keys(dtype: str, dim: int, work: list) -> None:
    """Scores that rise along the keys, by 0 to 20 powers of two every 64 keys, rows of
    different slopes side by side (in one warp): sums and outputs are rescaled at some tiles
    and not at others, 7.9 being just too little for one tile and enough for two."""
    heads, scale = 4, 1 / np.sqrt(dim)
    cache, o, q, starts = _batch(dtype, heads, 4, dim, 32, work, seed=35)
    for s, (n, _m) in enumerate(work):
        pos = torch.arange(n, device="cuda")
        pages = torch.tensor(o.table[s], device="cuda")[pos // 32]
        rise = 4.0 * ((pos % 1024) / 64.0)   # keys of f16: the slope begins again every 1024
        cache.k[0, pages, :, pos % 32, 0] = rise[:, None].to(DTYPES[dtype])
    o.k[:] = cache.k.double().cpu().numpy()
    slopes = torch.tensor([0.0, 9.0, 7.9, 20.0, -9.0, 3.0, 12.0], device="cuda")
    at = torch.arange(q.shape[0], device="cuda")[:, None] + 2 * torch.arange(heads, device="cuda")
    q[:, :, 0] = (slopes[at % 7] * np.log(2) / (scale * 4.0)).to(q.dtype)
    got, lse = _attend(cache, q, len(work), starts)
    _check_rows(got, lse, q.double().cpu().numpy(), o, list(range(len(work))), starts, 0, scale, dtype)


# ------------------------------------------------------------------ strided pools
@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [("f16", 12, 4, 128), ("bf16", 8, 8, 64)])
def test_strided_pools(dtype: str, heads: int, kv_heads: int, dim: int) -> None:
    """Keys and values interleaved in one tensor, rows outside heads: attention, copy on
    write and compaction give what a contiguous pool gives."""
    lens, page = [300, 41, 17, 700], 32
    plain, o = _filled(dtype, page, kv_heads, dim, lens, layers=2, layer=1, seed=41, extra=9)
    pages = plain.k.shape[1]
    both = torch.zeros((2, pages, page, 2, kv_heads, dim), dtype=DTYPES[dtype], device="cuda")
    k, v = both[:, :, :, 0].transpose(2, 3), both[:, :, :, 1].transpose(2, 3)
    k.copy_(plain.k)
    v.copy_(plain.v)
    assert not k.is_contiguous()
    cache = PagedKVCache(k, v, plain.block_table.clone(), plain.lengths.clone(), plain.refs.clone())
    g = torch.Generator(device="cuda").manual_seed(42)
    new = [300, 1, 5, 40]
    starts = [0] + np.cumsum(new).tolist()
    q = torch.randn((starts[-1], heads, dim), generator=g, device="cuda").to(DTYPES[dtype])
    outs = [c.attend(q, [0, 1, 2, 3], starts, layer=1) for c in (plain, cache)]
    assert torch.equal(*outs)
    _check_rows(outs[1].double().cpu().numpy(), None, q.double().cpu().numpy(), o, [0, 1, 2, 3], starts, 1,
                1 / np.sqrt(dim), dtype)
    for c in (plain, cache):
        c.truncate([0], [0])
        c.fork([3], [0])
        c.reserve([0, 3], [1, 2])
        c.compact()
        c.status()
    for name in ("block_table", "lengths", "refs"):
        assert torch.equal(getattr(plain, name), getattr(cache, name)), name
    live = plain.refs > 0
    for a, b in ((plain.k, k), (plain.v, v)):  # bits, NaN past the tokens included
        assert torch.equal(a[:, live].contiguous().view(torch.int16), b[:, live].contiguous().view(torch.int16))
