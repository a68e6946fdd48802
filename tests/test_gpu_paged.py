"""The paged K/V cache on the device against its oracle (needs a B200).

* page operations: tables, lengths, reference counts and pool contents equal the oracle's
  after every step of random sequences of steps, and after each refusal;
* attention: every element within a bound derived from the roundings it is made of, for
  each dtype, head layout, page size and a set of lengths around the tile borders, with NaN
  in every place of the pool that no token holds;
* streams, graphs, strides, padded batches.
"""
from __future__ import annotations

import math
import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]

from moe_sm100 import _lib  # noqa: E402
from moe_sm100.paged import PagedKVCache  # noqa: E402
from oracle.paged_oracle import OracleError, PagedOracle, attend_chunk  # noqa: E402

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def _pair(layers, pages, page, kv_heads, dim, seqs, blocks, dtype="f16"):
    cache = PagedKVCache.allocate(layers=layers, pages=pages, page_size=page, kv_heads=kv_heads,
                                  head_dim=dim, sequences=seqs, max_blocks=blocks,
                                  dtype=DTYPES[dtype])
    return cache, PagedOracle(layers, pages, page, kv_heads, dim, seqs, blocks)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _same_tables(cache, o):
    assert cache.block_table.tolist() == o.table
    assert cache.lengths.tolist() == o.lengths
    assert cache.refs.tolist() == o.refs


def _same_tokens(cache, o):
    """The cached tokens of every sequence, bit for bit."""
    k, v = cache.k.double().cpu().numpy(), cache.v.double().cpu().numpy()
    for s, n in enumerate(o.lengths):
        for b in range(o.blocks(n)):
            rows = min(n - b * o.page, o.page)
            p = o.table[s][b]
            np.testing.assert_array_equal(k[:, p, :, :rows], o.k[:, p, :, :rows])
            np.testing.assert_array_equal(v[:, p, :, :rows], o.v[:, p, :, :rows])


def _append_all(cache, o, seqs, counts, rng):
    """New tokens of every layer on both sides."""
    starts = [0] + np.cumsum(counts).tolist()
    for layer in range(cache.k.shape[0]):
        k, v = (torch.from_numpy(rng.standard_normal((starts[-1], cache.kv_heads, cache.head_dim))
                                 .astype(np.float32)).cuda().to(cache.dtype) for _ in range(2))
        cache.append(k, v, _i32(seqs), _i32(starts), layer=layer)
        o.append(layer, k.double().cpu().numpy(), v.double().cpu().numpy(), seqs, starts)


# ------------------------------------------------------------------ pages
@pytest.mark.parametrize("page,pages,dim,dtype", [(16, 60, 64, "bf16"), (64, 35, 128, "f16")])
def test_random_steps_match_the_oracle(page: int, pages: int, dim: int, dtype: str) -> None:
    rng, nrng = random.Random(page), np.random.default_rng(page)
    cache, o = _pair(2, pages, page, 2, dim, 14, 9, dtype)
    for step in range(120):
        seqs = rng.sample(range(14), rng.randint(1, 5))
        kind = rng.choice(["grow", "grow", "fork", "cut", "compact", "free"])
        failed = False
        try:
            if kind == "grow":
                counts = [rng.choice([0, 1, 1, page - 1, page, 2 * page + 3]) for _ in seqs]
                cache.reserve(seqs, counts)
                o.reserve(seqs, counts)
            elif kind == "fork" and len(seqs) > 1:
                cache.fork([seqs[0]] * (len(seqs) - 1), seqs[1:])
                o.fork([seqs[0]] * (len(seqs) - 1), seqs[1:])
            elif kind == "cut":
                to = [rng.randint(0, o.lengths[s]) for s in seqs]
                cache.truncate(seqs, to)
                o.truncate(seqs, to)
            elif kind == "free":
                cache.free(seqs)
                o.truncate(seqs, [0] * len(seqs))
            elif kind == "compact" and step % 3 == 0:
                cache.compact()
                o.compact()
        except OracleError:
            failed = True
        if failed:
            with pytest.raises(_lib.MoeError):
                cache.status()
        else:
            cache.status()
            if kind == "grow":
                _append_all(cache, o, seqs, counts, nrng)
        _same_tables(cache, o)
        o.check_invariants()
    _same_tokens(cache, o)


def test_copy_on_write_of_many_holders_at_once() -> None:
    """All holders of one partly filled page grow in one call: each takes a copy, and the
    page that nobody holds any more is free."""
    cache, o = _pair(3, 40, 32, 2, 64, 9, 3)
    rng = np.random.default_rng(1)
    cache.reserve([4], [45])
    o.reserve([4], [45])
    _append_all(cache, o, [4], [45], rng)
    kids = [0, 1, 2, 3, 5, 6, 7, 8]
    cache.fork([4] * 8, kids)
    o.fork([4] * 8, kids)
    every = kids + [4]
    cache.reserve(every, [1] * 9)
    o.reserve(every, [1] * 9)
    _append_all(cache, o, every, [1] * 9, rng)
    cache.status()
    _same_tables(cache, o)
    _same_tokens(cache, o)
    assert o.refs.count(9) == 1 and sum(o.refs) == 18


def test_reserve_over_many_sequences_and_a_large_pool() -> None:
    """More entries than the planning CTA has threads, more pages than one step scans."""
    n, pages = 1500, 40000
    cache, o = _pair(1, pages, 16, 1, 64, n, 40)
    rng = random.Random(3)
    order = rng.sample(range(n), n)
    counts = [rng.randint(0, 300) for _ in range(n)]
    for c, s, x in ((cache, order, counts), (o, order, counts)):
        c.reserve(s, x)
    cut = [rng.randint(0, o.lengths[s]) for s in order]
    for c in (cache, o):
        c.truncate(order, cut)
        c.reserve(order, counts)
    cache.status()
    _same_tables(cache, o)


@pytest.mark.parametrize("call,code", [
    (lambda c: c.reserve([0, 1, 0], [1, 1, 1]), _lib.MOE_ERR_INVALID),
    (lambda c: c.reserve([0, 4], [1, 1]), _lib.MOE_ERR_INVALID),
    (lambda c: c.reserve([-1], [1]), _lib.MOE_ERR_INVALID),
    (lambda c: c.reserve([0], [-1]), _lib.MOE_ERR_INVALID),
    (lambda c: c.reserve([0], [16 * 6 - 20 + 1]), _lib.MOE_ERR_INVALID),    # past the table
    (lambda c: c.reserve([0], [2 ** 31 - 1]), _lib.MOE_ERR_INVALID),
    (lambda c: c.reserve([0, 3], [16 * 6 - 20, 16 * 6]), _lib.MOE_ERR_NO_PAGES),
    (lambda c: c.fork([0, 1], [3, 3]), _lib.MOE_ERR_INVALID),
    (lambda c: c.fork([0], [0]), _lib.MOE_ERR_INVALID),
    (lambda c: c.fork([0, 3], [3, 2]), _lib.MOE_ERR_INVALID),               # parent and child
    (lambda c: c.fork([0], [1]), _lib.MOE_ERR_INVALID),                     # not empty
    (lambda c: c.fork([9], [3]), _lib.MOE_ERR_INVALID),
    (lambda c: c.truncate([0], [21]), _lib.MOE_ERR_INVALID),
    (lambda c: c.truncate([0], [-1]), _lib.MOE_ERR_INVALID),
    (lambda c: c.truncate([0, 0], [1, 2]), _lib.MOE_ERR_INVALID),
    (lambda c: c.copy_pages([0, 1], [7, 7]), _lib.MOE_ERR_INVALID),
    (lambda c: c.copy_pages([0, 7], [7, 5]), _lib.MOE_ERR_INVALID),
    (lambda c: c.copy_pages([0], [10]), _lib.MOE_ERR_INVALID),
    (lambda c: c.copy_pages([-1], [5]), _lib.MOE_ERR_INVALID),
])
def test_refusals_change_nothing(call, code: int) -> None:
    cache, _o = _pair(1, 10, 16, 1, 64, 4, 6)
    cache.reserve([0, 1], [20, 33])
    cache.k.normal_()
    cache.status()
    before = [t.clone() for t in (cache.block_table, cache.lengths, cache.refs, cache.k)]
    call(cache)
    with pytest.raises(_lib.MoeError) as e:
        cache.status()
    assert e.value.code == code
    cache.status()  # reported once
    for a, b in zip(before, (cache.block_table, cache.lengths, cache.refs, cache.k)):
        assert torch.equal(a, b)


def test_argument_checks() -> None:
    cache, _o = _pair(2, 10, 16, 2, 64, 4, 6)
    row = torch.zeros((3, 2, 64), dtype=torch.float16, device="cuda")
    ok = dict(seqs=_i32([0]), starts=_i32([0, 3]))
    cache.reserve([], [])
    cache.reserve([0], [3])
    with pytest.raises(TypeError):
        cache.append(row.float(), row, **ok)
    with pytest.raises(TypeError):
        cache.append(row.cpu(), row, **ok)
    with pytest.raises(ValueError):
        cache.append(row, row[:2], **ok)
    with pytest.raises(ValueError):
        cache.append(row[:, :1], row[:, :1], **ok)
    with pytest.raises(ValueError):
        cache.append(row, row, layer=2, **ok)
    with pytest.raises(ValueError):
        cache.append(row, row, _i32([0]), _i32([0, 1, 3]))
    with pytest.raises(TypeError):
        cache.append(row, row, _i32([0]).long(), _i32([0, 3]))
    with pytest.raises(TypeError):
        cache.append(row, row, _i32([0]).cpu(), _i32([0, 3]))
    with pytest.raises(ValueError):
        cache.reserve([0, 1], [1])
    with pytest.raises(ValueError):
        cache.attend(torch.zeros((3, 3, 64), dtype=torch.float16, device="cuda"), **ok)
    with pytest.raises(ValueError):
        cache.attend(torch.zeros((3, 4, 128), dtype=torch.float16, device="cuda")[..., ::2], **ok)
    with pytest.raises(ValueError):
        cache.attend(row, out=row[:2], **ok)
    with pytest.raises(ValueError):
        cache.attend(row, lse=torch.zeros((3, 4), device="cuda"), **ok)
    with pytest.raises(ValueError):
        cache.attend(row, scale=0.0, **ok)
    with pytest.raises(ValueError):
        cache.attend(row, scale=float("nan"), **ok)
    odd = torch.zeros(3 * 2 * 64 + 4, dtype=torch.float16, device="cuda")[4:].view(3, 2, 64)
    with pytest.raises(ValueError):  # 8-byte aligned
        cache.attend(odd, **ok)
    empty = torch.empty((0, 2, 64), dtype=torch.float16, device="cuda")
    assert cache.attend(empty, _i32([]), _i32([0])).shape == empty.shape
    other = PagedKVCache.allocate(layers=2, pages=10, page_size=32, kv_heads=2, head_dim=64,
                                  sequences=4, max_blocks=6)
    with pytest.raises(ValueError):
        cache.compact(into=other)
    cache.status()


@pytest.mark.parametrize("more", [0, 5])
def test_compact_into_another_pool(more: int) -> None:
    cache, o = _pair(2, 30, 16, 2, 128, 6, 5)
    rng = np.random.default_rng(2)
    seqs = [0, 1, 2, 3, 4]
    for c in (cache, o):
        c.reserve(seqs, [50, 3, 16, 0, 70])
    _append_all(cache, o, seqs, [50, 3, 16, 0, 70], rng)
    for c in (cache, o):
        c.truncate([0], [0])
        c.fork([4], [0])
    live = sum(r > 0 for r in o.refs)
    into, oi = _pair(2, live + more, 16, 2, 128, 8, 7)
    into.k.fill_(9)
    cache.compact(into=into)
    o.compact(oi)
    cache.status()
    _same_tables(into, oi)
    _same_tokens(into, oi)
    assert (into.k[:, live:] == 9).all()  # pages past the live ones are left alone
    _same_tables(cache, o)
    small, _ = _pair(2, live - 1, 16, 2, 128, 8, 7)
    cache.compact(into=small)
    with pytest.raises(_lib.MoeError) as e:
        cache.status()
    assert e.value.code == _lib.MOE_ERR_NO_PAGES
    assert (small.block_table == -1).all() and (small.k == 0).all()


def test_copy_pages() -> None:
    cache, o = _pair(2, 12, 32, 3, 64, 1, 1)
    cache.k.normal_()
    cache.v.normal_()
    o.k[:], o.v[:] = cache.k.double().cpu().numpy(), cache.v.double().cpu().numpy()
    cache.copy_pages([3, 3, 0], [11, 4, 7])
    o.copy_pages([3, 3, 0], [11, 4, 7])
    cache.status()
    np.testing.assert_array_equal(cache.k.double().cpu().numpy(), o.k)
    np.testing.assert_array_equal(cache.v.double().cpu().numpy(), o.v)


def test_append_strided_rows_and_padding() -> None:
    """Rows of a fused projection (strided views), padded rows ignored, a strided pool."""
    pool = torch.zeros((2, 9, 16, 2, 3, 64), dtype=torch.bfloat16, device="cuda")
    k, v = pool[:, :, :, 0].transpose(2, 3), pool[:, :, :, 1].transpose(2, 3)  # rows outside heads
    cache = PagedKVCache(k, v, torch.full((3, 3), -1, dtype=torch.int32, device="cuda"),
                         torch.zeros(3, dtype=torch.int32, device="cuda"),
                         torch.zeros(9, dtype=torch.int32, device="cuda"))
    o = PagedOracle(2, 9, 16, 3, 64, 3, 3)
    fused = torch.randn((40, 9, 64), device="cuda").to(torch.bfloat16)
    kk, vv = fused[:, 3:6], fused[:, 6:]
    for c in (cache, o):
        c.reserve([2, 0], [20, 13])
    cache.append(kk, vv, [2, 0], [0, 20, 33], layer=1)
    o.append(1, kk.double().cpu().numpy(), vv.double().cpu().numpy(), [2, 0], [0, 20, 33])
    cache.status()
    _same_tables(cache, o)
    np.testing.assert_array_equal(k.double().cpu().numpy(), o.k)
    np.testing.assert_array_equal(v.double().cpu().numpy(), o.v)


def test_append_reports_missing_pages_and_too_many_rows() -> None:
    cache, _o = _pair(1, 4, 16, 1, 64, 2, 2)
    row = torch.ones((5, 1, 64), dtype=torch.float16, device="cuda")
    cache.reserve([0], [3])
    cache.append(row, row, [0], [0, 5])      # five rows of a sequence of three tokens
    with pytest.raises(ValueError):
        cache.status()
    cache.lengths[1] = 5                     # tokens without pages
    cache.append(row, row, [1], [0, 5])
    with pytest.raises(ValueError):
        cache.status()
    cache.append(row, row, [7], [0, 5])
    with pytest.raises(ValueError):
        cache.status()


# ------------------------------------------------------------------ attention
def _filled(dtype, page, kv_heads, dim, lens, layers=1, layer=0, seed=0, extra=3, nan=True):
    """A cache of random tokens whose pages lie anywhere, NaN everywhere else."""
    rng = random.Random(seed)
    blocks = [-(-n // page) for n in lens]
    pages = sum(blocks) + extra
    cache, o = _pair(layers, pages, page, kv_heads, dim, len(lens), max(max(blocks), 1) + 1, dtype)
    free = rng.sample(range(pages), pages)
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache.k.copy_(torch.randn(cache.k.shape, generator=g, device="cuda"))
    cache.v.copy_(torch.randn(cache.v.shape, generator=g, device="cuda"))
    keep = torch.zeros((pages, page), dtype=torch.bool)
    for s, n in enumerate(lens):
        for b in range(blocks[s]):
            p = free.pop()
            o.table[s][b], o.refs[p] = p, 1
            keep[p, :min(n - b * page, page)] = True
        o.lengths[s] = n
    if nan:
        gone = ~keep.cuda()[None, :, None, :, None]
        cache.k.masked_fill_(gone, float("nan"))
        cache.v.masked_fill_(gone, float("nan"))
    cache.block_table.copy_(torch.tensor(o.table, dtype=torch.int32))
    cache.lengths.copy_(torch.tensor(o.lengths, dtype=torch.int32))
    cache.refs.copy_(torch.tensor(o.refs, dtype=torch.int32))
    o.k[:], o.v[:] = cache.k.double().cpu().numpy(), cache.v.double().cpu().numpy()
    return cache, o


def _check_rows(got, lse, q, o, seqs, starts, layer, scale, dtype):
    """Every element within the roundings it is made of.

    p_j is rounded to the cache's dtype for the product with v (half a step of 1 relative:
    u), the result once more (u): u * (sum p |v| + |out|).  In fp32: a score is a sum of
    dim exact products, off by at most dim * 2^-23 * size in any order and with truncating
    adders, where size = scale * max sum |q_i k_i| also bounds the score; the exponential's
    argument and value add 2^-21 (1 + size).  Both move p relatively, so they enter as
    e * sum p |v|, twice (numerator and denominator).  Sums of n terms add n * 2^-24 at most, in blocks.
    """
    u = torch.finfo(DTYPES[dtype]).eps / 2
    for i, s in enumerate(seqs):
        a, b = starts[i], starts[i + 1]
        if a == b:
            continue
        k, v = o.cached(layer, s)
        ref, ref_lse, mag = attend_chunk(q[a:b], k, v, scale)
        group = q.shape[1] // o.shape[2]
        size = max((scale * (np.abs(q[a:b, h]) @ np.abs(k[:, h // group]).T).max()
                    for h in range(q.shape[1])), default=0.0) if len(k) else 0.0
        e = q.shape[2] * 2.0 ** -23 * size + 2.0 ** -21 * (1 + size) + len(k) * 2.0 ** -24
        tol = u * (mag + np.abs(ref)) * 1.01 + 2 * e * mag + 1e-30
        err = np.abs(got[a:b] - ref)
        assert np.isfinite(got[a:b]).all(), (i, s)
        assert (err <= tol + torch.finfo(DTYPES[dtype]).tiny).all(), (
            i, s, float((err / (tol + 1e-30)).max()), np.unravel_index((err - tol).argmax(), err.shape))
        if lse is not None:
            seen = np.isfinite(ref_lse)
            assert (lse[a:b][~seen] == -np.inf).all()
            assert (np.abs(lse[a:b][seen] - ref_lse[seen]) <= e + 2.0 ** -22 * np.abs(ref_lse[seen])
                    + 1e-6).all()


def _attend_case(dtype, heads, kv_heads, dim, page, work, layers=1, layer=0, seed=0, scale=None,
                 pad=0):
    lens, new = [n for n, _ in work], [m for _, m in work]
    cache, o = _filled(dtype, page, kv_heads, dim, lens, layers, layer, seed)
    starts = [0] + np.cumsum(new).tolist()
    rows = starts[-1] + pad
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = (1.5 * torch.randn((rows, heads, dim), generator=g, device="cuda")).to(DTYPES[dtype])
    order = list(range(len(work)))
    random.Random(seed).shuffle(order)       # batch order is not table order
    starts = [0] + np.cumsum([new[s] for s in order]).tolist()
    lse = torch.full((rows, heads), 7.0, device="cuda")
    out = torch.full_like(q, 3.0)
    cache.attend(q, _i32(order), _i32(starts), layer=layer, scale=scale, out=out, lse=lse)
    cache.status()
    used = starts[-1]
    assert (out[used:] == 3).all() and (lse[used:] == 7).all()  # rows behind the last sequence
    _check_rows(out.double().cpu().numpy(), lse.double().cpu().numpy(), q.double().cpu().numpy(), o,
                order, starts, layer, 1 / math.sqrt(dim) if scale is None else scale, dtype)
    again = torch.full_like(out, 3.0)
    cache.attend(q, _i32(order), _i32(starts), layer=layer, scale=scale, out=again)
    assert torch.equal(out, again)           # deterministic


EDGES = [(1, 1), (2, 1), (15, 1), (16, 1), (17, 1), (127, 1), (128, 1), (129, 1), (255, 1),
         (256, 1), (257, 1), (1000, 1)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(96, 8, 128), (8, 8, 64), (12, 4, 64), (16, 2, 128),
                                                (7, 1, 128), (96, 1, 64)])
@pytest.mark.parametrize("page", [16, 64])
def test_decode_around_the_borders(dtype: str, heads: int, kv_heads: int, dim: int, page: int) -> None:
    _attend_case(dtype, heads, kv_heads, dim, page, EDGES, seed=heads + page)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim,page,work", [
    ("f16", 96, 8, 128, 64, [(300, 300)]),                         # a whole prompt
    ("bf16", 96, 8, 128, 32, [(700, 10), (11, 11), (400, 33)]),    # 128-row borders of a group of 12
    ("f16", 16, 2, 128, 128, [(129, 16), (128, 17), (1025, 32), (1024, 31), (640, 128)]),
    ("bf16", 8, 8, 64, 16, [(700, 256), (256, 256), (257, 257), (255, 255), (513, 127), (130, 128)]),
    ("f16", 8, 8, 64, 256, [(1500, 1), (1500, 700), (1500, 64), (3, 2)]),
    ("bf16", 12, 4, 64, 64, [(2000, 1), (900, 300), (0, 0), (5, 5), (1, 1), (640, 0)]),
    ("f16", 96, 1, 64, 16, [(50, 3), (200, 2), (333, 1), (90, 40)]),
    ("bf16", 7, 1, 128, 32, [(290, 37), (291, 73), (37, 37)]),
])
def test_chunks(dtype, heads, kv_heads, dim, page, work) -> None:
    _attend_case(dtype, heads, kv_heads, dim, page, work, seed=len(work))


def test_long_context_split_over_the_gpu() -> None:
    _attend_case("f16", 8, 2, 128, 64, [(20011, 1), (3, 1)], seed=4)
    _attend_case("bf16", 16, 2, 64, 128, [(9001, 40)], seed=5)


@pytest.mark.parametrize("dtype,dim", [("f16", 128), ("bf16", 64)])
def test_rows_around_the_unit_sizes(dtype: str, dim: int) -> None:
    """Chunks whose rows end at and around every size at which another form of the kernel
    takes over, with few and with many older tokens, all in one batch."""
    sizes = (15, 16, 17, 31, 32, 33, 64, 65, 127, 128, 129, 255, 256, 257, 288, 289, 384, 385)
    _attend_case(dtype, 4, 4, dim, 32, [(m + (0, 1, 63, 130, 500)[i % 5], m) for i, m in enumerate(sizes)],
                 seed=dim)


@pytest.mark.parametrize("heads,kv_heads", [(200, 1), (34, 2), (5, 5)])
def test_unusual_groups(heads: int, kv_heads: int) -> None:
    _attend_case("f16", heads, kv_heads, 64, 16, [(70, 1), (130, 3), (9, 9), (1, 1), (300, 40)], seed=heads)


def test_pool_past_32_bit_offsets() -> None:
    """Pages whose bytes lie past 2^32 in the pool: append, copy on write, attention."""
    layers, pages, page = 2, 18000, 64
    k, v = (torch.empty((layers, pages, 8, page, 128), dtype=torch.float16, device="cuda") for _ in range(2))
    assert k.numel() * 2 > 1 << 32
    table = torch.full((3, 4), -1, dtype=torch.int32, device="cuda")
    lengths = torch.zeros(3, dtype=torch.int32, device="cuda")
    refs = torch.ones(pages, dtype=torch.int32, device="cuda")
    refs[-6:] = 0                            # only the last pages are free
    cache = PagedKVCache(k, v, table, lengths, refs)
    g = torch.Generator(device="cuda").manual_seed(3)
    new = [torch.randn((100, 8, 128), generator=g, device="cuda").half() for _ in range(2)]
    cache.reserve([0], [100])
    cache.append(*new, [0], [0, 100], layer=1)
    cache.fork([0], [2])
    cache.reserve([2], [1])
    one = [torch.randn((1, 8, 128), generator=g, device="cuda").half() for _ in range(2)]
    cache.append(*one, [2], [0, 1], layer=1)
    q = torch.randn((1, 96, 128), generator=g, device="cuda").half()
    out = cache.attend(q, [2], [0, 1], layer=1)
    cache.status()
    assert table.tolist()[0][:2] == [pages - 6, pages - 5] and table.tolist()[2][:2] == [pages - 6, pages - 4]
    kk, vv = (torch.cat([a, b]).double().cpu().numpy() for a, b in zip(new, one))
    ref, _lse, mag = attend_chunk(q.double().cpu().numpy(), kk, vv, 1 / math.sqrt(128))
    u = 2.0 ** -11
    # as _check_rows: two roundings, and the fp32 scores (below 2^-11 too) twice
    assert (np.abs(out.double().cpu().numpy() - ref) <= u * (mag + np.abs(ref)) + 2 * u * mag).all()


def test_starts_past_the_rows_are_reported() -> None:
    cache, _o = _filled("f16", 16, 2, 64, [77, 40], seed=2)
    q = torch.randn((4, 4, 64), device="cuda").half()
    out = torch.full_like(q, 5.0)
    for starts in ([0, 2, 9], [0, 3, 2], [-3, 2, 4]):
        cache.attend(q, [0, 1], starts, out=out)
        with pytest.raises(ValueError):
            cache.status()


def test_two_streams_at_once() -> None:
    """Attention calls on one cache that overlap on two streams."""
    cache, _o = _filled("bf16", 32, 2, 128, [3000, 1700, 64, 900], seed=5)
    g = torch.Generator(device="cuda").manual_seed(2)
    qs = [torch.randn((n, 16, 128), generator=g, device="cuda").bfloat16() for n in (4, 400)]
    args = [([0, 1, 2, 3], [0, 1, 2, 3, 4]), ([3, 0], [0, 150, 400])]
    args = [tuple(_i32(v) for v in a) for a in args]
    want = [cache.attend(q, *a) for q, a in zip(qs, args)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            got[i].append(cache.attend(qs[i], *args[i], stream=streams[i]))
    torch.cuda.synchronize()
    cache.status()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_two_graphs_of_one_cache_replayed_in_turn() -> None:
    cache, _o = _filled("f16", 16, 2, 64, [500, 90], seed=6, nan=False)
    g = torch.Generator(device="cuda").manual_seed(2)
    qs = [torch.randn((n, 8, 64), generator=g, device="cuda").half() for n in (2, 60)]
    args = [(_i32([0, 1]), _i32([0, 1, 2])), (_i32([1, 0]), _i32([0, 20, 60]))]
    want = [cache.attend(q, *a) for q, a in zip(qs, args)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q, a in zip(qs, args):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(cache.attend(q, *a))
    for _ in range(3):
        for i in (0, 1, 1, 0):
            outs[i].zero_()
            graphs[i].replay()
            assert torch.equal(outs[i], want[i])
    cache.status()


def test_many_short_sequences() -> None:
    rng = random.Random(8)
    _attend_case("bf16", 8, 2, 64, 16, [(rng.randint(1, 90), 1) for _ in range(700)], seed=8)


def test_more_units_than_the_plan_holds_on_chip() -> None:
    """More than 512 units of 256 rows, and more entries than the planning CTA has threads,
    chunks among the last of them."""
    _attend_case("f16", 16, 1, 64, 16, [(230 + i, 230) for i in range(40)], seed=10)
    rng = random.Random(11)
    work = [(rng.randint(1, 70), 1) for _ in range(1400)] + [(300, 300), (170, 65), (9, 9), (64, 40)]
    _attend_case("bf16", 4, 2, 64, 16, work, seed=11)


def test_layers_scale_and_padding() -> None:
    _attend_case("f16", 8, 2, 128, 32, [(200, 3), (40, 1)], layers=3, layer=2, seed=6, scale=0.25,
                 pad=9)


def test_rows_that_see_nothing() -> None:
    """More new rows than tokens, and a sequence without tokens: 0 and -inf."""
    cache, o = _filled("f16", 16, 2, 64, [5, 0, 300], seed=1)
    q = torch.randn((320, 4, 64), device="cuda").half()
    lse = torch.zeros((320, 4), device="cuda")
    starts = [0, 9, 11, 320]
    out = cache.attend(q, [0, 1, 2], starts, lse=lse)
    cache.status()
    _check_rows(out.double().cpu().numpy(), lse.double().cpu().numpy(), q.double().cpu().numpy(), o,
                [0, 1, 2], starts, 0, 0.125, "f16")
    assert (out[:4] == 0).all() and (out[9:11] == 0).all() and (out[11:20] == 0).all()
    assert torch.isinf(lse[:4]).all() and torch.isinf(lse[9:20]).all()


def test_large_scores() -> None:
    """Scores of some thousands: the running maximum, not the range of exp, decides."""
    cache, o = _filled("bf16", 32, 1, 64, [400], seed=3)
    q = (300 * torch.randn((2, 4, 64), device="cuda")).bfloat16()
    out = cache.attend(q, [0], [0, 2], scale=1.0)
    k, v = o.cached(0, 0)
    ref, _l, _m = attend_chunk(q.double().cpu().numpy(), k, v, 1.0)
    # softmax is one-hot but for scores closer than the fp32 error of a score of ~1e4
    # (64 * 2^-23 * 1e4 < 0.1): the checked rows have a clear winner
    s = np.einsum("mhd,nd->mhn", q.double().cpu().numpy(), k[:, 0])
    s[0, :, -1] = -np.inf
    top = np.sort(s, axis=-1)
    clear = top[..., -1] - top[..., -2] > 20
    assert clear.any()
    got = out.double().cpu().numpy()
    assert np.isfinite(got).all()
    # one value of weight 1 (others below e^-19): only the two roundings remain
    u = 2.0 ** -8
    assert (np.abs(got - ref)[clear] <= 2 * u * np.abs(ref)[clear] + 1e-5).all()


def test_strided_queries_and_outputs() -> None:
    cache, o = _filled("f16", 16, 2, 64, [77, 30], seed=2)
    big = torch.randn((20, 3, 8, 64), device="cuda").half()
    q = big[::2, 1]
    hold = torch.zeros((10, 4, 8, 64), device="cuda").half()
    out = hold[:, 2].transpose(0, 1).contiguous().transpose(0, 1)   # heads outside rows
    lse = torch.zeros((8, 10), device="cuda").t()
    cache.attend(q, [1, 0], [0, 4, 10], out=out, lse=lse)
    cache.status()
    _check_rows(out.double().cpu().numpy(), lse.double().cpu().numpy(), q.double().cpu().numpy(), o,
                [1, 0], [0, 4, 10], 0, 0.125, "f16")


def test_the_same_sequence_twice_reads_twice() -> None:
    """Both entries get the attention of their sequence.  Where the shares cut a unit is not
    the same for the two, and so neither is the order of the fp32 sums: each is held to the
    bound of its own roundings (see _check_rows), not to the other's bits."""
    cache, o = _filled("f16", 16, 2, 64, [77], seed=2)
    q = torch.randn((3, 4, 64), device="cuda").half()
    qq = torch.cat([q, q])
    out = cache.attend(qq, [0, 0], [0, 3, 6])
    cache.status()
    _check_rows(out.double().cpu().numpy(), None, qq.double().cpu().numpy(), o, [0, 0], [0, 3, 6],
                0, 0.125, "f16")


def test_attend_reports_bad_pages_and_sequences() -> None:
    cache, _o = _filled("f16", 16, 2, 64, [77, 40], seed=2)
    q = torch.randn((2, 4, 64), device="cuda").half()
    good = cache.attend(q, [0, 1], [0, 1, 2])
    cache.status()
    cache.block_table[0, 2] = 1 << 20        # read as zeros, reported
    out = cache.attend(q, [0, 1], [0, 1, 2])
    with pytest.raises(ValueError):
        cache.status()
    assert torch.equal(out[1], good[1])
    out = cache.attend(q, [5, 1], [0, 1, 2])
    with pytest.raises(ValueError):
        cache.status()
    assert torch.equal(out[1], good[1]) and (out[0] == 0).all()


def test_streams_and_graph_replay() -> None:
    """A decode step (reserve, append, attend) captured once and replayed: the same tables
    and outputs as the steps run one by one on another stream."""
    lens = [30, 64, 5]
    caches = [_filled("f16", 16, 2, 64, lens, seed=9, extra=40, nan=False)[0] for _ in range(2)]
    for c in caches:  # room for the steps in the table
        wide = torch.full((3, 20), -1, dtype=torch.int32, device="cuda")
        wide[:, :c.block_table.shape[1]] = c.block_table
        c.__init__(c.k, c.v, wide, c.lengths, c.refs)
    g = torch.Generator(device="cuda").manual_seed(1)
    steps = [[torch.randn((3, n, 64), generator=g, device="cuda").half() for n in (2, 2, 4)]
             for _ in range(20)]
    seqs, ones, starts = _i32([2, 0, 1]), _i32([1, 1, 1]), _i32([0, 1, 2, 3])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    want = []
    for k, v, q in steps:
        caches[0].reserve(seqs, ones, stream=side)
        caches[0].append(k, v, seqs, starts, stream=side)
        want.append(caches[0].attend(q, seqs, starts, stream=side))
    caches[0].status(stream=side)
    bufs = [t.clone() for t in steps[0]]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        caches[1].reserve(seqs, ones)
        caches[1].append(bufs[0], bufs[1], seqs, starts)
        out = caches[1].attend(bufs[2], seqs, starts)
    for step, ref in zip(steps, want):
        for b, t in zip(bufs, step):
            b.copy_(t)
        graph.replay()
        assert torch.equal(out, ref)
    caches[1].status()
    for name in ("block_table", "lengths", "refs", "k", "v"):
        assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), name
