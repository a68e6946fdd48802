"""Offsets and sequences of a batch over the paged cache (needs a B200): rows that belong to
no entry are left alone by ``append``, ``attend`` and ``forward_cached`` alike."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]

from moe_sm100.paged import PagedKVCache  # noqa: E402
from oracle.attention_oracle import AttnConfig, glm4_attention_block  # noqa: E402
from oracle.cases import AttnSpec, make_attn_case  # noqa: E402
from test_gpu_attention_cached import TOL_BLOCK, TOL_DELTA, _cache, _layer, _rel  # noqa: E402
from test_gpu_paged import _check_rows, _filled, _i32  # noqa: E402


def _places(cache, s: int) -> tuple:
    """Keys and values of a sequence's places, layer 0, [tokens, heads, dim]."""
    n = int(cache.lengths[s])
    ids = cache.block_table[s, :-(-n // cache.page_size)].long()
    return tuple(p[0][ids].transpose(1, 2).reshape(-1, cache.kv_heads, cache.head_dim)[:n].clone()
                 for p in (cache.k, cache.v))


# a batch sliced out of a larger one: its rows begin after the first
SLICES = [([1], [4, 8]), ([1, 0], [4, 6, 8]), ([0], [7, 8]), ([1, 0, 2], [2, 2, 5, 6])]


@pytest.mark.parametrize("seqs,starts", SLICES)
def test_append_leaves_rows_before_the_first_entry_alone(seqs: list, starts: list) -> None:
    cache, o = _filled("f16", 16, 2, 64, [20, 33, 5], seed=4)
    k, v = (torch.randn((10, 2, 64), device="cuda").half() for _ in range(2))
    before = [_places(cache, s) for s in range(3)]
    cache.append(k, v, seqs, starts)
    cache.status()
    o.append(0, k.double().cpu().numpy(), v.double().cpu().numpy(), seqs, starts)
    for s in range(3):
        new = sum(starts[i + 1] - starts[i] for i, x in enumerate(seqs) if x == s)
        for got, was, want in zip(_places(cache, s), before[s], o.cached(0, s)):
            old = got.shape[0] - new
            assert torch.equal(got[:old], was[:old])
            np.testing.assert_array_equal(got.double().cpu().numpy(), want)


@pytest.mark.parametrize("seqs,starts", SLICES)
def test_attend_leaves_rows_before_the_first_entry_alone(seqs: list, starts: list) -> None:
    cache, o = _filled("f16", 16, 2, 64, [20, 33, 5], seed=4)
    q = torch.randn((10, 4, 64), device="cuda").half()
    out, lse = torch.full_like(q, 3.0), torch.full((10, 4), 7.0, device="cuda")
    cache.attend(q, seqs, starts, out=out, lse=lse)
    cache.status()
    for rows in (slice(0, starts[0]), slice(starts[-1], 10)):
        assert (out[rows] == 3).all() and (lse[rows] == 7).all()
    _check_rows(out.double().cpu().numpy(), lse.double().cpu().numpy(), q.double().cpu().numpy(), o,
                seqs, starts, 0, 0.125, "f16")


@pytest.mark.parametrize("seqs,starts", SLICES)
def test_the_block_leaves_rows_before_the_first_entry_alone(seqs: list, starts: list) -> None:
    spec = AttnSpec(hidden=512, heads=16, kv_heads=2, head_dim=128, tokens=40, seed=71)
    x, t = make_attn_case(spec)
    al = _layer(spec, t, 64)
    cache = _cache(spec, 3, 3, 16)
    lens = [20, 33, 5]
    for s, n in enumerate(lens):  # all but the new tokens, which are their sequences' last
        cache.reserve([s], [n])
        al.forward_cached(torch.from_numpy(x[:n]).cuda(), cache, [s], [0, n])
    before = [_places(cache, s) for s in range(3)]
    new = {s: starts[i + 1] - starts[i] for i, s in enumerate(seqs)}
    batch = np.random.default_rng(5).standard_normal((10, spec.hidden)).astype(np.float32)
    out = torch.full((10, spec.hidden), 3.0, device="cuda")
    al.forward_cached(torch.from_numpy(batch).cuda(), cache, seqs, starts, out=out)
    cache.status()
    al.status()
    assert (out[:starts[0]] == 3).all() and (out[starts[-1]:] == 3).all()
    for s, n in enumerate(lens):
        old = n - new.get(s, 0)
        for got, was in zip(_places(cache, s), before[s]):
            assert torch.equal(got[:old], was[:old])
    for i, s in enumerate(seqs):
        rows = slice(starts[i], starts[i + 1])
        if new[s] == 0:
            continue
        whole = np.concatenate([x[:lens[s] - new[s]], batch[rows]])
        ref = glm4_attention_block(whole, t, AttnConfig.from_hf(spec.hf_config()))[-new[s]:]
        got = out[rows].cpu().numpy()
        assert _rel(got, ref) <= TOL_BLOCK and _rel(got - batch[rows], ref - batch[rows]) <= TOL_DELTA
    al.close()


# ------------------------------------------------------------------ batches that are refused
def _bits(cache) -> tuple:
    return tuple(t.clone().view(torch.int16) for t in (cache.k, cache.v))


def _status_raises_once(cache) -> None:
    with pytest.raises(ValueError):
        cache.status()
    cache.status()


BAD_BATCHES = [
    ([0], [0, 9]),                # ends past the rows
    ([0, 1], [0, 2, 9]),
    ([0, 1], [0, 3, 2]),          # decreases
    ([0, 1, 2], [0, 5, 3, 8]),
    ([0, 1], [-3, 2, 4]),
    ([0], [2147483647, -2147483648]),
    ([0, 0], [0, 2, 4]),          # the same sequence with rows in two entries
    ([2, 1, 0, 1], [0, 1, 2, 3, 4]),
]


@pytest.mark.parametrize("seqs,starts", BAD_BATCHES)
def test_append_refuses_a_bad_batch_as_a_whole(seqs: list, starts: list) -> None:
    cache, _o = _filled("bf16", 16, 2, 64, [20, 33, 12], seed=4)
    k, v = (torch.randn((8, 2, 64), device="cuda").bfloat16() for _ in range(2))
    before = _bits(cache)
    cache.append(k, v, seqs, starts)
    _status_raises_once(cache)
    assert all(torch.equal(a, b) for a, b in zip(before, _bits(cache)))


def test_append_refuses_among_many_entries() -> None:
    """More entries than a CTA has threads and more sequences than a warp's bits; the last
    one is wrong, then none is."""
    n = 700
    cache, o = _filled("f16", 16, 1, 64, [3] * n, seed=5, nan=False)
    k, v = (torch.randn((n, 1, 64), device="cuda").half() for _ in range(2))
    seqs = np.random.default_rng(1).permutation(n).tolist()
    before = _bits(cache)
    for bad_seqs, bad_starts in ((seqs[:-1] + [seqs[3]], list(range(n + 1))),
                                 (seqs, list(range(n)) + [n + 1])):
        cache.append(k, v, bad_seqs, bad_starts)
        _status_raises_once(cache)
        assert all(torch.equal(a, b) for a, b in zip(before, _bits(cache)))
    cache.append(k, v, seqs, list(range(n + 1)))
    cache.status()
    o.append(0, k.double().cpu().numpy(), v.double().cpu().numpy(), seqs, list(range(n + 1)))
    np.testing.assert_array_equal(cache.k.double().cpu().numpy(), o.k)
    np.testing.assert_array_equal(cache.v.double().cpu().numpy(), o.v)


def test_append_of_entries_without_rows() -> None:
    """Padding entries: no rows, any sequence, the same one as often as wanted."""
    cache, o = _filled("f16", 16, 2, 64, [20, 33, 12], seed=4, nan=False)
    k, v = (torch.randn((8, 2, 64), device="cuda").half() for _ in range(2))
    cache.append(k, v, [0, 0, 1, -1, 0, 99, 0], [0, 0, 0, 2, 2, 4, 4, 4])
    cache.status()
    o.append(0, k.double().cpu().numpy(), v.double().cpu().numpy(), [1, 0], [0, 2, 4])
    np.testing.assert_array_equal(cache.k.double().cpu().numpy(), o.k)
    np.testing.assert_array_equal(cache.v.double().cpu().numpy(), o.v)


def test_append_leaves_out_what_has_no_place() -> None:
    """A sequence that does not exist, more rows than tokens: the other rows are written."""
    cache, o = _filled("f16", 16, 2, 64, [20, 3, 12], seed=4, nan=False)
    k, v = (torch.randn((9, 2, 64), device="cuda").half() for _ in range(2))
    kk, vv = k.double().cpu().numpy(), v.double().cpu().numpy()
    cache.append(k, v, [0, 99, 2], [0, 2, 5, 6])
    _status_raises_once(cache)
    o.append(0, kk[[0, 1, 5]], vv[[0, 1, 5]], [0, 2], [0, 2, 3])
    cache.append(k, v, [1], [0, 5])
    _status_raises_once(cache)
    o.append(0, kk[2:5], vv[2:5], [1], [0, 3])
    np.testing.assert_array_equal(cache.k.double().cpu().numpy(), o.k)
    np.testing.assert_array_equal(cache.v.double().cpu().numpy(), o.v)


def test_the_block_refuses_a_bad_batch_as_a_whole() -> None:
    spec = AttnSpec(hidden=512, heads=16, kv_heads=2, head_dim=128, tokens=40, seed=72)
    x, t = make_attn_case(spec)
    al = _layer(spec, t, 64)
    cache = _cache(spec, 3, 3, 16)
    for s, n in enumerate((20, 33, 12)):
        cache.reserve([s], [n])
        al.forward_cached(torch.from_numpy(x[:n]).cuda(), cache, [s], [0, n])
    before = _bits(cache)
    batch = torch.randn((8, spec.hidden), device="cuda")
    for seqs, starts in BAD_BATCHES:
        out = torch.full_like(batch, 3.0)
        al.forward_cached(batch, cache, seqs, starts, out=out)
        _status_raises_once(cache)
        assert all(torch.equal(a, b) for a, b in zip(before, _bits(cache)))
        assert (out == 3).all()
    al.status()
    out = al.forward_cached(batch, cache, [0, 99, 2], [0, 2, 5, 8])  # one entry has no sequence
    _status_raises_once(cache)
    assert torch.equal(out[2:5], batch[2:5])
    good = al.forward_cached(batch, cache, [0, 2], [0, 2, 5])[:2]
    assert _rel(out[:2].cpu().numpy(), good.double().cpu().numpy()) <= TOL_BLOCK
    al.close()


def test_attend_refuses_wrong_offsets_as_a_whole() -> None:
    """Decreasing offsets would give rows to two entries; more entries than the planning CTA
    has threads, the wrong one among the last or the first."""
    cache, _o = _filled("f16", 16, 2, 64, [20, 33, 12], seed=4)
    q = torch.randn((8, 4, 64), device="cuda").half()
    out, lse = torch.full_like(q, 3.0), torch.full((8, 4), 7.0, device="cuda")
    many = [[0] * 1500 + [8], [0] * 1499 + [3, 2], [5, 3] + [8] * 1499]
    batches = [(s, t) for s, t in BAD_BATCHES if len(set(s)) == len(s)] + \
        [([0, 1, 2] * 500, t) for t in many[1:]]
    for seqs, starts in batches:
        cache.attend(q, seqs, starts, out=out, lse=lse)
        _status_raises_once(cache)
        assert (out == 3).all() and (lse == 7).all()
    cache.attend(q, [0, 1, 2] * 500, many[0], out=out, lse=lse)  # the last entry has all rows
    cache.status()
    assert (out != 3).any(dim=(1, 2)).all()


def test_the_block_on_more_entries_than_a_cta_checks() -> None:
    """One token of 600 sequences in one batch and in two; then a batch whose last entry is
    wrong."""
    spec = AttnSpec(hidden=512, heads=16, kv_heads=2, head_dim=128, tokens=40, seed=74)
    x, t = make_attn_case(spec)
    al = _layer(spec, t, 700)
    n = 600
    batch = torch.from_numpy(np.random.default_rng(6).standard_normal((n, spec.hidden)).astype(np.float32)).cuda()
    outs, caches = [], [_cache(spec, n, 1, 16) for _ in range(2)]
    for cache, cuts in zip(caches, ([0, n], [0, 300, n])):
        cache.reserve(list(range(n)), [1] * n)
        got = []
        for a, b in zip(cuts, cuts[1:]):
            got.append(al.forward_cached(batch[a:b], cache, list(range(a, b)), list(range(b - a + 1))))
        cache.status()
        outs.append(torch.cat(got))
    al.status()
    delta = [(o - batch).double().cpu().numpy() for o in outs]
    assert _rel(*delta) <= TOL_DELTA
    before = _bits(caches[0])
    for seqs, starts in ((list(range(n - 1)) + [5], list(range(n + 1))),
                         (list(range(n)), list(range(n)) + [n - 2])):
        out = torch.full_like(batch, 3.0)
        al.forward_cached(batch, caches[0], seqs, starts, out=out)
        _status_raises_once(caches[0])
        assert (out == 3).all() and all(torch.equal(a, b) for a, b in zip(before, _bits(caches[0])))
    al.close()
