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
