"""The GLM-4 attention block over the paged cache (needs a B200): sequences fed in chunks and
token by token, in batches, against the oracle's block over each whole sequence.

The device rounds q, k, v and P to f16 as the whole-sequence path does, so the tolerances
are that path's (tests/test_gpu_attention.py): block output rel-L2 2e-3, attention part 1e-2.
"""
from __future__ import annotations

import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]

from moe_sm100.attention import AttentionConfig, AttentionLayer  # noqa: E402
from moe_sm100.packing import pack_layer  # noqa: E402
from moe_sm100.paged import PagedKVCache  # noqa: E402
from oracle.attention_oracle import AttnConfig, glm4_attention_block  # noqa: E402
from oracle.cases import AttnSpec, make_attn_case  # noqa: E402

TOL_BLOCK, TOL_DELTA = 2e-3, 1e-2


def _rel(a: np.ndarray, b: np.ndarray) -> float:
    return float(np.linalg.norm(a.astype(np.float64) - b) / np.linalg.norm(b.astype(np.float64)))


def _layer(spec: AttnSpec, t: dict, max_tokens: int) -> AttentionLayer:
    blob, meta = pack_layer(t)
    al = AttentionLayer(AttentionConfig.glm4_moe(spec.hf_config(), max_tokens=max_tokens))
    al.bind_host(blob, meta)
    return al


def _cache(spec: AttnSpec, seqs: int, blocks: int, page: int, layers: int = 1) -> PagedKVCache:
    return PagedKVCache.allocate(layers=layers, pages=seqs * blocks + 2, page_size=page,
                                 kv_heads=spec.kv_heads, head_dim=spec.head_dim, sequences=seqs,
                                 max_blocks=blocks)


SPECS = {
    "glm47_heads": (AttnSpec(hidden=1024, heads=96, kv_heads=8, head_dim=128, tokens=150, seed=61), 16),
    "gqa8": (AttnSpec(hidden=512, heads=16, kv_heads=2, head_dim=128, tokens=330, seed=62), 64),
    "mha_hd64": (AttnSpec(hidden=512, heads=8, kv_heads=8, head_dim=64, tokens=200, seed=63,
                          qk_norm=False, partial_rotary_factor=1.0, rope_theta=10000.0), 32),
}


@pytest.mark.parametrize("name", sorted(SPECS))
def test_chunks_and_tokens_match_the_whole_sequence(name: str) -> None:
    spec, page = SPECS[name]
    x, t = make_attn_case(spec)
    al = _layer(spec, t, 512)
    rng = random.Random(7)
    # three sequences of different lengths over the same weights, in one batch per step
    lens = [spec.tokens, spec.tokens // 2 + 1, 3]
    xs = [x, np.ascontiguousarray(x[::-1][:lens[1]]), np.ascontiguousarray(x[5:8])]
    refs = [glm4_attention_block(v, t, AttnConfig.from_hf(spec.hf_config())) for v in xs]
    cache = _cache(spec, 4, -(-spec.tokens // page), page)
    done, outs = [0, 0, 0], [np.zeros_like(v) for v in xs]
    while any(d < n for d, n in zip(done, lens)):
        new = [min(n - d, rng.choice([1, 1, 2, 7, 40, 130])) for d, n in zip(done, lens)]
        order = rng.sample(range(3), 3)
        starts = [0] + np.cumsum([new[s] for s in order]).tolist()
        batch = np.concatenate([xs[s][done[s]:done[s] + new[s]] for s in order])
        cache.reserve([s + 1 for s in order], [new[s] for s in order])
        out = al.forward_cached(torch.from_numpy(batch).cuda(), cache, [s + 1 for s in order], starts)
        out = out.cpu().numpy()
        for i, s in enumerate(order):
            outs[s][done[s]:done[s] + new[s]] = out[starts[i]:starts[i + 1]]
            done[s] += new[s]
    cache.status()
    al.status()
    for got, ref, v in zip(outs, refs, xs):
        assert np.isfinite(got).all()
        eb, ed = _rel(got, ref), _rel(got - v, ref - v)
        assert eb <= TOL_BLOCK and ed <= TOL_DELTA, (eb, ed)
    al.close()


def test_branches_of_one_prompt_in_a_graph() -> None:
    """A prompt, forked into four branches that decode different tokens, the step captured
    and replayed (the run of the cache's operators together), against the whole sequences."""
    spec = AttnSpec(hidden=512, heads=16, kv_heads=2, head_dim=128, tokens=60, seed=64)
    x, t = make_attn_case(spec)
    al = _layer(spec, t, 256)
    cache = _cache(spec, 6, 6, 16, layers=2)
    prompt = x[:41]
    kids = [1, 2, 3, 5]
    cache.reserve([0], [41])
    al.forward_cached(torch.from_numpy(prompt).cuda(), cache, [0], [0, 41], layer=1)
    cache.fork([0] * 4, kids)
    seqs = torch.tensor(kids, dtype=torch.int32, device="cuda")
    ones, starts = torch.ones_like(seqs), torch.arange(5, dtype=torch.int32, device="cuda")
    steps = np.random.default_rng(3).standard_normal((20, 4, spec.hidden)).astype(np.float32)
    buf = torch.zeros((4, spec.hidden), device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        cache.reserve(seqs, ones)
        out = al.forward_cached(buf, cache, seqs, starts, layer=1)
    got = []
    for i in range(20):
        buf.copy_(torch.from_numpy(steps[i]))
        graph.replay()
        got.append(out.cpu().numpy().copy())
    cache.status()
    al.status()
    got = np.stack(got)
    for b in range(4):
        whole = np.concatenate([prompt, steps[:, b]])
        ref = glm4_attention_block(whole, t, AttnConfig.from_hf(spec.hf_config()))[41:]
        eb, ed = _rel(got[:, b], ref), _rel(got[:, b] - steps[:, b], ref - steps[:, b])
        assert eb <= TOL_BLOCK and ed <= TOL_DELTA, (b, eb, ed)
    # the branches are cut back to the prompt and freed: every page is the parent's again
    cache.truncate(kids, [41] * 4)
    cache.free(kids)
    cache.compact()
    cache.status()
    assert cache.lengths.tolist() == [41, 0, 0, 0, 0, 0]
    assert cache.refs.tolist() == [1, 1, 1] + [0] * (cache.refs.shape[0] - 3)
    al.close()


def test_padded_batches_and_refusals() -> None:
    spec = AttnSpec(hidden=512, heads=8, kv_heads=8, head_dim=64, tokens=20, seed=65)
    x, t = make_attn_case(spec)
    al = _layer(spec, t, 32)
    cache = _cache(spec, 2, 2, 16)
    xd = torch.from_numpy(x).cuda()
    cache.reserve([0, 1], [9, 4])
    seqs, starts = [0, 1], [0, 9, 13]
    out = torch.full_like(xd, 7.0)
    al.forward_cached(xd, cache, seqs, starts, out=out)
    cache.status()
    assert (out[13:] == 7).all()  # rows behind the last sequence are left alone
    ref = glm4_attention_block(x[:9], t, AttnConfig.from_hf(spec.hf_config()))
    assert _rel(out[:9].cpu().numpy(), ref) <= TOL_BLOCK
    with pytest.raises(ValueError):
        al.forward_cached(torch.zeros((33, 512), device="cuda"), cache, [0], [0, 33])  # > max_tokens
    with pytest.raises(ValueError):
        al.forward_cached(xd, cache, seqs, starts, layer=1)
    with pytest.raises(ValueError):
        al.forward_cached(xd, cache, seqs, starts, out=xd)
    with pytest.raises(TypeError):
        al.forward_cached(xd.cpu(), cache, seqs, starts)
    with pytest.raises(ValueError):
        al.forward_cached(xd[:, :256], cache, seqs, starts)
    other = PagedKVCache.allocate(layers=1, pages=4, page_size=16, kv_heads=2, head_dim=64,
                                  sequences=2, max_blocks=2)
    with pytest.raises(ValueError):
        al.forward_cached(xd, other, seqs, starts)
    half = PagedKVCache.allocate(layers=1, pages=4, page_size=16, kv_heads=8, head_dim=64, sequences=2,
                                 max_blocks=2, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        al.forward_cached(xd, half, seqs, starts)
    assert al.forward_cached(xd[:0], cache, [], [0]).shape == (0, 512)
    out = al.forward_cached(xd[:13], cache, [0, 9], [0, 9, 13])  # no such sequence
    with pytest.raises(ValueError):
        cache.status()
    assert torch.isfinite(out).all()
    al.close()
