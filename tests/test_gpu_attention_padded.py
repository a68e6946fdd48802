"""The GLM-4 attention block over the paged cache on padded batches (needs a B200): rows that
belong to no entry may hold anything."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]

from moe_sm100._lib import MoeError  # noqa: E402
from oracle.cases import AttnSpec, make_attn_case  # noqa: E402
from test_gpu_attention_cached import _cache, _layer  # noqa: E402


@pytest.mark.parametrize("value", [float("nan"), float("inf"), 3.0e38])
def test_padded_rows_report_nothing(value: float) -> None:
    spec = AttnSpec(hidden=512, heads=16, kv_heads=2, head_dim=128, tokens=30, seed=73)
    x, t = make_attn_case(spec)
    al = _layer(spec, t, 64)
    outs = []
    for fill in (0.0, value):
        cache = _cache(spec, 2, 2, 16)
        cache.reserve([0, 1], [9, 4])
        batch = torch.full((20, spec.hidden), fill, device="cuda")
        batch[3:16] = torch.from_numpy(x[:13]).cuda()
        out = torch.full_like(batch, 7.0)
        al.forward_cached(batch, cache, [0, 1], [3, 12, 16], out=out)
        cache.status()
        al.status()
        assert (out[:3] == 7).all() and (out[16:] == 7).all()
        outs.append((out, cache.k, cache.v))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    # a row of an entry is still checked (3e38 squared is infinite, and x / inf is zero: the
    # norm of such a row is finite)
    batch[5, 1] = value
    al.forward_cached(batch, cache, [0, 1], [3, 12, 16])
    if value == 3.0e38:
        al.status()
    else:
        with pytest.raises(MoeError):
            al.status()
    al.close()
