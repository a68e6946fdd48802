"""Values that attention over the paged cache has to keep apart (needs a B200): what a page
holds past a sequence's end."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]

from test_gpu_paged import _attend_case  # noqa: E402


# ------------------------------------------------------------------ past the end
@pytest.mark.parametrize("dtype,dim", [("f16", 128), ("bf16", 64)])
@pytest.mark.parametrize("heads,kv_heads", [(8, 8), (24, 2)])
@pytest.mark.parametrize("page", [16, 256])
def test_many_more_new_rows_than_tokens(dtype: str, dim: int, heads: int, kv_heads: int, page: int) -> None:
    """Rows without a token and rows with a few, in units of every size, next to long chunks
    (so that the shares hold whole units); the pages hold NaN past the tokens."""
    _attend_case(dtype, heads, kv_heads, dim, page,
                 [(10, 300), (5, 320), (1, 70), (64, 500), (65, 130), (2000, 1000), (0, 200)], seed=page + heads)
