"""The paged K/V cache without a GPU: the oracle's rules, and every refusal that the host
makes before it touches CUDA."""
from __future__ import annotations

import ctypes
import random
from ctypes import byref, c_int64, c_void_p

import numpy as np
import pytest
import torch

from moe_sm100 import _lib
from moe_sm100.paged import _ATTEND_ARGS, PagedKVCache
from oracle.paged_oracle import OracleError, PagedOracle, attend_chunk


# ------------------------------------------------------------------ the oracle
def test_oracle_keeps_its_invariants_under_random_steps() -> None:
    rng = random.Random(5)
    o = PagedOracle(1, 40, 4, 1, 2, 12, 8)
    done = 0
    for _ in range(600):
        seqs = rng.sample(range(12), rng.randint(1, 4))
        try:
            kind = rng.randrange(4)
            if kind == 0:
                o.reserve(seqs, [rng.randint(0, 9) for _ in seqs])
            elif kind == 1 and len(seqs) > 1:
                o.fork([seqs[0]] * (len(seqs) - 1), seqs[1:])
            elif kind == 2:
                o.truncate(seqs, [rng.randint(0, max(o.lengths[s], 1)) for s in seqs])
            else:
                o.compact()
            done += 1
        except OracleError:
            pass
        o.check_invariants()
    assert done > 200


def test_oracle_copies_a_shared_page_before_it_is_written() -> None:
    o = PagedOracle(2, 10, 4, 1, 2, 3, 4)
    o.reserve([0], [6])
    x = np.arange(6 * 2, dtype=float).reshape(6, 1, 2)
    o.append(1, x, -x, [0], [0, 6])
    o.fork([0, 0], [1, 2])
    assert o.refs[:2] == [3, 3]
    o.reserve([1], [1])
    assert o.table[1][1] != o.table[0][1] and o.refs[:3] == [3, 2, 1]
    for s in (0, 1, 2):
        np.testing.assert_array_equal(o.cached(1, s)[0][:6], x)
    o.append(1, x[:1] + 100, x[:1], [1], [0, 1])
    np.testing.assert_array_equal(o.cached(1, 0)[0], x)


def test_oracle_attention_of_one_token_is_its_value() -> None:
    rng = np.random.default_rng(0)
    v = rng.standard_normal((1, 1, 8))
    out, lse, _ = attend_chunk(rng.standard_normal((1, 2, 8)), np.ones((1, 1, 8)), v, 0.5)
    np.testing.assert_allclose(out[0, 0], v[0, 0])
    assert np.isfinite(lse).all()
    out, lse, _ = attend_chunk(rng.standard_normal((3, 2, 8)), np.ones((1, 1, 8)), v, 0.5)
    assert (out[:2] == 0).all() and (lse[:2] == -np.inf).all() and np.isfinite(lse[2]).all()


# ------------------------------------------------------------------ refusals of the host
def _cfg(**kw) -> _lib.MoeKvConfigC:
    base = dict(k=16, v=16, k_strides=(c_int64 * 4)(4096, 2048, 1024, 64),
                v_strides=(c_int64 * 4)(4096, 2048, 1024, 64), block_table=16, lengths=16, refs=16,
                scratch=16, dtype=_lib.MOE_KV_F16, layers=1, pages=2, kv_heads=2, page_size=16,
                head_dim=64, sequences=4, max_blocks=3, device=0)
    base.update(kw)
    return _lib.MoeKvConfigC(**base)


@pytest.mark.parametrize("bad,code", [
    (dict(dtype=7), _lib.MOE_ERR_UNSUPPORTED),
    (dict(head_dim=96), _lib.MOE_ERR_UNSUPPORTED),
    (dict(page_size=24), _lib.MOE_ERR_UNSUPPORTED),
    (dict(page_size=8), _lib.MOE_ERR_UNSUPPORTED),
    (dict(page_size=512), _lib.MOE_ERR_UNSUPPORTED),
    (dict(page_size=0), _lib.MOE_ERR_UNSUPPORTED),
    (dict(pages=0), _lib.MOE_ERR_INVALID),
    (dict(pages=(1 << 26) + 1), _lib.MOE_ERR_UNSUPPORTED),
    (dict(layers=0), _lib.MOE_ERR_INVALID),
    (dict(kv_heads=-1), _lib.MOE_ERR_INVALID),
    (dict(sequences=0), _lib.MOE_ERR_INVALID),
    (dict(sequences=65537), _lib.MOE_ERR_UNSUPPORTED),
    (dict(max_blocks=0), _lib.MOE_ERR_INVALID),
    (dict(k=None), _lib.MOE_ERR_INVALID),
    (dict(k=8), _lib.MOE_ERR_INVALID),
    (dict(refs=None), _lib.MOE_ERR_INVALID),
    (dict(scratch=None), _lib.MOE_ERR_INVALID),
    (dict(k_strides=(c_int64 * 4)(4096, 2048, 1024, 60)), _lib.MOE_ERR_INVALID),  # rows overlap
    (dict(v_strides=(c_int64 * 4)(4096, 2048, 1028, 64)), _lib.MOE_ERR_INVALID),  # not 16 bytes
    (dict(v_strides=(c_int64 * 4)(4096, 0, 1024, 64)), _lib.MOE_ERR_INVALID),     # pages overlap
])
def test_create_refuses(built_lib: str, bad: dict, code: int) -> None:
    h = c_void_p()
    assert _lib.lib().moe_kv_create(byref(_cfg(**bad)), byref(h)) == code
    assert _lib.lib().moe_last_error().decode()
    assert not h.value


def test_null_arguments_are_errors(built_lib: str) -> None:
    lib = _lib.lib()
    assert lib.moe_kv_create(None, None) == _lib.MOE_ERR_INVALID
    assert lib.moe_kv_scratch_bytes(None) == 0
    assert lib.moe_kv_scratch_bytes(byref(_cfg(pages=0))) == 0
    assert lib.moe_kv_scratch_bytes(byref(_cfg())) >= 4 * (16 + 3 * 4 + 2 + 4)
    assert lib.moe_kv_destroy(None) == _lib.MOE_OK
    assert lib.moe_kv_reserve(None, None, None, 1, None) == _lib.MOE_ERR_INVALID
    assert lib.moe_kv_fork(None, None, None, 1, None) == _lib.MOE_ERR_INVALID
    assert lib.moe_kv_truncate(None, None, None, 1, None) == _lib.MOE_ERR_INVALID
    assert lib.moe_kv_copy_pages(None, None, None, 1, None) == _lib.MOE_ERR_INVALID
    assert lib.moe_kv_compact(None, None, None) == _lib.MOE_ERR_INVALID
    assert lib.moe_kv_append(None, 0, None, None, 0, 0, 0, 0, None, None, 1, 1, None) == \
        _lib.MOE_ERR_INVALID
    assert lib.moe_kv_attend(None, None, None, 0, None) == _lib.MOE_ERR_INVALID
    assert lib.moe_kv_attend_workspace_bytes(None, 8, 1, 1) == 0
    assert lib.moe_kv_status(None, None) == _lib.MOE_ERR_INVALID


def test_cache_refuses_host_tensors_and_wrong_types(built_lib: str) -> None:
    pool = torch.zeros((1, 2, 2, 16, 64), dtype=torch.float16)
    table, lengths, refs = (torch.zeros(s, dtype=torch.int32) for s in ((4, 3), (4,), (2,)))
    with pytest.raises(TypeError):
        PagedKVCache(pool, pool, table, lengths, refs)
    with pytest.raises(TypeError):
        PagedKVCache(pool.float(), pool.float(), table, lengths, refs)
    with pytest.raises(TypeError):
        PagedKVCache(None, pool, table, lengths, refs)


def test_struct_sizes_match_the_header() -> None:
    # natural alignment of the C declarations
    assert ctypes.sizeof(_lib.MoeKvConfigC) == 2 * 8 + 8 * 8 + 4 * 8 + 9 * 4 + 4
    assert ctypes.sizeof(_lib.MoeKvAttendArgsC) == 3 * 8 + 6 * 8 + 2 * 8 + 4 * 4 + 4 + 4
    # the packed form that calls pass has the structure's bytes
    values = list(range(1, 16)) + [0.5]
    assert _ATTEND_ARGS.pack(*values) == bytes(_lib.MoeKvAttendArgsC(*values))


def test_error_code_of_an_exhausted_pool_is_a_runtime_error() -> None:
    with pytest.raises(RuntimeError) as e:
        _lib.check(_lib.MOE_ERR_NO_PAGES)
    assert e.value.code == _lib.MOE_ERR_NO_PAGES and not isinstance(e.value, ValueError)
