"""The 4-bit row format and the checks that need no GPU."""
import ctypes as C
import types

import numpy as np
import pytest
import torch

from elasticmm_b200 import KVPoolQ4, ScorePool, _lib
from elasticmm_b200.kv_pool import check_block_tables
from oracle import q4_oracle


@pytest.mark.parametrize("D", [64, 128, 256])
def test_row_bytes_and_the_error_of_a_row(D):
    assert KVPoolQ4.row_bytes(D) == q4_oracle.row_bytes(D) == {64: 48, 128: 80, 256: 160}[D]
    rng = np.random.default_rng(D)
    x = rng.standard_normal((50, D)).astype(np.float16).astype(np.float32)
    x[1] *= 100
    x[2] += 7
    x[3] = 1.5
    rows = q4_oracle.encode_rows(x)
    assert rows.shape == (50, q4_oracle.row_bytes(D))
    got = q4_oracle.decode_rows(rows, D)
    g = x.reshape(50, -1, 32).astype(np.float64)
    span = g.max(-1) - g.min(-1)
    # half a step of the code; the grid's own shift: o is rounded by at most 2^-11 of itself (so is the place of the
    # ends, through s, by 8 steps of 2^-11)
    top = np.abs(g).max(-1)
    tol = span / 30 * (1 + 2.0 ** -10) + 2.0 ** -11 * top * 1.1 + 8 * span / 15 * 2.0 ** -11
    assert (np.abs(got.reshape(50, -1, 32) - g) <= tol[..., None]).all()
    assert (got[3] == 1.5).all()


def test_rows_of_extreme_groups():
    x = np.zeros((5, 64), dtype=np.float32)
    x[0, 3] = np.nan
    x[1, 5], x[1, 6] = np.inf, -np.inf
    x[2] = 65504.0
    x[3, :32] = np.linspace(0, 2.0 ** -20, 32)
    got = q4_oracle.decode_rows(q4_oracle.encode_rows(x), 64)
    assert np.isnan(got[0, :32]).all() and (got[0, 32:] == 0).all()
    s = np.float64(np.float16(131008 / 15))
    assert np.isfinite(got[1]).all() and abs(got[1, 5] - 65504) <= s and abs(got[1, 6] + 65504) <= s
    assert (got[2] == 65504.0).all()
    assert np.abs(got[3] - x[3]).max() <= 2.0 ** -20
    assert (got[4] == 0).all()


def test_unsupported_head_sizes_are_refused():
    lib = _lib.load()
    for bad in (0, -1, 32, 96, 80, 512):
        assert lib.emm_q4_row_bytes(bad) == 0
        with pytest.raises(ValueError, match="64, 128 or 256"):
            KVPoolQ4.row_bytes(bad)


def test_pools_check_their_tensors():
    with pytest.raises(ValueError, match="uint8 layer tensors"):
        KVPoolQ4([torch.zeros(2, 4, 16, 2, 128, dtype=torch.uint8)], 128)   # 128 bytes are no row of 128 channels
    with pytest.raises(ValueError, match="uint8 layer tensors"):
        KVPoolQ4([torch.zeros(2, 4, 16, 2, 80, dtype=torch.int8)], 128)
    with pytest.raises(ValueError, match="CUDA"):
        KVPoolQ4([torch.zeros(2, 4, 16, 2, 80, dtype=torch.uint8)], 128)
    with pytest.raises(ValueError, match="fp32"):
        ScorePool([torch.zeros(4, 2, 16, dtype=torch.float16)])
    with pytest.raises(ValueError, match="CUDA"):
        ScorePool([torch.zeros(4, 2, 16)])


def test_block_tables_are_checked():
    pool = types.SimpleNamespace(device=torch.device("cpu"))
    tables, lens = torch.zeros(3, 5, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    assert check_block_tables(pool, tables, lens) == (3, 5)
    assert check_block_tables(pool, torch.zeros(3, 9, dtype=torch.int32)[:, :5], lens) == (3, 5)
    for bad in (tables.long(), tables[0], torch.zeros(5, 3, dtype=torch.int32).t(), tables[:, ::2],
                tables[:1].expand(3, 5)):
        with pytest.raises(ValueError, match="block_tables"):
            check_block_tables(pool, bad, lens)
    for bad in (lens.long(), lens[:2], torch.zeros(6, dtype=torch.int32)[::2], lens[None]):
        with pytest.raises(ValueError, match="seq_lens"):
            check_block_tables(pool, tables, bad)


def test_entries_refuse_null_pools():
    lib = _lib.load()
    n = C.c_uint64()
    assert lib.emm_q4_append(None, 128, 0, 0, 1, None, None, 0, 0, 0, 0, None, 1, None) == _lib.ERR_BAD_ARG
    assert lib.emm_q4_read(None, 128, 0, 0, 1, None, None, 0, 0, 0, 0, None, 1, None) == _lib.ERR_BAD_ARG
    assert lib.emm_q4_attend_workspace(None, 128, 1, 8, 16, 0, C.byref(n)) == _lib.ERR_BAD_ARG
    assert lib.emm_q4_attend(None, 128, 0, 0, None, 0, None, 0, None, 0, 0, None, 1, 8, 16, 1.0, None, None, 0,
                             None) == _lib.ERR_BAD_ARG
    assert lib.emm_select_tokens(None, None, 0, 0, None, 1, 4, 0, 0, None, None, None) == _lib.ERR_BAD_ARG
    assert lib.emm_keep_tokens(None, None, 1, 4, None, 0, 0, None, 1, None) == _lib.ERR_BAD_ARG
    assert lib.emm_reset_scores(None, None, 1, None) == _lib.ERR_BAD_ARG
    assert b"null" in lib.emm_last_error()


def test_selection_by_the_restatement():
    """Ties go to the earlier token, NaN is the smallest, the ends are always kept."""
    scores = np.zeros((1, 2, 1, 4), dtype=np.float32)
    scores[0, 1, 0] = [0, 5, 5, np.nan]     # positions 0..3
    scores[0, 0, 0] = [5, 1, -0.0, 9]       # positions 4..7
    got = q4_oracle.select_tokens(scores, [[1, 0]], [8], 4, 1, 1)
    assert got[0, 0, 0].tolist() == [0, 1, 2, 7]
    got = q4_oracle.select_tokens(scores, [[1, 0]], [7], 6, 0, 0)
    assert got[0, 0, 0].tolist() == [0, 1, 2, 4, 5, 6]
    got = q4_oracle.select_tokens(scores, [[1, 0]], [3], 5, 2, 0)
    assert got[0, 0, 0].tolist() == [0, 1, 2, -1, -1]


def test_configuration_of_a_4_bit_cache():
    from elasticmm_b200.engine.v0 import V0KVCacheConfig
    c = V0KVCacheConfig(kv_bits=4, num_kv_heads=8, dtype="bfloat16")
    c.validate()
    for D, row in ((64, 48), (128, 80), (256, 160)):
        d = V0KVCacheConfig(kv_bits=4, num_kv_heads=8, head_size=D)
        d.validate()
        assert d.page_bytes == 16 * 8 * row == 16 * 8 * KVPoolQ4.row_bytes(D)
    assert V0KVCacheConfig.from_dict(c.to_dict()) == c
    for bad in (dict(kv_bits=8), dict(kv_bits=4, head_size=96), dict(kv_bits=4, dtype="float32")):
        with pytest.raises(AssertionError):
            V0KVCacheConfig(**bad).validate()


def test_truncated_tables_give_their_blocks_back():
    from elasticmm_b200.engine.v0 import Request, V0BlockManager
    bm = V0BlockManager("decoding", 10, 0, 16)
    bm.allocate_blocks(Request.of_length("a", 70))  # five blocks
    assert bm.truncate_blocks("a", 33) == [3, 4] and bm.get_block_table("a") == [0, 1, 2]
    assert bm.get_num_avail_gpu_blocks() == 7 and bm.free_gpu_blocks_list[-2:] == [3, 4]
    assert bm.truncate_blocks("a", 48) == [] and bm.truncate_blocks("a", 1000) == []
    assert bm.truncate_blocks("a", 0) == [0, 1, 2] and bm.get_block_table("a") == []
    with pytest.raises(ValueError):
        bm.truncate_blocks("b", 3)
    with pytest.raises(ValueError):
        bm.truncate_blocks("a", -1)


def _bound_append(L=2, H=1, D=64):
    """A bound append of a pool without a GPU: (append, pool, calls that reached the library with the pool's handle)."""
    calls, lib = [], _lib.load()

    def entry(handle, *args):
        if handle is None:
            return lib.emm_q4_append(handle, *args)
        calls.append((handle, *args))
        return _lib.OK

    pool = KVPoolQ4.__new__(KVPoolQ4)
    pool._h, pool.num_layers, pool.num_kv_heads, pool.head_dim = 77, L, H, D
    pool.ctx = types.SimpleNamespace(device=torch.device("cpu"), _lib=types.SimpleNamespace(emm_pool_destroy=lambda h: _lib.OK))
    pool._emm_q4_append = entry
    kv = torch.zeros(L, 3, H, D, dtype=torch.float16)
    return pool.bind_append(kv, kv.clone(), torch.arange(3)), pool, calls


def test_a_bound_append_ends_with_its_pool():
    append, pool, calls = _bound_append()
    append(1, 0)
    assert append.raw(0, 0) == _lib.OK and [c[0] for c in calls] == [77, 77]
    pool.close()
    with pytest.raises(_lib.EmmError, match="null pool"):
        append(0, 0)
    assert append.raw(1, 0) == _lib.ERR_BAD_ARG and len(calls) == 2


def test_a_released_append_is_refused():
    append, pool, calls = _bound_append()
    assert append.release() == _lib.OK and append.release() == _lib.OK
    with pytest.raises(_lib.EmmError, match="null pool"):
        append(0, 0)
    assert append.raw(1, 0) == _lib.ERR_BAD_ARG and calls == []
    pool.close()
