"""Calls of the 4-bit cache and of token eviction at the edges of what their documents allow, against the restatement."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from elasticmm_b200 import KVPool, ScorePool, _lib
from gpu_util import assert_clean
from oracle import q4_oracle
from test_gpu_q4 import check_out, check_scores, ctx, dev, random_pool, score_values, tables_for  # noqa: F401

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


# ------------------------------------------------------------------------------------- blocks outside the pool
@pytest.mark.parametrize("D,H,BS,bad_place", [(128, 4, 16, 1), (128, 8, 16, 0), (64, 4, 16, 3), (256, 4, 32, 1), (128, 4, 8, 5), (128, 4, 5, 4)])
def test_a_bad_block_hides_no_other_sequences_tokens(ctx, D, H, BS, bad_place):
    """Every CTA goes through many short sequences. A few have one block outside the pool; the sequences behind them keep
    all their tokens, in the result and in the weights."""
    n, B = 64, 900
    lens = [n] * B
    per = -(-n // BS)
    pool, bytes_ = random_pool(1, B * per, BS, H, D, False, 1)
    tables = tables_for(lens, B * per, BS, 2)
    broken, bad = tables.copy(), list(range(7, B, 97))
    broken[bad, bad_place] = B * per
    q = torch.randn(B, H, D, generator=torch.Generator().manual_seed(3)).to(BF)
    before = np.random.default_rng(4).random((B * per, H, BS), dtype=np.float32)
    scores = ScorePool([dev(before)], ctx)
    out = pool.attend(0, q.cuda(), dev(broken), dev(np.array(lens, dtype=np.int32)), scores=scores)
    assert ctx.status() == (_lib.ERR_ID_RANGE, B * per)
    # the tokens of a bad block are left out: the same sequence without that block
    left, left_lens = tables.copy(), np.array(lens)
    left[bad, bad_place:-1] = tables[bad, bad_place + 1:]
    left_lens[bad] -= min(BS, n - bad_place * BS)
    ref, weights, bound, spread = q4_oracle.attend(bytes_[0], D, q.double().numpy(), left, left_lens, D ** -0.5)
    check_out(out, ref, bound, spread, BF)
    check_scores(scores.layers[0], before, left, left_lens, weights, spread, 1)
    assert_clean(ctx)


@pytest.mark.parametrize("bad_place", [0, 24, 25, 31, 32, 47])
@pytest.mark.parametrize("D,BS,dtype", [(128, 16, BF), (64, 16, FP), (128, 8, FP)])
def test_a_bad_block_hides_no_later_tokens_of_its_sequence(ctx, D, BS, dtype, bad_place):
    """Sequences of many table windows of 32 blocks, one for each SM and more, all with the same block missing."""
    n, H, B = 1100 // BS * BS, 8, 160
    NB = n // BS
    pool, bytes_ = random_pool(1, NB, BS, H, D, False, 1)
    table = tables_for([n], NB, BS, 2)
    broken = table.copy()
    broken[0, bad_place] = -3
    q = torch.randn(1, H, D, generator=torch.Generator().manual_seed(3)).to(dtype)
    out = pool.attend(0, q.cuda().repeat(B, 1, 1), dev(broken.repeat(B, 0)), dev(np.full(B, n, dtype=np.int32)))
    assert ctx.status() == (_lib.ERR_ID_RANGE, -3)
    ref, _, bound, spread = q4_oracle.attend(bytes_[0], D, q.double().numpy(), np.delete(table, bad_place, 1), [n - BS], D ** -0.5)
    check_out(out, ref, bound, spread, dtype)
    assert_clean(ctx)


# ------------------------------------------------------------------------------------------------- token selection
_FIRST_SELECTION = """
import sys
import numpy as np, torch
from elasticmm_b200 import ScorePool
from oracle import q4_oracle
n, BS = int(sys.argv[1]), int(sys.argv[2])
values = np.random.default_rng(n).random((1, n // BS, 1, BS), dtype=np.float32)
scores = ScorePool([torch.from_numpy(values[0]).cuda()])
tables = np.random.default_rng(1).permutation(n // BS).astype(np.int32)[None]
index, lens = scores.select_tokens(torch.from_numpy(tables).cuda(), torch.tensor([n], dtype=torch.int32, device="cuda"),
                                   500, recent=20, sink=3)
assert (index.cpu().numpy() == q4_oracle.select_tokens(values, tables, [n], 500, 20, 3)).all()
assert lens.tolist() == [500]
scores.ctx.check_status()
print("selected")
"""


@pytest.mark.parametrize("n,BS", [(11680, 16), (11681, 1), (12288, 16), (12289, 1), (51200, 16), (51201, 1)])
def test_the_first_selection_of_a_process(n, BS):
    """Tables of every capacity launch without a larger call before them: around 48 KiB of keys, with and without the
    kernel's static shared memory, and around the most keys that are held at all."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", _FIRST_SELECTION, str(n), str(BS)], cwd=root, capture_output=True, text=True,
                         timeout=300, env={**os.environ, "PYTHONPATH": root})
    assert run.returncode == 0 and "selected" in run.stdout, run.stderr[-2000:]


# -------------------------------------------------------------------------------------------------------- eviction
def _any_pool(ctx, kind, L, NB, BS, H, hnd, seed):
    """(pool, its logical contents [L, 2, NB, BS, H, row]) of 16-bit, 4-bit or byte rows."""
    if kind == "q4":
        return random_pool(L, NB, BS, H, 128, hnd, seed)
    D, store, dtype = {"64": (64, np.int16, BF), "128": (128, np.int16, BF), "5": (5, np.int16, FP), "301": (301, np.int16, FP),
                       "601 bytes": (601, np.uint8, torch.uint8)}[kind]
    ref = np.random.default_rng(seed).integers(0, 1 << (7 if store == np.uint8 else 15), (L, 2, NB, BS, H, D)).astype(store)
    if hnd:
        layers = [dev(x.swapaxes(2, 3)).view(dtype).permute(0, 1, 3, 2, 4) for x in ref]
    else:
        layers = [dev(x).view(dtype) for x in ref]
    return KVPool(layers, ctx), ref


@pytest.mark.parametrize("hnd", [False, True], ids=["nhd", "hnd"])
@pytest.mark.parametrize("kind", ["64", "128", "q4", "5", "301", "601 bytes"])
@pytest.mark.parametrize("BS", [1, 5, 48])
@pytest.mark.parametrize("keep,recent,sink", [(64, 10, 3), (1, 0, 0), (200, 100, 100), (257, 0, 4)])
def test_select_and_keep_in_blocks_of_any_size(ctx, kind, BS, keep, recent, sink, hnd):
    """Blocks of one token and of sizes that are no power of two; rows of more vectors than a block has threads; few and
    many CTAs to a row."""
    L, H = 2, 3
    lens = [0, 1, 63, 64, 65, 257, 258, 300, 1111]
    NB = sum(-(-n // BS) for n in lens) + 4
    pool, ref = _any_pool(ctx, kind, L, NB, BS, H, hnd, keep)
    values = score_values((L, NB, H, BS), keep)
    scores = ScorePool(list(dev(values).unbind(0)), ctx)
    tables = tables_for(lens, NB, BS, 6, extra=1)
    t_d, l_d = dev(tables), dev(np.array(lens, dtype=np.int32))
    index, new_lens = scores.select_tokens(t_d, l_d, keep, recent=recent, sink=sink)
    want = q4_oracle.select_tokens(values, tables, lens, keep, recent, sink)
    assert (index.cpu().numpy() == want).all() and new_lens.tolist() == [min(n, keep) for n in lens]
    pool.keep_tokens(index, t_d, l_d)
    scores.keep_tokens(index, t_d, l_d)
    assert_clean(ctx)
    ref = ref.copy()
    q4_oracle.keep_tokens(ref, want, tables, lens, keep)
    for l in range(L):
        assert (pool.layers[l].contiguous().view(torch.from_numpy(ref).dtype).cpu().numpy() == ref[l]).all()
    moved = values[:, None].swapaxes(3, 4)[..., None].copy()
    q4_oracle.keep_tokens(moved, want, tables, lens, keep)
    for l in range(L):
        assert np.array_equal(scores.layers[l].cpu().numpy(), moved[l, 0, ..., 0].swapaxes(1, 2), equal_nan=True)


@pytest.mark.parametrize("BS", [16, 5])
@pytest.mark.parametrize("D,L,B", [(128, 1, 1), (128, 1, 70), (128, 2, 80), (48, 1, 2), (80, 1, 1), (256, 1, 1), (1024, 1, 1)])
def test_rows_shared_by_several_ctas(ctx, D, L, B, BS):
    """One, two and four CTAs to a row, with and without bytes that do not fill a CTA's vectors evenly."""
    H, n, keep = 2, 333, 150
    lens = [n - b for b in range(B)]
    NB = sum(-(-m // BS) for m in lens)
    ref = np.random.default_rng(D).integers(0, 1 << 15, (L, 2, NB, BS, H, D)).astype(np.int16)
    pool = KVPool([dev(x).view(BF) for x in ref], ctx)
    values = score_values((L, NB, H, BS), D)
    scores = ScorePool(list(dev(values).unbind(0)), ctx)
    tables = tables_for(lens, NB, BS, 6)
    t_d, l_d = dev(tables), dev(np.array(lens, dtype=np.int32))
    index, _ = scores.select_tokens(t_d, l_d, keep, recent=20, sink=1)
    want = q4_oracle.select_tokens(values, tables, lens, keep, 20, 1)
    assert (index.cpu().numpy() == want).all()
    pool.keep_tokens(index, t_d, l_d)
    assert_clean(ctx)
    q4_oracle.keep_tokens(ref, want, tables, lens, keep)
    for l in range(L):
        assert (pool.layers[l].view(torch.int16).cpu().numpy() == ref[l]).all()


# ------------------------------------------------------------------------------------------------------------ rows
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("D,H,BS,hnd", [(64, 3, 16, False), (128, 2, 5, True), (256, 1, 16, False)])
def test_rows_read_into_memory_off_32_byte_boundaries(ctx, D, H, BS, hnd, dtype):
    """The C entry with outputs at an odd element, gaps between tokens, layers and planes: every row equal to what read()
    gives, zeros for a padding slot and a reported one, and nothing written between them."""
    L, NB, T = 3, 8, 21
    pool, _ = random_pool(L, NB, BS, H, D, hnd, 3, gain=4.0)
    g = torch.Generator().manual_seed(D)
    slots = torch.randperm(NB * BS, generator=g)[:T].cuda()
    slots[4], slots[9] = -1, NB * BS
    key, value = pool.read(slots, dtype, 1, 2)
    assert ctx.status() == (_lib.ERR_ID_RANGE, NB * BS)
    token, layer = H * D + 3, T * (H * D + 3) + 11
    out = torch.full((2, 2 * layer + 1), 7.0, dtype=dtype, device="cuda")
    at = [out[p].data_ptr() + 2 * (1 - p) for p in (0, 1)]  # elements 1 of the first plane, 0 of the second
    rc = ctx._lib.emm_q4_read(pool._h, D, _lib.DTYPE_FP16 if dtype == FP else _lib.DTYPE_BF16, 1, 2, at[0], at[1], layer * 2,
                              token * 2, layer * 2, token * 2, slots.data_ptr(), T, torch.cuda.current_stream().cuda_stream)
    assert rc == _lib.OK and ctx.status() == (_lib.ERR_ID_RANGE, NB * BS)
    want = torch.full_like(out, 7.0)
    for p, rows in enumerate((key, value)):
        for l in range(2):
            for t in range(T):
                first = (1 - p) + l * layer + t * token
                want[p, first:first + H * D] = rows[l, t].flatten()
    assert torch.equal(out, want)
    assert (key[:, [4, 9]] == 0).all() and (value[:, [4, 9]] == 0).all()
    assert_clean(ctx)
