"""Calls of the 4-bit cache and of token eviction at the edges of what their documents allow, against the restatement."""
import numpy as np
import pytest
import torch

from elasticmm_b200 import ScorePool, _lib
from gpu_util import assert_clean
from oracle import q4_oracle
from test_gpu_q4 import check_out, check_scores, ctx, dev, random_pool, tables_for  # noqa: F401

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
