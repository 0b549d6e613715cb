"""Calls of the 4-bit cache and of token eviction at the edges of what their documents allow, against the restatement."""
import os
import subprocess
import sys

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
