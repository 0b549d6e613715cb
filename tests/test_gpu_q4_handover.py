"""Blocks that enter a 4-bit worker: whose weights they have, one request or several at a time, from 16 bits or 4."""
import numpy as np
import pytest
import torch

from elasticmm_b200.engine.v0 import V0Worker
from test_gpu_q4_worker import BS, D, H, L, NB, _worker

pytestmark = pytest.mark.gpu


def _blocks(n, seed, dtype=torch.bfloat16):
    return torch.randn(L, 2, n, BS, H, D, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _weights(w):
    return np.stack([x.cpu().numpy() for x in w.scores.layers])


@pytest.mark.parametrize("many", [False, True], ids=["one", "many"])
@pytest.mark.parametrize("bits", [4, 16])
def test_written_blocks_start_without_weights(many, bits):
    """The weights that an earlier request left in the blocks go; those of all others stay."""
    if bits == 4:
        w, source = _worker(), _worker()
    else:
        w, source = (V0Worker(dtype="bfloat16", device="cuda:0", block_size=BS) for _ in range(2))
        for x in (w, source):
            x.init_kvcache(NB, L, H, D)
    w.init_scores()
    for l, layer in enumerate(w.scores.layers):
        layer.fill_(1.0 + l)
    want = _weights(w)
    source.write_kv_blocks(list(range(6)), _blocks(6, 1))
    if many:
        w.write_kv_blocks_many([[7, 3], [], [20]], source.extract_kv_blocks_many([[0, 5], [], [2]]))
    else:
        w.write_kv_blocks([7, 3, 20], source.extract_kv_blocks([0, 5, 2]))
    want[:, [7, 3, 20]] = 0
    assert (_weights(w) == want).all()
    assert torch.equal(w.extract_kv_blocks([7, 3, 20]), source.extract_kv_blocks([0, 5, 2]))
    if bits == 4 and not many:
        w.write_kv_blocks([1, 22], _blocks(2, 2))  # a 16-bit worker's
        want[:, [1, 22]] = 0
        assert (_weights(w) == want).all()
    w.ctx.check_status()


def test_an_eviction_after_a_hand_over_goes_by_the_new_requests_weights():
    """A prompt enters blocks that an evicted request left with large weights: they do not choose what stays."""
    w = _worker()
    w.init_scores()
    for layer in w.scores.layers:
        layer.copy_(torch.arange(NB, 0, -1, device="cuda").view(-1, 1, 1).expand_as(layer))
    ids = [9, 4, 17]
    w.write_kv_blocks(ids, _blocks(3, 3))
    tables = torch.tensor([ids], dtype=torch.int32, device="cuda")
    for layer in w.scores.layers:
        layer[17, :, 5] = 1e-3  # position 37 was looked at, no other
    res = w.evict_tokens(tables, torch.tensor([3 * BS], dtype=torch.int32, device="cuda"), 2)
    assert (res["index"].cpu() == torch.tensor([0, 37])).all()
