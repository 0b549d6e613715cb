"""Blocks that enter a 4-bit worker: whose weights they have, one request or several at a time, from 16 bits or 4."""
import asyncio

import numpy as np
import pytest
import torch

from elasticmm_b200.engine.v0 import TransferMethod, V0KVTransferManager, V0Worker
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


@pytest.mark.parametrize("layout", ["nhd", "hnd"])
@pytest.mark.parametrize("source", ["nhd", "hnd"])
def test_several_requests_of_a_16_bit_worker_enter_together(layout, source):
    """write_kv_blocks_many holds what write_kv_blocks does request by request, and takes all of a call or nothing."""
    wide = V0Worker(dtype="bfloat16", device="cuda:0", block_size=BS)
    wide.init_kvcache(NB, L, H, D, layout=source)
    for t in wide.kv_cache:
        t.normal_()
    one, many = _worker(layout), _worker(layout)
    src, dst = [[5, 0, 23], [], [7], [1, 2]], [[1, 22, 3], [], [9], [0, 14]]
    parts = wide.extract_kv_blocks_many(src)
    many.write_kv_blocks_many(dst, parts)
    for s, d in zip(src, dst):
        if s:
            one.write_kv_blocks(d, wide.extract_kv_blocks(s))
    for a, b in zip(one.kv_cache, many.kv_cache):
        assert torch.equal(a, b)
    held = [t.clone() for t in many.kv_cache]
    other = wide.extract_kv_blocks_many([[3], [4, 6]])
    for ids, data in (([[3], [3, 4]], other), ([[3], [4, NB]], other), ([[3], [4]], other), ([[3]], other),
                      ([[3], [4, 6]], [other[0], other[1].float()]), ([[3], [4, 6]], [other[0], other[1].cpu()]),
                      ([[3], [4, 6]], [other[0], many.extract_kv_blocks([4, 6])])):
        with pytest.raises(Exception):
            many.write_kv_blocks_many(ids, data)
        assert all(torch.equal(a, b) for a, b in zip(held, many.kv_cache))
    many.write_kv_blocks_many([], [])
    many.write_kv_blocks_many([[3], [4]], one.extract_kv_blocks_many([[22], [0]]))  # bytes, as before
    assert torch.equal(many.extract_kv_blocks([3, 4]), one.extract_kv_blocks([22, 0]))
    many.ctx.check_status()


def test_a_transfer_into_4_bits_does_the_same_with_and_without_batching():
    wide = V0Worker(dtype="bfloat16", device="cuda:0", block_size=BS)
    wide.init_kvcache(NB, L, H, D)
    for t in wide.kv_cache:
        t.normal_()
    got = []
    for batching in (False, True):
        w = _worker()
        mgr = V0KVTransferManager(transfer_method=TransferMethod.P2P_COPY, enable_batching=batching, batch_size=2,
                                  batch_timeout=3600.0)
        mgr.register_worker(0, wide, "prefill")
        mgr.register_worker(1, w, "decoding")
        for i, (s, d) in enumerate((([0, 4], [8, 1]), ([2], [3]), ([9, 7, 6], [0, 2, 20]))):
            assert asyncio.run(mgr.transfer_kv_cache(f"r{i}", 0, 1, s, d)), mgr.last_result
        assert mgr.flush(), mgr.last_result
        got.append([t.clone() for t in w.kv_cache])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_the_broadcast_form_moves_4_bit_blocks_as_bytes(monkeypatch):
    message = []

    def broadcast(t, src, group):
        if sending:
            message.append(t.clone())
        else:
            assert t.dtype == message[-1].dtype
            t.copy_(message[-1])

    monkeypatch.setattr("torch.distributed.broadcast", broadcast)
    a, b = _worker(), _worker("hnd")
    wide = V0Worker(dtype="bfloat16", device="cuda:0", block_size=BS)
    wide.init_kvcache(NB, L, H, D)
    for t in wide.kv_cache:
        t.normal_()
    a.write_kv_blocks([1, 2, 3], _blocks(3, 7))
    packed = a.extract_kv_blocks([3, 1])
    sending = True
    res = a.collective_transfer_kv(None, 0, [3, 1], packed.shape, "torch.uint8", "send")
    assert res["bytes"] == packed.numel()
    sending = False
    a.collective_transfer_kv(None, 0, [8, 9], packed.shape, a.get_kv_cache_layout()["dtype"], "recv")
    assert torch.equal(a.extract_kv_blocks([8, 9]), packed)
    sending = True
    wide.collective_transfer_kv(None, 0, [4, 0], (L, 2, 2, BS, H, D), "bfloat16", "send")
    sending = False
    b.collective_transfer_kv(None, 0, [5, 6], (L, 2, 2, BS, H, D), "bfloat16", "recv")
    a.write_kv_blocks([5, 6], wide.extract_kv_blocks([4, 0]))
    assert torch.equal(b.read_kv_blocks([5, 6]), a.read_kv_blocks([5, 6]))
    for worker, dtype, mode in ((a, "bfloat16", "send"), (wide, "uint8", "send"), (wide, "uint8", "recv"), (a, "int8", "recv")):
        with pytest.raises(ValueError, match="Unsupported dtype"):
            worker.collective_transfer_kv(None, 0, [0], (1,), dtype, mode)


@pytest.mark.parametrize("layout", ["nhd", "hnd"])
def test_4_bit_blocks_swap_in_both_layouts(layout):
    w = _worker(layout, cpu=4)
    w.write_kv_blocks([2, 3], _blocks(2, 5))
    before = w.extract_kv_blocks([2, 3]).clone()
    w.swap_blocks(["r"], [2, 3], [1, 0], is_swap_in=False)
    w.wait_for_all_swap_out()
    w.write_kv_blocks([2, 3], _blocks(2, 6))
    w.swap_blocks(["r"], [0, 1], [8, 9], is_swap_in=True)
    w.wait_for_all_swap_in()
    assert torch.equal(w.extract_kv_blocks([9, 8]), before)
