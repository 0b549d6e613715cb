"""The 4-bit cache through the worker: configuration, hand-over from a 16-bit worker, decode with eviction, swap."""
import numpy as np
import pytest
import torch

from elasticmm_b200 import KVPoolQ4
from elasticmm_b200.engine.v0 import Request, V0BlockManager, V0KVCacheConfig, V0Worker
from oracle import q4_oracle

pytestmark = pytest.mark.gpu

L, NB, BS, H, D = 2, 24, 16, 4, 128


def _worker(layout="nhd", cpu=0):
    c = V0KVCacheConfig(block_size=BS, max_num_gpu_blocks=NB, max_num_cpu_blocks=cpu, dtype="bfloat16", num_layers=L,
                        num_kv_heads=H, head_size=D, layout=layout, kv_bits=4)
    w = V0Worker.from_config(c, device="cuda:0")
    assert isinstance(w.pool, KVPoolQ4) and w.pool.block_bytes() == c.block_bytes
    return w


def _rows(x):
    f = x.float().cpu().numpy()
    return q4_oracle.encode_rows(f.reshape(-1, D)).reshape(*f.shape[:-1], -1)


@pytest.mark.parametrize("layout", ["nhd", "hnd"])
@pytest.mark.parametrize("source", ["nhd", "hnd"])
def test_blocks_of_a_16_bit_worker_enter_a_4_bit_one(layout, source):
    wide = V0Worker(dtype="bfloat16", device="cuda:0", block_size=BS)
    wide.init_kvcache(NB, L, H, D, layout=source)
    for t in wide.kv_cache:
        t.normal_()
    w = _worker(layout)
    src, dst = [5, 0, 23, 7], [1, 22, 3, 9]
    data = wide.extract_kv_blocks(src)
    w.write_kv_blocks(dst, data)
    want = _rows(data)
    packed = w.extract_kv_blocks(dst)  # the rows' bytes
    assert packed.dtype == torch.uint8 and (packed.cpu().numpy() == want).all()
    back = w.read_kv_blocks(dst)
    o, v = q4_oracle.decode_parts(want, D)
    assert back.shape == data.shape
    assert torch.equal(back.cpu(), torch.from_numpy(o.astype(np.float32) + v.astype(np.float32)).to(torch.bfloat16))
    other = _worker(layout)
    other.write_kv_blocks([4, 5, 6, 7], packed)  # bytes move as they are
    assert torch.equal(other.read_kv_blocks([4, 5, 6, 7]), back)
    layout_info = w.get_kv_cache_layout()
    assert layout_info["kv_bits"] == 4 and layout_info["head_dim"] == D
    with pytest.raises(ValueError):
        w.write_kv_blocks(dst, data[..., :64])
    with pytest.raises(Exception):
        w.write_kv_blocks([1, 1, 2, 3], data)
    with pytest.raises(RuntimeError):
        wide.read_kv_blocks(src)
    with pytest.raises(RuntimeError):
        wide.attend(0, None, None, None)
    with pytest.raises(ValueError, match="kv_bits"):
        V0Worker(kv_bits=8)


def test_swap_and_scores_move_with_blocks():
    w = _worker(cpu=4)
    w.write_kv_blocks([2, 3], torch.randn(L, 2, 2, BS, H, D, dtype=torch.bfloat16, device="cuda"))
    before = w.extract_kv_blocks([2, 3]).clone()
    w.swap_blocks(["r"], [2, 3], [0, 1], is_swap_in=False)
    w.wait_for_all_swap_out()
    w.swap_blocks(["r"], [0, 1], [8, 9], is_swap_in=True)
    w.wait_for_all_swap_in()
    assert torch.equal(w.extract_kv_blocks([8, 9]), before)
    s = w.init_scores()
    s.layers[1][2] = 3.0
    moved = s.gather([2])
    s.scatter([8], moved)
    assert (s.layers[1][8] == 3.0).all()


def test_weights_follow_a_compaction():
    w = _worker()
    w.write_kv_blocks([6, 7], torch.randn(L, 2, 2, BS, H, D, dtype=torch.bfloat16, device="cuda"))
    before = w.extract_kv_blocks([6, 7]).clone()
    s = w.init_scores()
    for layer in s.layers:
        layer[6], layer[7] = 6.0, 7.0
    assert w.compact_blocks([6, 7], [0, 1])["blocks"] == 2
    assert torch.equal(w.extract_kv_blocks([0, 1]), before)
    for layer in s.layers:
        assert (layer[0] == 6.0).all() and (layer[1] == 7.0).all()


def test_decode_evict_and_free():
    """Requests decode, are cut back, give blocks back, and decode on in what they kept."""
    w = _worker()
    w.init_scores()
    bm = V0BlockManager("decoding", NB, 0, BS)
    lens, keep = {"a": 90, "b": 40}, 48
    for rid, n in lens.items():
        bm.allocate_blocks(Request.of_length(rid, n + 1))
    g = torch.Generator().manual_seed(4)

    def tables():
        width = max(len(bm.get_block_table(r)) for r in lens)
        return torch.tensor([bm.get_block_table(r) + [0] * (width - len(bm.get_block_table(r))) for r in lens],
                            dtype=torch.int32, device="cuda")

    slots = torch.tensor([s for r, n in lens.items() for s in bm.get_slot_mapping(r, range(n))], device="cuda")
    kv = [torch.randn(L, slots.numel(), H, D, generator=g).to(torch.bfloat16).cuda() for _ in range(2)]
    w.reset_scores(slots)
    w.reshape_and_cache_all_layers(*kv, slots)

    def step(cur):
        new = torch.tensor([bm.get_slot_mapping(r, [n])[0] for r, n in zip(lens, cur)], device="cuda")
        kv = [torch.randn(L, 2, H, D, generator=g).to(torch.bfloat16).cuda() for _ in range(2)]
        w.reset_scores(new)
        w.reshape_and_cache_all_layers(*kv, new)
        cur = [n + 1 for n in cur]
        l_d, t = torch.tensor(cur, dtype=torch.int32, device="cuda"), tables()
        for l in range(L):
            q = torch.randn(2, 2 * H, D, generator=g).to(torch.bfloat16)
            out = w.attend(l, q.cuda(), t, l_d).double().cpu().numpy()
            pool = w.kv_cache[l].cpu().numpy()
            want, _, _, _ = q4_oracle.attend(pool, D, q.double().numpy(), t.cpu().numpy(), cur, D ** -0.5)
            # relative error of a bf16 rounding, 2^-8 at most, and as much again for the weights
            assert np.linalg.norm(out - want) <= 2 * 2.0 ** -8 * np.linalg.norm(want)
        return cur, t, l_d

    cur, t, l_d = step(list(lens.values()))
    weights = np.stack([x.cpu().numpy() for x in w.scores.layers])
    before = np.stack([x.cpu().numpy() for x in w.kv_cache])
    res = w.evict_tokens(t, l_d, keep, recent=8, sink=4)
    want = q4_oracle.select_tokens(weights, t.cpu().numpy(), cur, keep, 8, 4)
    assert (res["index"].cpu().numpy() == want).all() and res["seq_lens"].tolist() == [48, 41]
    q4_oracle.keep_tokens(before, want, t.cpu().numpy(), cur, keep)
    assert (np.stack([x.cpu().numpy() for x in w.kv_cache]) == before).all()
    cur = res["seq_lens"].tolist()
    free = bm.get_num_avail_gpu_blocks()
    assert len(bm.truncate_blocks("a", cur[0])) == 3 and bm.get_num_avail_gpu_blocks() == free + 3
    for r, n in zip(lens, cur):
        bm.expand_blocks_for_seq_len(r, n + 1)
    cur, _, _ = step(cur)
    assert cur == [49, 42]
    assert "error" in w.evict_tokens(tables(), torch.tensor(cur, dtype=torch.int32, device="cuda"), 8, recent=9)
    w.ctx.check_status()


def test_blocks_move_between_4_bit_workers():
    a, b = _worker(), _worker()
    a.write_kv_blocks(list(range(6)), torch.randn(L, 2, 6, BS, H, D, dtype=torch.bfloat16, device="cuda"))
    plan = a.extract_kv_blocks([1, 4])
    b.write_kv_blocks([10, 11], plan)
    assert torch.equal(b.extract_kv_blocks([10, 11]), plan)
    a.pool.copy_blocks(b.pool, [0, 5], [2, 3])
    assert torch.equal(b.extract_kv_blocks([2, 3]), a.extract_kv_blocks([0, 5]))
