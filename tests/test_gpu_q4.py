"""The 4-bit cache, its decode attention and token eviction against the 64-bit restatement.

Tolerances, per output value, with h = finfo(dtype).eps / 2 the half step of the output type:

  attention  h |ref| for the final rounding, plus bound = sum_t p_t (|o| + |s (c - 8)| + s c) times
             2^-11: out = sum p s c + sum p (o - 8 s). A weight p rounded to 16 bits, p (1 + d) with |d| <= 2^-11, is the
             same in both sums and adds at most 2^-11 p |o + s (c - 8)|; the product p s, rounded once more, enters the
             first sum only and adds at most 2^-11 p s c; plus bound times
             2 * 2^-17 * spread: a logit is a sum of at most 2^7 + 2^1 terms in 32 bits, so it is off by at most 2^-17 of
             the sum of their absolute values (spread), a weight by that share, and its sum by the same once more;
             plus 2^-24, the smallest step of an fp16 result.
  weights    the share 2 * 2^-17 * spread + 2^-20 (exp2 and the division) of the weight, plus 2^-23 of the sum it joins.
  rows       equal byte for byte; what is read back is the decoded value in 32 bits, rounded once.
"""
import numpy as np
import pytest
import torch

from elasticmm_b200 import KVPool, KVPoolQ4, ScorePool, _lib, get_context
from gpu_util import assert_clean, configure
from oracle import q4_oracle

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


@pytest.fixture()
def ctx():
    c = get_context(0)
    configure(c)
    return c


def new_layers(L, NB, BS, H, D, hnd, fill=0):
    row = KVPoolQ4.row_bytes(D)
    if hnd:
        return [torch.full((2, NB, H, BS, row), fill, dtype=torch.uint8, device="cuda").permute(0, 1, 3, 2, 4) for _ in range(L)]
    return [torch.full((2, NB, BS, H, row), fill, dtype=torch.uint8, device="cuda") for _ in range(L)]


def rows_of(x):
    """16-bit tensor [..., D] -> bytes by the restatement."""
    f = x.float().numpy()
    return q4_oracle.encode_rows(f.reshape(-1, f.shape[-1])).reshape(*f.shape[:-1], -1)


def random_pool(L, NB, BS, H, D, hnd, seed, gain=1.0, shift=0.3):
    """(KVPoolQ4, its bytes [L, 2, NB, BS, H, row]) of normal values."""
    rng = np.random.default_rng(seed)
    bytes_ = np.stack([np.stack([
        q4_oracle.encode_rows((rng.standard_normal((NB * BS * H, D)) * gain + shift * p).astype(np.float16).astype(np.float32))
        .reshape(NB, BS, H, -1) for p in (1, 0)]) for _ in range(L)])
    layers = new_layers(L, NB, BS, H, D, hnd)
    for t, b in zip(layers, bytes_):
        t.copy_(torch.from_numpy(b))
    return KVPoolQ4(layers, D), bytes_


def tables_for(lens, NB, BS, seed, extra=0):
    """Disjoint shuffled tables; the entries behind a sequence are far outside the pool."""
    need = [-(-n // BS) for n in lens]
    assert sum(need) <= NB
    ids = np.random.default_rng(seed).permutation(NB)
    width = max([1, *need]) + extra
    t = np.full((len(lens), width), 1 << 30, dtype=np.int32)
    at = 0
    for b, k in enumerate(need):
        t[b, :k] = ids[at:at + k]
        at += k
    return t


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def check_out(got, ref, bound, spread, dtype, what=""):
    h = torch.finfo(dtype).eps / 2
    tol = h * np.abs(ref) + bound * (2.0 ** -11 + 2 * 2.0 ** -17 * spread[..., None]) + 2.0 ** -24
    err = np.abs(got.double().cpu().numpy() - ref)
    assert (err <= tol).all(), f"{what}: {np.max(err / tol)} of the tolerance at {np.unravel_index(np.argmax(err / tol), err.shape)}"


def check_scores(got, before, tables, lens, weights, spread, group):
    """All of [NB, H, BS]: the sequences' entries within their tolerance, the others untouched."""
    got, want = got.double().cpu().numpy(), before.astype(np.float64).copy()
    tol = np.zeros_like(want)
    NB, H, BS = want.shape
    for b, n in enumerate(lens):
        for t in range(n):
            blk, off = tables[b][t // BS], t % BS
            w = weights[b][:, t]
            want[blk, :, off] += w
            share = 2 * 2.0 ** -17 * spread[b].reshape(H, group).max(-1) + 2.0 ** -20
            tol[blk, :, off] = w * share + 2.0 ** -23 * np.abs(want[blk, :, off]) + 2.0 ** -40
    err = np.abs(got - want)
    assert (err <= tol).all(), f"weights off by {np.max(err - tol)}"


# ------------------------------------------------------------------------------------------------------ append / read
@pytest.mark.parametrize("D,H,BS,dtype,hnd", [
    (128, 4, 16, BF, False), (128, 3, 5, FP, True), (64, 8, 16, FP, False), (64, 1, 1, BF, True), (256, 2, 16, BF, True),
    (256, 5, 7, FP, False)])
@pytest.mark.parametrize("T", [1, 37])
def test_append_and_read(ctx, D, H, BS, dtype, hnd, T):
    L, NB = 3, -(-40 // BS)
    g = torch.Generator().manual_seed(D + T)
    key, value = torch.randn(L, T, H, D, generator=g).to(dtype), (torch.randn(L, T, H, D, generator=g) * 5 + 1).to(dtype)
    slots = torch.randperm(NB * BS, generator=g)[:T].clone()
    if T > 1:
        slots[3] = -1
    want = np.full((L, 2, NB * BS, H, q4_oracle.row_bytes(D)), 0xA5, dtype=np.uint8)
    ok = (slots >= 0).numpy()
    for l in range(L):
        for p, x in enumerate((key[l], value[l])):
            want[l, p, slots.numpy()[ok]] = rows_of(x)[ok]
    k_d, v_d, s_d = key.cuda(), value.cuda(), slots.cuda()

    def bytes_of(pool):
        return np.stack([t.contiguous().cpu().numpy().reshape(2, NB * BS, H, -1) for t in pool.layers])

    one, all_, bound = (KVPoolQ4(new_layers(L, NB, BS, H, D, hnd, 0xA5), D, ctx) for _ in range(3))
    for l in range(L):
        one.append(l, k_d[l], v_d[l], s_d)
    before = ctx.launch_count
    all_.append_all_layers(k_d, v_d, s_d)
    assert ctx.launch_count == before + 1
    b = bound.bind_append(k_d, v_d, s_d)
    for l in range(L):
        b(l)
    for pool in (one, all_, bound):
        assert (bytes_of(pool) == want).all()
    rk, rv = all_.read(s_d, dtype)
    for p, got in ((0, rk), (1, rv)):
        o, v = q4_oracle.decode_parts(want[:, p][:, slots.clamp(min=0).numpy()], D)
        ref = torch.from_numpy((o.astype(np.float32) + v.astype(np.float32))).to(dtype)
        ref[:, ~torch.from_numpy(ok)] = 0
        assert torch.equal(got.cpu(), ref)
    part = all_.read(s_d, dtype, 1, 2)
    assert torch.equal(part[0], rk[1:]) and torch.equal(part[1], rv[1:])
    other = FP if dtype == BF else BF
    assert all_.read(s_d, other)[0].dtype == other
    assert all_.read(s_d[:0], dtype)[0].shape == (L, 0, H, D)
    assert_clean(ctx)


def test_append_extreme_groups(ctx):
    """Constant, tiny, huge, infinite and NaN groups, and both zeros."""
    D, H = 128, 2
    x = torch.zeros(6, H, D)
    x[0] = 3.0
    x[1, 0, :32] = torch.linspace(0, 2.0 ** -22, 32)
    x[2, 1] = torch.linspace(-65504, 65504, D)
    x[3, 0, 5], x[3, 1, 77] = float("inf"), float("-inf")
    x[4, 0, 33], x[4, 1, 127] = float("nan"), float("nan")
    x[5] = -0.0
    for dtype in (FP, BF):
        key = x.to(dtype)
        pool = KVPoolQ4(new_layers(1, 1, 16, H, D, False), D, ctx)
        slots = torch.arange(6, device="cuda")
        pool.append(0, key.cuda(), key.cuda(), slots)
        want = rows_of(key)
        got = pool.layers[0][:, 0, :6].cpu().numpy()
        assert (got[0] == want).all() and (got[1] == want).all()
        k, _ = pool.read(slots, dtype)
        assert torch.isnan(k[0, 4, 0, 32:64]).all() and torch.isfinite(k[0, 4, 0, :32]).all()
        assert torch.isfinite(k[0, 3]).all() and (k[0, 0] == 3.0).all() and (k[0, 5] == 0).all()
    # larger than fp16 can hold: clamped
    big = torch.full((1, H, D), 1e30, dtype=BF, device="cuda")
    pool.append(0, big, -big, slots[:1])
    k, v = pool.read(slots[:1], BF)
    assert (k == torch.tensor(65504.0, dtype=BF)).all() and (v == -torch.tensor(65504.0, dtype=BF)).all()
    assert_clean(ctx)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_append_quotients_near_a_half_and_out_of_range(ctx, D, dtype):
    """Groups whose quotients fall on or next to halves, groups far from zero (the offset's rounding shifts the codes out
    of their range), tiny and subnormal groups, and many random ones: every byte as the definition has it."""
    H, T = 2, 600
    g = torch.Generator().manual_seed(D)
    x = torch.randn(T, H, D, generator=g)
    x[100:200] = torch.randint(0, 31, (100, H, D), generator=g).float() / 2  # steps of a half
    x[200:300] = x[200:300] * 0.01 + torch.randn(100, H, 1, generator=g) * 30
    x[300:350] = x[300:350] * 2.0 ** -22
    x[350:400] = x[350:400] * 1e4
    x[400:450, :, ::2] = 1000.0
    x[450:500] = torch.randint(-8, 8, (50, H, D), generator=g).float() + 0.5 + 2.0 ** -7 * torch.randint(-1, 2, (50, H, D), generator=g)
    key, value = x.to(dtype), (x * 0.37).to(dtype)
    pool = KVPoolQ4(new_layers(1, -(-T // 16), 16, H, D, False), D, ctx)
    pool.append(0, key.cuda(), value.cuda(), torch.arange(T, device="cuda"))
    got = pool.layers[0].cpu().numpy().reshape(2, -1, H, KVPoolQ4.row_bytes(D))[:, :T]
    assert (got[0] == rows_of(key)).all() and (got[1] == rows_of(value)).all()
    assert_clean(ctx)


def test_append_strided_rows_and_packed_blocks(ctx):
    """Slices of a fused projection at an odd offset, and the packed blocks of a 16-bit pool."""
    D, H, T, L, BS = 64, 3, 11, 2, 4
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(L, T, 1 + 2 * H * D + 5, generator=g).to(BF)
    k, v = qkv[:, :, 1:1 + H * D].unflatten(-1, (H, D)), qkv[:, :, 1 + H * D:1 + 2 * H * D].unflatten(-1, (H, D))
    d = qkv.cuda()
    kd, vd = d[:, :, 1:1 + H * D].unflatten(-1, (H, D)), d[:, :, 1 + H * D:1 + 2 * H * D].unflatten(-1, (H, D))
    pool = KVPoolQ4(new_layers(L, 4, BS, H, D, False), D, ctx)
    slots = torch.arange(T, device="cuda") + 2
    pool.append_all_layers(kd, vd, slots)
    for l in range(L):
        got = pool.layers[l].cpu().numpy().reshape(2, 16, H, -1)[:, 2:2 + T]
        assert (got[0] == rows_of(k[l])).all() and (got[1] == rows_of(v[l])).all()
    wide = KVPool([torch.randn(2, 6, BS, H, D, device="cuda").to(FP) for _ in range(L)], ctx)
    ids = [4, 0, 5]
    packed = wide.gather(ids)  # [L, 2, n, BS, H, D]
    slots = torch.tensor([i * BS + t for i in (1, 3, 0) for t in range(BS)], device="cuda")
    pool.append_all_layers(packed[:, 0].flatten(1, 2), packed[:, 1].flatten(1, 2), slots)
    for l in range(L):
        got = pool.layers[l].cpu().numpy()
        for i, to in zip(ids, (1, 3, 0)):
            assert (got[:, to] == rows_of(wide.layers[l][:, i].cpu())).all()
    assert_clean(ctx)


def test_rows_refusals_and_bad_slots(ctx):
    D, H, BS, NB = 128, 2, 16, 3
    pool = KVPoolQ4(new_layers(2, NB, BS, H, D, False, 7), D, ctx)
    key = torch.ones(4, H, D, dtype=FP, device="cuda")
    slots = torch.tensor([5, NB * BS, -1, 1 << 40], device="cuda")
    pool.append(0, key, key, slots)
    rc, detail = ctx.status()
    assert rc == _lib.ERR_ID_RANGE and detail in (NB * BS, 1 << 40)
    got = pool.layers[0].cpu().numpy().reshape(2, NB * BS, H, -1)
    assert (got[:, 5] == rows_of(key[:1].cpu())[0]).all()
    assert (np.delete(got, 5, 1) == 7).all() and (pool.layers[1] == 7).all()
    k, v = pool.read(slots, FP, 0, 1)
    assert ctx.status()[0] == _lib.ERR_ID_RANGE
    assert (k[0, 0] == 1).all() and (k[0, 1:] == 0).all() and (v[0, 1:] == 0).all()
    for bad in (dict(key=key.float()), dict(key=key[:3]), dict(key=key.to(BF)), dict(slots=slots[:3]), dict(slots=slots.int()),
                dict(key=key.transpose(0, 1)), dict(key=key[..., :64]), dict(key=key.cpu())):
        args = {"key": key, "slots": slots, **bad}
        with pytest.raises(ValueError):
            pool.append(0, args["key"], key, args["slots"])
    with pytest.raises(_lib.EmmError):
        pool.append(2, key, key, slots)
    with pytest.raises(ValueError):
        pool.append_all_layers(key.expand(3, 4, H, D), key.expand(3, 4, H, D), slots)
    with pytest.raises(_lib.EmmError):  # layers that overlap
        pool.append_all_layers(key.expand(2, 4, H, D), key.expand(2, 4, H, D), slots)
    with pytest.raises(ValueError):
        pool.read(slots, torch.float32)
    with pytest.raises(ValueError):
        pool.read(slots, FP, 1, 2)
    bound = pool.bind_append(torch.ones(2, 4, H, D, dtype=FP, device="cuda"), torch.ones(2, 4, H, D, dtype=FP, device="cuda"), slots)
    with pytest.raises(_lib.EmmError):
        bound(2)
    assert bound.raw(-1, 0) == _lib.ERR_BAD_ARG
    odd = torch.zeros(2 * NB * BS * H * 80 + 8, dtype=torch.uint8, device="cuda")[8:].view(2, NB, BS, H, 80)
    with pytest.raises(ValueError, match="16-byte"):
        KVPoolQ4([odd], D, ctx)
    wrong = KVPool(new_layers(1, NB, BS, H, 64, False), ctx)  # an ordinary byte pool is no 4-bit pool of 128 channels
    rc = ctx._lib.emm_q4_append(wrong._h, D, 0, 0, 1, key.data_ptr(), key.data_ptr(), 0, 512, 0, 512, slots.data_ptr(), 4, 0)
    assert rc == _lib.ERR_BAD_ARG
    assert_clean(ctx)


# ----------------------------------------------------------------------------------------------------------- attention
LENS = [0, 1, 15, 16, 17, 33, 64, 255, 700]


@pytest.mark.parametrize("hnd", [False, True], ids=["nhd", "hnd"])
@pytest.mark.parametrize("D,H,group,BS,dtype", [
    (128, 4, 7, 16, BF), (128, 8, 8, 16, FP), (128, 3, 1, 16, FP), (64, 8, 4, 16, BF), (64, 5, 2, 8, FP), (256, 2, 3, 32, BF),
    (256, 1, 16, 16, FP), (128, 1, 64, 16, BF), (128, 2, 9, 5, BF), (64, 12, 1, 1, FP), (128, 9, 5, 48, FP),
    (128, 8, 2, 8, BF), (256, 2, 8, 8, FP), (128, 2, 4, 2, BF), (256, 1, 2, 1, BF), (128, 1, 8, 4, FP), (128, 4, 8, 64, BF)])
def test_attend(ctx, D, H, group, BS, dtype, hnd):
    NB = sum(-(-n // BS) for n in LENS) + 3
    pool, bytes_ = random_pool(2, NB, BS, H, D, hnd, D + H)
    tables = tables_for(LENS, NB, BS, 1)
    g = torch.Generator().manual_seed(group)
    q = (torch.randn(len(LENS), H * group, D, generator=g) * 1.5).to(dtype)
    lens = dev(np.array(LENS, dtype=np.int32))
    before = np.random.default_rng(2).random((2, NB, H, BS), dtype=np.float32)
    scores = ScorePool(list(dev(before).unbind(0)), ctx)
    plain = pool.attend(1, q.cuda(), dev(tables), lens)
    out = pool.attend(1, q.cuda(), dev(tables), lens, scores=scores)
    assert_clean(ctx)
    ref, weights, bound, spread = q4_oracle.attend(bytes_[1], D, q.double().numpy(), tables, LENS, D ** -0.5)
    check_out(plain, ref, bound, spread, dtype, "plain")
    check_out(out, ref, bound, spread, dtype, "with scores")
    assert (plain[0] == 0).all() and plain.dtype == dtype
    check_scores(scores.layers[1], before[1], tables, LENS, weights, spread, group)
    assert (scores.layers[0].cpu().numpy() == before[0]).all()


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 127, 128, 129, 1023, 4097, 20000])
@pytest.mark.parametrize("D,H,group,dtype", [(128, 8, 8, BF), (128, 2, 4, FP), (64, 1, 12, FP)])
def test_attend_one_sequence(ctx, n, D, H, group, dtype):
    """One sequence alone: the long axis is split over the whole GPU and joined."""
    BS = 16
    NB = -(-n // BS) + 1
    pool, bytes_ = random_pool(1, NB, BS, H, D, False, n)
    tables = tables_for([n], NB, BS, 3)
    q = torch.randn(1, H * group, D, generator=torch.Generator().manual_seed(n)).to(dtype)
    before = np.zeros((NB, H, BS), dtype=np.float32)
    scores = ScorePool([dev(before)], ctx)
    out = pool.attend(0, q.cuda(), dev(tables), dev(np.array([n], dtype=np.int32)), scores=scores)
    assert_clean(ctx)
    ref, weights, bound, spread = q4_oracle.attend(bytes_[0], D, q.double().numpy(), tables, [n], D ** -0.5)
    check_out(out, ref, bound, spread, dtype)
    check_scores(scores.layers[0], before, tables, [n], weights, spread, group)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_attend_extreme_values(ctx, dtype):
    """Large and small values and queries, one token that takes all the weight, a large scale; NaN stays in its row."""
    D, H, group, BS, n = 128, 2, 2, 16, 100
    NB = 16
    for gain, qgain, scale in ((200.0, 0.01, None), (1e-3, 3.0, None), (1.0, 40.0, None), (1.0, 1e-4, 50.0), (3000.0, 1e-4, None),
                               (1.0, 1.0, 0.0), (1.0, 1.0, -0.3)):
        pool, bytes_ = random_pool(1, NB, BS, H, D, False, 3, gain=gain)
        tables = tables_for([n, 3], NB, BS, 1)
        q = (torch.randn(2, H * group, D, generator=torch.Generator().manual_seed(1)) * qgain).to(dtype)
        out = pool.attend(0, q.cuda(), dev(tables), dev(np.array([n, 3], dtype=np.int32)), scale=scale)
        ref, _, bound, spread = q4_oracle.attend(bytes_[0], D, q.double().numpy(), tables, [n, 3], D ** -0.5 if scale is None else scale)
        check_out(out, ref, bound, spread, dtype, f"gain {gain} {qgain} {scale}")
    # a query of zeros is a mean; NaN in a query or in a cached row reaches the rows that use it and no others
    q = torch.zeros(2, H * group, D, dtype=dtype)
    q[1, 0, 5] = float("nan")
    out = pool.attend(0, q.cuda(), dev(tables), dev(np.array([n, 3], dtype=np.int32)))
    assert torch.isnan(out[1, 0]).all() and torch.isfinite(out[1, 1:]).all() and torch.isfinite(out[0]).all()
    bad = torch.zeros(1, H, D, dtype=dtype, device="cuda")
    bad[0, 1, 40] = float("nan")
    good = torch.zeros_like(bad)
    slot = torch.tensor([int(tables[0][2]) * BS + 4], device="cuda")  # position 36
    q = torch.randn(2, H * group, D, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    lens = dev(np.array([n, 3], dtype=np.int32))
    pool.append(0, good, bad, slot)  # a NaN among the values: its group of channels
    out = pool.attend(0, q, dev(tables), lens)
    nan = torch.isnan(out.cpu())
    assert nan[0, 2:, 32:64].all() and not nan[0, 2:, :32].any() and not nan[0, 2:, 64:].any()
    assert not nan[0, :2].any() and not nan[1].any()
    pool.append(0, bad, good, slot)  # among the keys: all channels
    out = pool.attend(0, q, dev(tables), lens)
    nan = torch.isnan(out.cpu())
    assert nan[0, 2:].all() and not nan[0, :2].any() and not nan[1].any()
    short = pool.attend(0, q, dev(tables), dev(np.array([36, 3], dtype=np.int32)))  # behind the end it does not count
    assert torch.isfinite(short).all()
    assert_clean(ctx)


def test_attend_ignores_what_lies_behind_the_end(ctx):
    """Rows of NaN and infinite scales behind a sequence's last token, in its last block and in no one's block."""
    D, H, group, BS = 128, 4, 2, 16
    lens = [5, 16, 50, 97]
    pool, bytes_ = random_pool(1, 32, BS, H, D, False, 9)
    tables = tables_for(lens, 32, BS, 4, extra=2)
    poisoned = np.full_like(bytes_, 0xFF)
    for b, n in enumerate(lens):
        for t in range(n):
            poisoned[0][:, tables[b][t // BS], t % BS] = bytes_[0][:, tables[b][t // BS], t % BS]
    q = torch.randn(4, H * group, D, generator=torch.Generator().manual_seed(3)).to(BF)
    want = pool.attend(0, q.cuda(), dev(tables), dev(np.array(lens, dtype=np.int32)))
    pool.layers[0].copy_(torch.from_numpy(poisoned[0]))
    got = pool.attend(0, q.cuda(), dev(tables), dev(np.array(lens, dtype=np.int32)))
    assert_clean(ctx)
    assert torch.equal(got, want)
    ref, _, bound, spread = q4_oracle.attend(bytes_[0], D, q.double().numpy(), tables, lens, D ** -0.5)
    check_out(got, ref, bound, spread, BF)


def test_attend_arguments(ctx):
    """Strided queries and outputs, in place, a scale, a bound on the lengths, an odd table view, an empty batch."""
    D, H, group, BS = 128, 2, 4, 16
    lens = [40, 7, 90]
    pool, bytes_ = random_pool(1, 16, BS, H, D, False, 4)
    tables = tables_for(lens, 16, BS, 4)
    heads = H * group
    fused = torch.randn(3, (heads + 2 * H) * D + 3, generator=torch.Generator().manual_seed(3)).to(BF).cuda()
    q = fused[:, :heads * D].unflatten(-1, (heads, D))
    lens_d, tables_d = dev(np.array(lens, dtype=np.int32)), dev(tables)
    wide = torch.zeros(3, tables.shape[1] + 5, dtype=torch.int32, device="cuda")
    wide[:, :tables.shape[1]] = tables_d
    ref, _, bound, spread = q4_oracle.attend(bytes_[0], D, q.double().cpu().numpy(), tables, lens, 0.2)
    out = torch.zeros(3, 2, heads, D, dtype=BF, device="cuda")
    got = pool.attend(0, q, wide[:, :tables.shape[1]], lens_d, scale=0.2, out=out[:, 1], max_len=90)
    assert got.data_ptr() == out[:, 1].data_ptr() and (out[:, 0] == 0).all()
    check_out(got, ref, bound, spread, BF)
    mine = q.contiguous().clone()
    assert pool.attend(0, mine, tables_d, lens_d, scale=0.2, out=mine) is mine
    assert torch.equal(mine, got)
    odd = torch.zeros(3 * heads * D + 1, dtype=BF, device="cuda")[1:].view(3, heads, D)  # 2-byte aligned only
    odd.copy_(q)
    assert torch.equal(pool.attend(0, odd, tables_d, lens_d, scale=0.2), got)
    assert pool.attend(0, q[:0], tables_d[:0], lens_d[:0]).shape == (0, heads, D)
    none = pool.attend(0, q, tables_d[:, :0], lens_d * 0)
    assert (none == 0).all()
    assert_clean(ctx)
    for bad in (dict(q=q.float()), dict(q=q[:, :7]), dict(q=q[..., :64]), dict(q=q[:2]), dict(t=tables_d.long()), dict(l=lens_d.long()),
                dict(q=q.transpose(0, 1)), dict(max_len=tables.shape[1] * BS + 1), dict(max_len=-1), dict(out=out[:2, 1]),
                dict(out=out[:, 1].float()), dict(q=q.cpu())):
        with pytest.raises(ValueError):
            pool.attend(0, bad.get("q", q), bad.get("t", tables_d), bad.get("l", lens_d), out=bad.get("out"), max_len=bad.get("max_len"))
    with pytest.raises(_lib.EmmError):
        pool.attend(1, q, tables_d, lens_d)
    with pytest.raises(_lib.EmmError):
        pool.attend(0, q, tables_d, lens_d, scale=float("nan"))
    with pytest.raises(_lib.EmmError):
        pool.attend(0, q, tables_d, lens_d, scale=1e39)  # infinite in 32 bits
    with pytest.raises(_lib.EmmError):
        pool.attend(0, q, tables_d, lens_d, scores=ScorePool([torch.zeros(15, H, BS, device="cuda")], ctx))
    many = torch.zeros(3, 65 * H, D, dtype=BF, device="cuda")
    with pytest.raises(ValueError, match="at most 64"):
        pool.attend(0, many, tables_d, lens_d)
    assert_clean(ctx)


def test_attend_reports_bad_lengths_and_blocks(ctx):
    D, H, group, BS = 128, 2, 2, 16
    pool, bytes_ = random_pool(1, 16, BS, H, D, False, 4)
    tables = tables_for([48, 48, 20], 16, BS, 4)
    q = torch.randn(3, H * group, D, generator=torch.Generator().manual_seed(3)).to(FP)
    lens = dev(np.array([-5, 1000, 20], dtype=np.int32))
    out = pool.attend(0, q.cuda(), dev(tables), lens)
    rc, detail = ctx.status()
    assert rc == _lib.ERR_LENGTH and detail in (-5, 1000)
    ref, _, bound, spread = q4_oracle.attend(bytes_[0], D, q.double().numpy(), tables, [0, 48, 20], D ** -0.5)
    check_out(out, ref, bound, spread, FP)
    broken = tables.copy()
    broken[1, 1] = 16  # positions 16..31 of sequence 1
    broken[2, 0], broken[2, 1] = -1, 1 << 30  # all of sequence 2
    scores = ScorePool([torch.zeros(16, H, BS, device="cuda")], ctx)
    out = pool.attend(0, q.cuda(), dev(broken), dev(np.array([48, 48, 20], dtype=np.int32)), scores=scores)
    rc, detail = ctx.status()
    assert rc == _lib.ERR_ID_RANGE and detail in (16, -1, 1 << 30)
    short = tables.copy()
    short[1, 1] = tables[1, 2]
    ref, weights, bound, spread = q4_oracle.attend(bytes_[0], D, q.double().numpy(), short, [48, 32, 0], D ** -0.5)
    check_out(out, ref, bound, spread, FP)
    check_scores(scores.layers[0], np.zeros((16, H, BS), dtype=np.float32), short, [48, 32, 0], weights, spread, group)
    assert (out[2] == 0).all()
    assert_clean(ctx)


@pytest.mark.parametrize("D,group,dtype", [(64, 8, FP), (128, 3, BF), (256, 4, BF), (256, 1, FP)])
def test_attend_one_head_long(ctx, D, group, dtype):
    """One KV head, and tokens for every SM: all warps of a block work on the same head."""
    BS, lens = 16, [40001, 5]
    NB = sum(-(-n // BS) for n in lens)
    pool, bytes_ = random_pool(1, NB, BS, 1, D, False, 6)
    tables = tables_for(lens, NB, BS, 4)
    q = torch.randn(2, group, D, generator=torch.Generator().manual_seed(3)).to(dtype)
    scores = ScorePool.like(pool)
    out = pool.attend(0, q.cuda(), dev(tables), dev(np.array(lens, dtype=np.int32)), scores=scores)
    assert_clean(ctx)
    ref, weights, bound, spread = q4_oracle.attend(bytes_[0], D, q.double().numpy(), tables, lens, D ** -0.5)
    check_out(out, ref, bound, spread, dtype)
    check_scores(scores.layers[0], np.zeros((NB, 1, BS), dtype=np.float32), tables, lens, weights, spread, group)
    scores.close()
    with pytest.raises(ValueError, match="closed"):
        pool.attend(0, q.cuda(), dev(tables), dev(np.array(lens, dtype=np.int32)), scores=scores)


def test_attend_logits_far_below_zero(ctx):
    """Logits of -1e31 and less: the largest still takes all the weight, and its row comes out rounded once."""
    D, H, BS, n = 128, 1, 16, 40
    rng = np.random.default_rng(5)
    x = rng.standard_normal((2, 4 * BS, H, D)).astype(np.float16).astype(np.float32)
    x[0, :, 0, :32] = 0
    x[0, :, 0, 0] = -4.0 - np.arange(4 * BS) % 7
    x[0, 29, 0, 0] = -2.0  # position 29; nowhere else above -4
    layer = np.stack([q4_oracle.encode_rows(p.reshape(-1, D)) for p in x]).reshape(2, 4, BS, H, -1)
    pool = KVPoolQ4([dev(layer)], D, ctx)
    tables = np.arange(4, dtype=np.int32)[None]
    q = torch.zeros(1, 2, D, dtype=BF)
    q[0, :, 0] = 1e32
    scores = ScorePool.like(pool)
    out = pool.attend(0, q.cuda(), dev(tables), dev(np.array([n], dtype=np.int32)), scores=scores)
    # one weight is 1 and the others are 0 exactly, so nothing but the product p s c and the result are rounded
    value = q4_oracle.decode_rows(layer[1].reshape(-1, layer.shape[-1]), D)[29]
    tol = 2.0 ** -9 * np.abs(value) + 2.0 ** -11 * 16 * 0.5
    assert (np.abs(out.double().cpu().numpy() - value) <= tol).all()
    want = torch.zeros(4, H, BS)
    want[1, 0, 13] = 2  # both query heads
    assert torch.equal(scores.layers[0].cpu(), want)
    assert_clean(ctx)


def test_attend_many_short_sequences_in_wide_tables(ctx):
    """More sequences than a block has threads, most of them empty, in tables for far longer ones (a padded batch)."""
    D, H, group, BS = 64, 2, 2, 16
    rng = np.random.default_rng(3)
    lens = np.where(rng.random(700) < 0.6, 0, rng.integers(1, 50, 700)).tolist()
    NB = sum(-(-n // BS) for n in lens)
    pool, bytes_ = random_pool(1, NB, BS, H, D, False, 4)
    tables = tables_for(lens, NB, BS, 4, extra=2000)
    q = torch.randn(700, H * group, D, generator=torch.Generator().manual_seed(3)).to(BF)
    before = rng.random((NB, H, BS), dtype=np.float32)
    scores = ScorePool([dev(before)], ctx)
    out = pool.attend(0, q.cuda(), dev(tables), dev(np.array(lens, dtype=np.int32)), scores=scores)
    assert_clean(ctx)
    ref, weights, bound, spread = q4_oracle.attend(bytes_[0], D, q.double().numpy(), tables, lens, D ** -0.5)
    check_out(out, ref, bound, spread, BF)
    check_scores(scores.layers[0], before, tables, lens, weights, spread, group)


@pytest.mark.parametrize("hnd", [False, True], ids=["nhd", "hnd"])
def test_offsets_past_32_bits(ctx, hnd):
    """Blocks that begin more than 2^32 bytes into their plane hold, read and move what the same blocks of a small pool do."""
    D, H, group, BS, n = 128, 8, 4, 16, 200
    k = -(-n // BS)
    NB = (5 << 30) // (BS * H * 80)
    g = torch.Generator().manual_seed(1)
    key, value = torch.randn(n, H, D, generator=g).to(BF).cuda(), torch.randn(n, H, D, generator=g).to(BF).cuda()
    q = torch.randn(1, H * group, D, generator=g).to(BF).cuda()
    lens = dev(np.array([n], dtype=np.int32))
    got = []
    for blocks, ids in ((k, np.arange(k)), (NB, np.concatenate([NB - 1 - np.arange(k - 2), [0, 1]]))):
        pool = KVPoolQ4([t for t in new_layers(1, blocks, BS, H, D, hnd)], D, ctx)
        scores = ScorePool.like(pool)
        tables = dev(ids[None].astype(np.int32))
        slots = (dev(ids)[:, None] * BS + torch.arange(BS, device="cuda")).flatten()[:n]
        pool.append(0, key, value, slots)
        rows = pool.read(slots, BF)
        out = pool.attend(0, q, tables, lens, scores=scores)
        index, _ = scores.select_tokens(tables, lens, 60, recent=5)
        pool.keep_tokens(index, tables, lens)
        kept = pool.read(slots[:60], BF)
        got.append([*rows, out, index, *kept])
        assert_clean(ctx)
        pool.close()
    for a, b in zip(*got):
        assert torch.equal(a, b)


# ----------------------------------------------------------------------------------------------------------- eviction
def score_values(shape, seed):
    """Weights with many ties, zeros of both signs, infinities and NaN."""
    rng = np.random.default_rng(seed)
    s = (rng.random(shape) ** 6).astype(np.float32)
    s[rng.random(shape) < 0.3] = 0.25
    s[rng.random(shape) < 0.1] = 0.0
    s[rng.random(shape) < 0.05] = -0.0
    s[rng.random(shape) < 0.02] = np.nan
    s[rng.random(shape) < 0.01] = np.inf
    s[rng.random(shape) < 0.01] = -3.5
    return s


@pytest.mark.parametrize("kind", ["bf16-nhd", "bf16-hnd", "q4-nhd", "q4-hnd", "odd"])
@pytest.mark.parametrize("keep,recent,sink", [(64, 10, 3), (1, 0, 0), (1, 1, 0), (200, 100, 100), (257, 0, 4), (5000, 3, 0), (16, 16, 0)])
def test_select_and_keep(ctx, kind, keep, recent, sink):
    L, H, BS = 2, 3, 16
    lens = [0, 1, 63, 64, 65, 257, 258, 300, 1111]
    NB = sum(-(-n // BS) for n in lens) + 4
    rng = np.random.default_rng(keep)
    if kind.startswith("q4"):
        pool, ref = random_pool(L, NB, BS, H, 128, kind.endswith("hnd"), 5)
    else:
        D, dt = (5, FP) if kind == "odd" else (64, BF)
        ref = rng.integers(0, 1 << 15, (L, 2, NB, BS, H, D)).astype(np.int16)
        if kind == "bf16-hnd":
            layers = [dev(x.swapaxes(2, 3)).view(dt).permute(0, 1, 3, 2, 4) for x in ref]
        else:
            layers = [dev(x).view(dt) for x in ref]
        pool = KVPool(layers, ctx)
    values = score_values((L, NB, H, BS), keep)
    scores = ScorePool(list(dev(values).unbind(0)), ctx)
    tables = tables_for(lens, NB, BS, 6, extra=1)
    t_d, l_d = dev(tables), dev(np.array(lens, dtype=np.int32))
    index, new_lens = scores.select_tokens(t_d, l_d, keep, recent=recent, sink=sink)
    want = q4_oracle.select_tokens(values, tables, lens, keep, recent, sink)
    assert (index.cpu().numpy() == want).all()
    assert new_lens.tolist() == [min(n, keep) for n in lens]
    for l in range(L):
        assert np.array_equal(scores.layers[l].cpu().numpy(), values[l], equal_nan=True)
    pool.keep_tokens(index, t_d, l_d)
    scores.keep_tokens(index, t_d, l_d)
    assert_clean(ctx)
    ref = ref.copy()
    q4_oracle.keep_tokens(ref, want, tables, lens, keep)
    for l in range(L):
        got = pool.layers[l].contiguous()
        assert (got.view(torch.int16 if ref.dtype == np.int16 else torch.uint8).cpu().numpy() == ref[l]).all()
    moved = values[:, None].swapaxes(3, 4)[..., None].copy()  # [L, 1, NB, BS, H, 1]
    q4_oracle.keep_tokens(moved, want, tables, lens, keep)
    for l in range(L):
        assert np.array_equal(scores.layers[l].cpu().numpy(), moved[l, 0, ..., 0].swapaxes(1, 2), equal_nan=True)


@pytest.mark.parametrize("n", [40000, 70001])
def test_select_and_keep_long(ctx, n):
    L, H, BS, keep = 1, 2, 32, n // 2
    NB = -(-n // BS)
    values = score_values((L, NB, H, BS), n)
    rows = np.random.default_rng(1).integers(0, 1 << 15, (L, 2, NB, BS, H, 8)).astype(np.int16)
    pool, scores = KVPool([dev(rows[0]).view(BF)], ctx), ScorePool([dev(values[0])], ctx)
    tables = tables_for([n], NB, BS, 6)
    t_d, l_d = dev(tables), dev(np.array([n], dtype=np.int32))
    index, _ = scores.select_tokens(t_d, l_d, keep, recent=100, sink=4)
    want = q4_oracle.select_tokens(values, tables, [n], keep, 100, 4)
    assert (index.cpu().numpy() == want).all()
    pool.keep_tokens(index, t_d, l_d)
    q4_oracle.keep_tokens(rows, want, tables, [n], keep)
    assert (pool.layers[0].view(torch.int16).cpu().numpy() == rows[0]).all()
    assert_clean(ctx)


def test_eviction_refusals_and_reports(ctx):
    L, NB, H, BS = 1, 8, 2, 16
    scores = ScorePool([torch.rand(NB, H, BS, device="cuda")], ctx)
    pool = KVPool([torch.zeros(2, NB, BS, H, 64, dtype=BF, device="cuda")], ctx)
    tables, lens = dev(tables_for([40, 20], NB, BS, 1)), dev(np.array([40, 20], dtype=np.int32))
    for keep, recent, sink in ((0, 0, 0), (-1, 0, 0), (8, 9, 0), (8, 4, 5), (8, -1, 0), (8, 0, -1), (2 ** 32 + 8, 0, 0), (8, 2 ** 32, 0)):
        with pytest.raises((ValueError, _lib.EmmError)):
            scores.select_tokens(tables, lens, keep, recent=recent, sink=sink)
    index, _ = scores.select_tokens(tables, lens, 8)
    for bad in (index.long(), index[..., ::2], index[:, :1], index[:, :, :1], index.cpu()):
        with pytest.raises(ValueError):
            pool.keep_tokens(bad, tables, lens)
    blocks = KVPool([torch.zeros(NB, H, 40, dtype=torch.float16, device="cuda")], ctx)
    with pytest.raises(_lib.EmmError):  # a block pool of another kind has no tokens
        blocks.keep_tokens(index, tables, lens)
    assert scores.select_tokens(tables[:0], lens[:0], 8)[0].shape == (1, 0, H, 8)
    # lengths and blocks outside are recorded; nothing outside the pool is read or written
    before = pool.layers[0].clone().normal_()
    pool.layers[0].copy_(before)
    _, new = scores.select_tokens(tables, dev(np.array([-1, 500], dtype=np.int32)), 8)
    assert ctx.status()[0] == _lib.ERR_LENGTH and new.tolist() == [0, 0]
    pool.keep_tokens(index, tables, dev(np.array([-1, 500], dtype=np.int32)))
    assert ctx.status()[0] == _lib.ERR_LENGTH
    assert torch.equal(pool.layers[0], before)
    broken = tables.clone()
    broken[0, 1] = NB
    scores.select_tokens(broken, lens, 8)
    assert ctx.status() == (_lib.ERR_ID_RANGE, NB)
    wild = torch.full_like(index, 1 << 30)
    wild[..., 1] = -7
    pool.keep_tokens(wild, tables, lens)  # positions outside the sequence are skipped
    assert_clean(ctx)
    assert torch.equal(pool.layers[0], before)
    scores.layers[0].fill_(1.0)
    scores.reset(torch.tensor([3, -1, NB * BS - 1], device="cuda"))
    want = torch.ones(NB, H, BS)
    want[0, :, 3] = want[NB - 1, :, BS - 1] = 0
    assert torch.equal(scores.layers[0].cpu(), want)
    scores.reset(torch.tensor([NB * BS], device="cuda"))
    assert ctx.status() == (_lib.ERR_ID_RANGE, NB * BS)
    with pytest.raises(ValueError):
        scores.reset(torch.tensor([3], dtype=torch.int32, device="cuda"))
    assert_clean(ctx)


# ------------------------------------------------------------------------------------------------------- all together
@pytest.mark.parametrize("hnd", [False, True], ids=["nhd", "hnd"])
def test_decode_with_eviction(ctx, hnd):
    """A prompt enters the cache, tokens are decoded with weights gathered, the cache is cut, its blocks move, decoding
    goes on: every step against the restatement on the same state."""
    L, H, group, D, BS, dtype = 2, 4, 2, 128, 16, BF
    lens = [70, 33, 130]
    B, NB, keep, recent, sink = len(lens), 48, 48, 8, 2
    room = 16
    tables = tables_for([n + room for n in lens], NB, BS, 8)
    t_d = dev(tables)
    pool = KVPoolQ4(new_layers(L, NB, BS, H, D, hnd), D, ctx)
    scores = ScorePool.like(pool)
    state = np.zeros((L, 2, NB, BS, H, 80), dtype=np.uint8)
    weight = np.zeros((L, NB, H, BS))
    g = torch.Generator().manual_seed(1)

    def slot(b, t):
        return int(tables[b][t // BS]) * BS + t % BS

    def put(key, value, slots):
        for l in range(L):
            for p, x in enumerate((key[l], value[l])):
                state[l, p].reshape(NB * BS, H, -1)[slots] = rows_of(x)

    prompt = [slot(b, t) for b, n in enumerate(lens) for t in range(n)]
    key, value = (torch.randn(L, len(prompt), H, D, generator=g).to(dtype) for _ in range(2))
    scores.layers[0].fill_(7.0)  # left by an earlier request
    scores.reset(torch.arange(NB * BS, device="cuda"))
    pool.append_all_layers(key.cuda(), value.cuda(), torch.tensor(prompt, device="cuda"))
    put(key, value, prompt)

    def decode(steps, cur, tabs):
        for _ in range(steps):
            new = [int(tabs[b][cur[b] // BS]) * BS + cur[b] % BS for b in range(B)]
            s_d = torch.tensor(new, device="cuda")
            scores.reset(s_d)
            cur = [n + 1 for n in cur]
            l_d = dev(np.array(cur, dtype=np.int32))
            key, value = (torch.randn(L, B, H, D, generator=g).to(dtype) for _ in range(2))
            put(key, value, new)
            for l in range(L):
                for b in range(B):
                    weight[l, new[b] // BS, :, new[b] % BS] = 0
                q = torch.randn(B, H * group, D, generator=g).to(dtype)
                active.append(l, key[l].cuda(), value[l].cuda(), s_d)
                out = active.attend(l, q.cuda(), dev(tabs), l_d, scores=scores)
                ref, w, bound, spread = q4_oracle.attend(state[l], D, q.double().numpy(), tabs, cur, D ** -0.5)
                check_out(out, ref, bound, spread, dtype)
                for b in range(B):
                    for t in range(cur[b]):
                        weight[l, tabs[b][t // BS], :, t % BS] += w[b][:, t]
                got = scores.layers[l].double().cpu().numpy()
                assert np.abs(got - weight[l]).max() < 1e-4 * weight[l].max()
                weight[l] = got  # the same starting point for the next step
        return cur

    active = pool
    cur = decode(3, lens, tables)
    l_d = dev(np.array(cur, dtype=np.int32))
    index, new_lens = scores.select_tokens(t_d, l_d, keep, recent=recent, sink=sink)
    want = q4_oracle.select_tokens(weight.astype(np.float32), tables, cur, keep, recent, sink)
    assert (index.cpu().numpy() == want).all()
    pool.keep_tokens(index, t_d, l_d)
    scores.keep_tokens(index, t_d, l_d)
    q4_oracle.keep_tokens(state, want, tables, cur, keep)
    view = weight[:, None].swapaxes(3, 4)[..., None]
    q4_oracle.keep_tokens(view, want, tables, cur, keep)
    for l in range(L):
        assert (pool.layers[l].cpu().numpy() == state[l]).all()
        assert (scores.layers[l].double().cpu().numpy() == weight[l]).all()
    cur = new_lens.tolist()
    assert cur == [48, 36, 48]
    # the requests' blocks move to another pool, as on a migration, weights along
    other = KVPoolQ4(new_layers(L, NB, BS, H, D, hnd), D, ctx)
    moved_scores = ScorePool.like(other)
    live = [int(i) for b in range(B) for i in tables[b][: -(-(cur[b] + 4) // BS)]]
    to = [(i * 7 + 3) % NB for i in live]
    assert len(set(to)) == len(to)
    other.scatter(to, pool.gather(live))
    scores.copy_blocks(moved_scores, live, to)
    remap = dict(zip(live, to))
    tables2 = np.array([[remap.get(int(i), 1 << 30) for i in row] for row in tables], dtype=np.int32)
    fresh, fresh_w = np.zeros_like(state), np.zeros_like(weight)
    fresh[:, :, to], fresh_w[:, to] = state[:, :, live], weight[:, live]
    state[:], weight[:] = fresh, fresh_w
    active, scores = other, moved_scores
    decode(3, cur, tables2)
    assert_clean(ctx)


def test_calls_replay_from_a_graph_and_run_on_other_streams(ctx):
    """A captured decode step replays on new lengths and queries; two graphs and an eager call do not share scratch."""
    L, H, group, D, BS = 1, 4, 4, 128, 16
    lens = [300, 80]
    pool, _ = random_pool(L, 40, BS, H, D, False, 4)
    tables = dev(tables_for([512, 96], 40, BS, 4))
    lens_d = dev(np.array(lens, dtype=np.int32))
    q = [torch.randn(2, H * group, D, device="cuda", dtype=FP) for _ in range(2)]
    scores = [ScorePool.like(pool) for _ in range(2)]
    key = torch.randn(2, H, D, device="cuda", dtype=FP)
    slots = torch.tensor([int(tables[0, 20]) * BS, int(tables[1, 5]) * BS], device="cuda")

    def step(i):
        pool.append(0, key, key, slots)
        out = pool.attend(0, q[i], tables, lens_d, scores=scores[i])
        index, left = scores[i].select_tokens(tables, lens_d, 64, recent=4)
        return out, index, left

    eager = [step(i) for i in range(2)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(2):
            step(i)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(i))
        graphs.append(graph)
    for s in scores:
        s.layers[0].zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(2):  # side by side
        with torch.cuda.stream(streams[i]):
            graphs[i].replay()
    torch.cuda.synchronize()
    for i in range(2):
        for a, b in zip(outs[i], eager[i]):
            assert torch.equal(a, b)
    lens_d.copy_(dev(np.array([512, 1], dtype=np.int32)))
    q[0].normal_()
    scores[0].layers[0].zero_()
    graphs[0].replay()
    got = [t.clone() for t in outs[0]]
    scores[0].layers[0].zero_()
    for a, b in zip(got, step(0)):
        assert torch.equal(a, b)
    assert_clean(ctx)
