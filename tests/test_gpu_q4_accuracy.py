"""Decode attention over the 4-bit cache where weights, scales and lengths lie far apart, against the 64-bit restatement.

Tolerances, per output value, with h = finfo(dtype).eps / 2 the half step of the output type and, as in the restatement,
bound = sum_t p_t (|o| + |s (c - 8)| + s c) and spread = the largest sum of |terms| of a logit:

  h |ref|                 the result's own rounding
  bound * 2^-15           a product p s enters in two 8-bit parts: the first cut (7 bits behind the leading one), the rest
                          rounded: 2^-16 of it; p against the offsets enters in two 11-bit parts: 2^-22; the tensor
                          cores cut each of at most 2 * 4 sums between two recentrings by at most 2^-23 of its size: 2^-20;
                          32-bit sums of a segment, of the subsets and of the parts: 2^-18 at the lengths here
  bound * 2 * 2^-17 * spread   a logit is a sum of at most 2^7 + 2^1 terms in 32 bits, and each weight is off by its logit's
                          error and by that of the sum
  2^-24                   the smallest step of an fp16 result
"""
import numpy as np
import pytest
import torch

from elasticmm_b200 import KVPoolQ4, get_context
from gpu_util import assert_clean, configure
from oracle import q4_oracle

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


@pytest.fixture()
def ctx():
    c = get_context(0)
    configure(c)
    return c


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def tolerance(ref, bound, spread, dtype):
    h = torch.finfo(dtype).eps / 2
    return h * np.abs(ref) + bound * (2.0 ** -15 + 2 * 2.0 ** -17 * spread[..., None]) + 2.0 ** -24


def check(got, ref, bound, spread, dtype):
    """got [copies, heads, D] against the one sequence's result [1, heads, D]."""
    err = np.abs(got.double().cpu().numpy() - ref)
    share = err / tolerance(ref, bound, spread, dtype)
    assert (share <= 1).all(), f"{share.max()} of the tolerance at {np.unravel_index(np.argmax(share), err.shape)}"


def whole_steps(n, H, D):
    """Values [n, H, D] of 0..15 whose groups all hold 0 and 15, so that scale 1 and offset 8 hold them exactly."""
    x = np.zeros((n, H, D), dtype=np.float32)
    x[:, :, 1::32] = 15.0
    return x


def run(ctx, key, value, q, BS, copies, dtype, scale=None):
    """The same sequence `copies` times in one call: with one for every SM, each is a segment of a CTA of its own."""
    n, H, D = key.shape
    NB = -(-n // BS)
    layer = np.zeros((2, NB * BS, H, q4_oracle.row_bytes(D)), dtype=np.uint8)
    for p, x in enumerate((key, value)):
        layer[p, :n] = q4_oracle.encode_rows(x.reshape(-1, D)).reshape(n, H, -1)
    layer = layer.reshape(2, NB, BS, H, -1)
    pool = KVPoolQ4([dev(layer)], D, ctx)
    tables = np.arange(NB, dtype=np.int32)[None]
    out = pool.attend(0, q.cuda().expand(copies, *q.shape[1:]).contiguous(), dev(tables.repeat(copies, 0)),
                      dev(np.full(copies, n, dtype=np.int32)), scale=scale)
    assert_clean(ctx)
    ref, _, bound, spread = q4_oracle.attend(layer, D, q.double().numpy(), tables, [n], D ** -0.5 if scale is None else scale)
    return out, ref, bound, spread


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("D,H,group,BS,copies", [(128, 8, 1, 16, 296), (128, 8, 8, 16, 296), (64, 8, 4, 16, 296), (256, 8, 2, 16, 148),
                                                 (128, 2, 4, 8, 148), (128, 8, 2, 16, 1)])
def test_a_large_scale_takes_no_bits_from_small_ones(ctx, D, H, group, BS, copies, dtype):
    """One token has half of the weight and a group of values with a scale above 2; thousands of others, each with 2^-13 of
    that weight, share the other half and hold groups with scales below 2^-8."""
    n, at = 8193, 100
    key = whole_steps(n, H, D)
    key[at, :, 0] = 13.0
    q = torch.zeros(1, H * group, D)
    q[..., 0] = float(np.log(2.0)) * D ** 0.5  # a step of the key doubles the weight
    q = q.to(dtype)
    rng = np.random.default_rng(D + group)
    small = 15 * 2.0 ** -8 * 0.99
    value = (rng.random((n, H, D)) * small).astype(np.float32)
    value[:, :, 33] += small / 2          # a mean of their own, so that nothing cancels
    value[at, :, :32] = np.linspace(-20, 20, 32)
    check(*run(ctx, key, value, q, BS, copies, dtype), dtype)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("exponent", [-20, -12, 0, 9])
def test_scales_over_the_whole_range_in_one_sequence(ctx, exponent, dtype):
    """Scales from 2^-20 to 2^12 side by side, a token apart and a group apart, under weights of 2^0 to 2^-13."""
    n, H, group, D, BS = 700, 4, 2, 128, 16
    rng = np.random.default_rng(exponent + 50)
    key = whole_steps(n, H, D)
    key[:, :, 0] = rng.integers(0, 14, (n, H))
    q = torch.zeros(1, H * group, D)
    q[..., 0] = float(np.log(2.0)) * D ** 0.5
    q = q.to(dtype)
    size = np.exp2(rng.integers(-20, 10, (n, H, D // 32))).astype(np.float32)
    size[:, :, 1] = 2.0 ** exponent       # one group in which all are alike
    size[: n // 2, :, 2] = 2.0 ** -20      # one that jumps
    size[n // 2:, :, 2] = 2.0 ** 9
    value = (rng.standard_normal((n, H, D // 32, 32)) * size[..., None]).reshape(n, H, D).astype(np.float16).astype(np.float32)
    check(*run(ctx, key, value, q, BS, 2, dtype), dtype)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("n,copies", [(577, 1), (8191, 148), (50000, 1)])
def test_ordinary_values_keep_32_bits_up_to_the_result(ctx, n, copies, dtype):
    """Normal keys and values, nearly equal weights: sums of thousands of products that cancel but for their mean."""
    H, group, D, BS = 4, 4, 128, 16
    rng = np.random.default_rng(n)
    key, value = (rng.standard_normal((n, H, D)).astype(np.float16).astype(np.float32) for _ in range(2))
    q = torch.randn(1, H * group, D, generator=torch.Generator().manual_seed(n)).to(dtype)
    check(*run(ctx, key, value, q, BS, copies, dtype), dtype)
