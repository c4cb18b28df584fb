"""A block's dot is summed in f32 whatever the type of y: moe_fp8_product and moe_fp8_layer where large products cancel and small ones
remain, and within tests/fp8_ref.py's bounds of f32 sums for results in 16 bits.

In the tests of whole numbers every eight neighbouring products hold +2^16 and -2^16 and six of magnitude 1 at most.  The magnitudes of all of
them together stay below 2^24, so every partial sum in any order is a whole number that f32 holds, and y is the true sum rounded once."""
import numpy as np
import pytest
import torch

import fp8_ref as R
from moe_prefetch.fp8 import Fp8Linear, Fp8Moe
from test_gpu_fp8 import DEV, DT, F8, SHAPES, gen, moe, np64, randn, vals, weight, within

pytestmark = pytest.mark.gpu


def ones(g, *shape):
    """-1, 0 and 1"""
    return torch.randint(-1, 2, shape, generator=g, device=DEV).float()


def cancelling(g, N, K):
    """Rows of a weight: of every eight columns 256 and -256, then -1, 0 and 1."""
    w = ones(g, N, K)
    w[:, ::8] = 256.0
    w[:, 1::8] = -256.0
    if K % 8 == 1:
        w[:, -1] = 1.0                                    # (a last 256 alone would stay)
    return w


def large_pairs(g, M, K):
    """Rows of x: of every eight columns 256 twice, then 1 or -1 by the row."""
    x = torch.where(torch.rand((M, 1), generator=g, device=DEV) < 0.5, -1.0, 1.0).repeat(1, K)
    x[:, ::8] = 256.0
    x[:, 1::8] = 256.0
    if K % 8 == 1:
        x[:, -1] = 1.0
    return x


def rounded(v, dt):
    return np64(torch.tensor(v, dtype=torch.float32).to(DT[dt]))


# up to 16 rows; 32 x 64 tiles that share K; 64 x 64; 256 x 128; each on 16 bytes and off
@pytest.mark.parametrize("M, N, K", [(1, 200, 640), (13, 100, 1009), (40, 200, 640), (70, 130, 643), (900, 960, 640), (800, 1100, 635),
                                     (1800, 3600, 640), (1800, 3600, 257)])
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_product_of_large_ones_that_cancel(M, N, K, given, dt):
    g = gen(M + K)
    w, x = cancelling(g, N, K), large_pairs(g, M, K)
    lin = Fp8Linear(w.to(F8), torch.ones((R.blocks(N), R.blocks(K)), device=DEV))
    want = np64(x) @ np64(w).T
    if given:
        y = lin(x.to(F8), torch.ones((M, R.blocks(K)), device=DEV), out_dtype=DT[dt])
    else:
        y = lin(x.to(DT[dt]))                             # (256 <= 448 < 2 * 256: scales of 1)
    np.testing.assert_array_equal(np64(y), rounded(want, dt))


# one launch for down and the sum (up to 4 pairs), up to 512 pairs, sixteen rows of a weight a wave, tiles
@pytest.mark.parametrize("T, E, K", [(1, 5, 2), (2, 5, 2), (10, 16, 4), (30, 6, 3), (120, 20, 4), (150, 80, 4), (200, 16, 4), (600, 3, 2)])
@pytest.mark.parametrize("H, I", [(272, 640), (270, 635)])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_layer_of_large_ones_that_cancel(T, E, K, H, I, dt):
    # gate . x is 32, where silu(g) is g in f32; up . x is 8 in two of every eight rows and 1/32, 0 or -1/32 in the others, with the sign of
    # the token: h is 256, 256 and six of 1 at most, times that sign, which down multiplies by 256 and -256 and by -1, 0 and 1
    g = gen(T + I)
    sign = torch.where(torch.rand((T,), generator=g, device=DEV) < 0.5, -1.0, 1.0)
    x = torch.zeros((T, H), device=DEV)
    x[:, 0], x[:, 1] = 256.0, sign
    gate, up = torch.zeros((E, I, H), device=DEV), torch.zeros((E, I, H), device=DEV)
    gate[:, :, 0] = 0.125
    u = ones(g, E, I) / 32.0
    u[:, ::8], u[:, 1::8] = 8.0, 8.0
    up[:, :, 1] = u
    down = torch.stack([cancelling(g, H, I) for _ in range(E)])
    s = [torch.ones((E, R.blocks(n), R.blocks(k)), device=DEV) for n, k in ((I, H), (I, H), (H, I))]
    m = Fp8Moe(up.to(F8), gate.to(F8), down.to(F8), *s)
    ids = torch.randint(0, E, (T, K), generator=g, device=DEV, dtype=torch.int32)
    h = 32.0 * np64(u)
    each = np.einsum("en,emn->em", h, np64(down))
    want = np64(sign)[:, None] * each[ids.cpu().numpy()].sum(axis=1)
    out = m(x.to(DT[dt]), ids=ids, w=torch.ones((T, K), device=DEV))[0]
    np.testing.assert_array_equal(np64(out), rounded(want, dt))


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("M, N, K", SHAPES)
def test_product_within_f32_sums(M, N, K, given, dt):
    g = gen(2 * M + 1000 * N + K)
    w, ws = weight(g, N, K)
    if given:
        x, _ = weight(g, M, K)
        xs = torch.exp(randn(g, M, R.blocks(K))) * 0.01
        xq, s = vals(x), np64(xs)
        y = Fp8Linear(w, ws)(x, xs, out_dtype=DT[dt])
    else:
        x = randn(g, M, K).to(DT[dt])
        xq, s = R.quantize(np64(x))
        y = Fp8Linear(w, ws)(x)
    want, err = R.product(xq, s, vals(w), np64(ws))
    within(np64(y), want, R.out_bound(want, err, dt))


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("T, E, K, H, I", [(1, 8, 2, 256, 128), (7, 60, 6, 1000, 200), (64, 16, 4, 256, 384), (150, 80, 4, 128, 256), (130, 4, 1, 257, 100),
                                           (700, 3, 2, 256, 640), (150, 80, 4, 160, 700), (150, 80, 4, 700, 160), (300, 4, 2, 144, 720)])
def test_layer_within_f32_sums(T, E, K, H, I, dt):
    g = gen(T + 10 * E + H + 1)
    m, up, gate, down = moe(g, E, K, H, I)
    x, logits = randn(g, T, H).to(DT[dt]), randn(g, T, E)
    out, ids, w = m(x, logits)
    f = lambda q: (vals(q[0]), np64(q[1]))
    want, err = R.layer(np64(x), ids.cpu().numpy(), np64(w), f(gate), f(up), f(down))
    within(np64(out), want, R.out_bound(want, err, dt))
