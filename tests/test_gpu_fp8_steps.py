"""The tile kernels of moe_fp8_product and moe_fp8_layer over many blocks of K: their scales are renewed every six blocks and their stages go
round three places, so K has 6, 7, 11 and more blocks (6 n, 6 n + 1, 6 n + 5), with a short last one and without, with rows on 16 bytes and
off, in every form of tiles that products and layers take, and with tiles in both directions whose last ones are not whole.

Products of whole numbers of at most 8 with scales of 1, 2 and 4 that differ by block and row: the magnitudes of all of a row's terms stay below
64 * 16 * K < 2^24, so sums in any order are exact in f32, and y is the true sum rounded once.  Layers are held to fp8_ref's bounds of f32 sums."""
import numpy as np
import pytest
import torch

import fp8_ref as R
from moe_prefetch.fp8 import Fp8Linear
from test_gpu_fp8 import DEV, DT, F8, gen, moe, np64, randn, vals, weight, within

pytestmark = pytest.mark.gpu

# K: 6, 7, 11 and 12 blocks; 6, 7 and 11 and a short one, on 16 bytes; 6, 8 and 12 and a short one off 16 bytes
DEPTHS = [768, 896, 1408, 1536, 800, 912, 1424, 775, 1100, 1660]


def whole_numbers(g, n, k):
    return torch.randint(-8, 9, (n, k), generator=g, device=DEV).float().to(F8)


def scales(g, *shape):
    return torch.exp2(torch.randint(0, 3, shape, generator=g, device=DEV).float())


def check_exact(M, N, K, dt):
    g = gen(M + N + K)
    w, x = whole_numbers(g, N, K), whole_numbers(g, M, K)
    ws, xs = scales(g, R.blocks(N), R.blocks(K)), scales(g, M, R.blocks(K))
    y = Fp8Linear(w, ws)(x, xs, out_dtype=DT[dt])
    want = R.dequant(vals(x), np64(xs), 1) @ R.dequant(vals(w), np64(ws), R.B).T
    np.testing.assert_array_equal(np64(y), np64(torch.tensor(want, dtype=torch.float32).to(DT[dt])))


# 500 x 2,500: 320 tiles of 64 x 64, 40 of 256 x 128
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("K", DEPTHS)
def test_product_of_64_x_64(K, dt):
    check_exact(500, 2500, K, dt)


# 2,600 x 3,000: 12 x 21 tiles of 256 x 128, in strips of eight, the last of five
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("K", DEPTHS)
def test_product_of_256_x_128(K, dt):
    check_exact(2600, 3000, K, dt)


# 70 x 300: 32 x 64 tiles, K shared by two groups of waves, from 32 blocks on by four
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("K", [*DEPTHS, 1, 16, 48, 100, 127, 128, 130, 144, 256, 272, 1664, 3200, 3968, 4000, 4080, 4096, 4112, 4224, 4240, 4352, 4608, 6400, 6528, 8000, 4100, 7000])
def test_product_with_k_shared(K, dt):
    check_exact(70, 300, K, dt)


@pytest.mark.parametrize("M, N, K", [(500, 2500, 2000), (1000, 1300, 900), (2600, 3000, 1100), (64, 1000, 2048), (30, 260, 5000)])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_product_of_quantized_rows(M, N, K, dt):
    # numbers of every size, x quantized on the way; a sample of the columns, each with its block of the weight's scales
    g = gen(M + N + K)
    w, ws = weight(g, N, K)
    x = randn(g, M, K).to(DT[dt])
    y = Fp8Linear(w, ws)(x)
    rows, cols = np.arange(0, M, 7), np.unique(np.r_[np.arange(0, N, 13), N - 1])
    xq, s = R.quantize(np64(x[rows]))
    xd, wd = R.dequant(xq, s, 1), R.dequant(vals(w), np64(ws), R.B)[cols]
    want = xd @ wd.T
    err = (2 * R.B + 1 + R.blocks(K) + 8) * R.U * (np.abs(xd) @ np.abs(wd).T)
    within(np64(y)[np.ix_(rows, cols)], want, R.out_bound(want, err, dt))


# 150 pairs an expert (tiles of 128 rows for gate and up) and 37 (of 64): H is the depth of gate and up, I that of down
@pytest.mark.parametrize("T, E, K", [(300, 4, 2), (150, 16, 4)])
@pytest.mark.parametrize("H, I", [(768, 896), (896, 1408), (1408, 768), (800, 912), (912, 1424), (1424, 800), (768, 1600), (2100, 768), (1600, 1100), (1100, 775),
                                  (2048, 768)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_layer_on_tiles(T, E, K, H, I, dt):
    g = gen(T + H + I)
    m, up, gate, down = moe(g, E, K, H, I, score="softmax")
    x, logits = randn(g, T, H).to(DT[dt]), randn(g, T, E)
    out, ids, w = m(x, logits)
    f = lambda q: (vals(q[0]), np64(q[1]))
    want, err = R.layer(np64(x), ids.cpu().numpy(), np64(w), f(gate), f(up), f(down))
    within(np64(out), want, R.out_bound(want, err, dt))
