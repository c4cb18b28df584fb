"""moe_fp8_product and moe_fp8_layer where their kernels change with the sizes: few and many pairs of an expert, rows too long for LDS at once,
weights off 16 bytes, the most pairs; against their definitions in 64 bits, within the bounds of tests/fp8_ref.py."""
import math

import numpy as np
import pytest
import torch

import fp8_ref as R
from moe_prefetch.fp8 import Fp8Linear, fp8_quantize
from test_gpu_fp8 import DEV, DT, check_layer, check_product, gen, moe, np64, randn, vals, weight, within

pytestmark = pytest.mark.gpu

LAYERS = [(1, 60, 3, 512, 1000), (1, 60, 4, 640, 1000), (1, 60, 5, 512, 1000), (2, 5, 2, 384, 7168), (1, 16, 4, 6000, 300), (2, 3, 2, 64, 14400),
          (20, 256, 4, 256, 128), (60, 20, 2, 7168, 128), (30, 4, 2, 7168, 64), (3, 40, 1, 20000, 40), (2, 3, 2, 64, 30000), (80, 128, 8, 128, 128),
          (150, 60, 4, 128, 256), (100, 60, 6, 200, 120), (64, 40, 4, 256, 256), (40, 8, 2, 272, 128), (65, 8, 2, 256, 128), (128, 64, 4, 130, 64),
          (129, 64, 4, 256, 64), (2, 256, 32, 128, 128), (4369, 20, 15, 32, 16), (700, 1, 1, 160, 144),
          (3, 2, 1, 1, 1), (40, 2, 2, 1, 5), (300, 2, 2, 5, 1), (600, 3, 2, 40, 130), (400, 2, 2, 256, 200)]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T, E, K, H, I", LAYERS)
def test_layer(T, E, K, H, I, dt):
    g = gen(3 * T + E + H)
    m, up, gate, down = moe(g, E, K, H, I)
    x, logits = randn(g, T, H).to(DT[dt]), randn(g, T, E)
    out, ids, w = m(x, logits)
    check_layer(x, ids, w, up, gate, down, out, dt)


@pytest.mark.parametrize("T, E, K, H, I", [(1, 9, 4, 384, 900), (4, 9, 1, 7168, 130), (13, 9, 4, 7168, 130), (33, 9, 2, 272, 7168), (250, 40, 2, 256, 128),
                                           (130, 200, 5, 208, 72)])
@pytest.mark.parametrize("mode", ["one", "twice", "outside", "most"])
def test_layer_given(T, E, K, H, I, mode):
    # all rows on one expert, however long; an expert twice for a token; ids outside the experts; nearly all rows on one expert
    g = gen(T + H)
    m, up, gate, down = moe(g, E, 0, H, I)
    x = randn(g, T, H)
    ids = torch.randint(0, E, (T, K), generator=g, device=DEV, dtype=torch.int32)
    w = randn(g, T, K)
    if mode == "one":
        ids[:] = E - 1
    elif mode == "twice":
        ids[:] = ids[:, :1]
    elif mode == "outside":
        ids[::2] = torch.tensor([-1, E, 2 ** 31 - 1, -2 ** 31, 256], dtype=torch.int32, device=DEV)[:K]
    else:
        ids[1:, :] = 3
    out = m(x, ids=ids, w=w)[0]
    check_layer(x, ids, w, up, gate, down, out, "f32")
    if mode == "outside":
        assert bool((out[::2] == 0).all())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("M, N, K", [(1, 1, 1 << 18), (20, 3, 100000), (7, 1 << 18, 3), (18, 1 << 18, 17), (40000, 16, 48), (17, 64, 128), (32, 64, 640),
                                     (33, 70, 1400), (500, 400, 2000), (16, 100, 6000), (9, 100, 7000), (16, 64, 3600)])
def test_product(M, N, K, dt):
    g = gen(M + N)
    w, ws = weight(g, N, K)
    x = randn(g, M, K).to(DT[dt])
    check_product(x, w, ws, Fp8Linear(w, ws)(x), dt)


@pytest.mark.parametrize("K", [640, 700])
@pytest.mark.parametrize("M", [2, 16, 40, 300])
def test_infinite_scale(M, K):
    # a weight's scale that is infinite: its rows are infinite with the sign of their dot, the others as ever
    g = gen(M)
    w, ws = weight(g, 200, K)
    w = torch.full_like(w.float(), 2.0).to(w.dtype)
    ws[1, -1] = math.inf
    x = 1.0 + randn(g, M, K).abs()
    x[1] *= -1.0
    y = Fp8Linear(w, ws)(x)
    assert bool((y[0, 128:] == math.inf).all()) and bool((y[1, 128:] == -math.inf).all())
    assert bool(torch.isfinite(y[:, :128]).all())


def test_two_streams_at_once():
    # one layer and one map, two streams that run beside each other with inputs of their own
    g = gen(8)
    m, up, gate, down = moe(g, 16, 4, 512, 256)
    w, ws = weight(g, 512, 512)
    lin = Fp8Linear(w, ws)
    xs = [(randn(g, T, 512).to(torch.bfloat16), randn(g, T, 16)) for T in (3, 40, 25, 300)]
    want = [m(lin(x), r)[0] for x, r in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(40):
        with torch.cuda.stream(streams[i % 2]):
            x, r = xs[(i + i // 4) % 4]
            got.append(((i + i // 4) % 4, m(lin(x), r)[0]))
    torch.cuda.synchronize()
    for k, y in got:
        assert torch.equal(y, want[k])
