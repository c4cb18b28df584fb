"""moe_fp8_quantize, moe_fp8_product and moe_fp8_layer against their definitions in 64 bits (tests/fp8_ref.py).

Codes and scales of the quantizer are equal; results of products and layers are within the bounds that fp8_ref derives from
their arithmetic, and half a step of their type."""
import math

import numpy as np
import pytest
import torch

import fp8_ref as R
from moe_prefetch.block import ScoredRouter
from moe_prefetch.fp8 import Fp8Linear, Fp8Moe, fp8_quantize

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
F8 = torch.float8_e4m3fn


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def np64(t):
    return t.double().cpu().numpy()


def vals(q):
    """The values of codes, from their bits."""
    return R.VALUES[q.contiguous().view(torch.uint8).cpu().numpy()]


def weight(g, *shape, spread=0.5):
    q = (randn(g, *shape) * 100.0).clamp(-448.0, 448.0).to(F8)
    s = torch.exp(spread * randn(g, *shape[:-2], R.blocks(shape[-2]), R.blocks(shape[-1]))) * 2e-4
    return q, s


def same(got, want):
    np.testing.assert_array_equal(got, want)


def within(got, y, bound):
    off = np.abs(got - y)
    bad = ~(off <= bound) & ~(np.isnan(got) & np.isnan(y))
    assert not bad.any(), (int(bad.sum()), float(np.nanmax(off / bound)), np.argwhere(bad)[:4])


# ---- the quantizer --------------------------------------------------------------
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("T, K", [(1, 1), (1, 128), (3, 127), (5, 129), (17, 8), (127, 257), (128, 128), (129, 260), (1, 5000),
                                  (300, 1000), (1000, 7), (64, 2048)])
def test_quantize(T, K, rows, dt):
    g = gen(T * 1000 + K)
    x = (randn(g, T, K) * torch.exp(3.0 * randn(g, T, 1))).to(DT[dt])
    q, s = fp8_quantize(x, rows=rows)
    assert q.dtype is F8 and q.shape == (T, K) and s.shape == (-(-T // rows), R.blocks(K))
    want, scale = R.quantize(np64(x), rows)
    same(np64(s), scale)
    same(vals(q), want)


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_quantize_special_values(dt, rows):
    g = gen(3)
    x = randn(g, 130, 300)
    x[0] = 0.0
    x[1, :128] = -0.0
    x[2, 5], x[2, 200], x[2, 299] = math.inf, -math.inf, math.nan
    x[3] = math.nan
    x[4] = math.inf
    x[5] = 448.0
    x[6], x[6, 3] = 1.0, 449.0
    x[7] = torch.linspace(-448, 448, 300, device=DEV)
    x[8] = 2.0 ** -24                                    # below the normal numbers of fp16
    x[9] = torch.linspace(2.0 ** -10, 2.0 ** -6, 300, device=DEV)
    x[9, ::128] = 448.0                                   # the rest below the normal numbers of e4m3
    x[10] = 65504.0 if dt == "f16" else 3.3e38
    if dt != "f16":
        x[11] = 1e-38
        x[12] = torch.tensor(list(range(300)), device=DEV, dtype=torch.float32) * 2.0 ** -140
    x = x.to(DT[dt])
    q, s = fp8_quantize(x, rows=rows)
    want, scale = R.quantize(np64(x), rows)
    same(np64(s), scale)
    same(vals(q), want)
    if rows == 1:
        same(np64(s)[3], [2.0 ** -126] * 3)
        assert np.isnan(vals(q)[3]).all()


def test_quantize_every_code_and_tie():
    # every value of e4m3 comes back, and the middles between neighbours go to the even one
    v = np.unique(R.VALUES[np.isfinite(R.VALUES)])
    mid = (v[1:] + v[:-1]) / 2
    x = np.full((2, 3 * 128), 448.0)
    x[0, :len(v)] = v
    x[1, :len(mid)] = mid
    x[:, ::128] = 448.0
    t = torch.tensor(x, device=DEV, dtype=torch.float32)
    q, s = fp8_quantize(t)
    same(np64(s), np.ones((2, 3)))
    same(vals(q), R.e4m3(x))
    keep = np.arange(len(v)) % 128 != 0
    same(vals(q)[0, :len(v)][keep], v[keep])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_strides(rows, dt):
    g = gen(4)
    big = randn(g, 150, 700).to(DT[dt])
    x = big[3:140, 5:405]
    qb = torch.full((140, 500), 7, dtype=torch.uint8, device=DEV)
    sb = torch.full((140, 9), -1.0, device=DEV)
    n = 137 if rows == 1 else 2
    q, s = qb[1:138, 3:403].view(F8), sb[2:2 + n, 1:5]
    got = fp8_quantize(x, rows=rows, q=q, scale=s)
    assert got[0] is q and got[1] is s
    want, scale = R.quantize(np64(x), rows)
    same(np64(s), scale)
    same(vals(q), want)
    qb[1:138, 3:403] = 7
    sb[2:2 + n, 1:5] = -1.0
    assert bool((qb == 7).all()) and bool((sb == -1.0).all())          # nothing beside


# ---- products -------------------------------------------------------------------
def check_product(x, w, ws, y, dt, xs=None):
    xq, s = R.quantize(np64(x)) if xs is None else (vals(x), np64(xs))
    want, err = R.product(xq, s, vals(w), np64(ws), cut=dt != "f32")
    within(np64(y), want, R.out_bound(want, err, dt))


SHAPES = [(1, 1, 1), (1, 16, 128), (2, 15, 100), (3, 17, 129), (5, 128, 16), (15, 129, 127), (16, 260, 256), (17, 64, 300), (33, 250, 1000),
          (63, 128, 512), (64, 128, 384), (65, 130, 640), (100, 257, 200), (128, 256, 256), (129, 384, 1024), (200, 100, 1537), (257, 513, 272),
          (600, 640, 512), (1, 2048, 2048), (8, 1000, 4096), (40, 300, 2048)]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M, N, K", SHAPES)
def test_product(M, N, K, dt):
    g = gen(M + 1000 * N + K)
    w, ws = weight(g, N, K)
    x = randn(g, M, K).to(DT[dt])
    y = Fp8Linear(w, ws)(x)
    assert y.dtype is DT[dt] and y.shape == (M, N)
    check_product(x, w, ws, y, dt)


@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M, N, K", SHAPES)
def test_product_given(M, N, K, out):
    g = gen(M + 1000 * N + K + 1)
    w, ws = weight(g, N, K)
    x, _ = weight(g, M, K)
    xs = torch.exp(randn(g, M, R.blocks(K))) * 0.01
    xs[::3] *= -1.0                                       # a scale is any number
    y = Fp8Linear(w, ws)(x, xs, out_dtype=DT[out])
    check_product(x, w, ws, y, out, xs)


@pytest.mark.parametrize("M", [1, 5, 40, 130, 300])
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("shift", [1, 4, 16])
def test_product_strides(M, given, shift):
    g = gen(M + shift)
    N, K = 200, 336
    wb, _ = weight(g, N + 2, K + shift + 16)
    w = wb[1:N + 1, shift:shift + K]
    ws = torch.rand((9, 10), generator=g, device=DEV)[2:4, 3:6] * 1e-3
    if given:
        xb, _ = weight(g, M + 1, K + 3 * shift)
        x = xb[1:, shift:shift + K]
        xs = torch.rand((M + 1, 8), generator=g, device=DEV)[1:, 2:5]
    else:
        x, xs = randn(g, M + 1, K + 3 * shift).to(torch.bfloat16)[1:, shift:shift + K], None
    yb = torch.full((M + 2, N + 7), -7.0, device=DEV)
    y = yb[1:M + 1, 3:N + 3]
    assert Fp8Linear(w, ws)(x, xs, out=y) is y
    check_product(x, w, ws, y, "f32", xs)
    y.fill_(-7.0)
    assert bool((yb == -7.0).all())


@pytest.mark.parametrize("M", [3, 70, 300])
def test_product_rows_with_nothing_finite(M):
    # a NaN or an infinity makes its own row NaN and no other; a row of zeros gives zeros
    g = gen(M)
    N, K = 130, 300
    w, ws = weight(g, N, K)
    x = randn(g, M, K)
    x[0, 17] = math.nan
    x[1, 299] = -math.inf
    x[2] = 0.0
    y = np64(Fp8Linear(w, ws)(x))
    assert np.isnan(y[:2]).all() and (y[2] == 0).all()
    want, err = R.product(*R.quantize(np64(x[2:])), vals(w), np64(ws))
    within(y[2:], want, R.out_bound(want, err, "f32"))


@pytest.mark.parametrize("M", [3, 70, 300])
def test_product_weight_nan(M):
    # a NaN in a weight makes its own column NaN
    g = gen(M)
    w, ws = weight(g, 150, 260)
    w.view(torch.uint8)[140, 259] = 0x7F
    x = randn(g, M, 260)
    y = np64(Fp8Linear(w, ws)(x))
    assert np.isnan(y[:, 140]).all() and np.isfinite(np.delete(y, 140, axis=1)).all()


@pytest.mark.parametrize("M", [4, 200])
def test_product_extreme_scales(M):
    # codes of the largest and the smallest size, scales over 60 powers of two
    g = gen(M)
    N, K = 140, 512
    w = torch.where(torch.rand((N, K), generator=g, device=DEV) < 0.5, 448.0, -(2.0 ** -9)).to(F8)
    x = torch.where(torch.rand((M, K), generator=g, device=DEV) < 0.5, -448.0, 2.0 ** -9).to(F8)
    ws = torch.exp2(torch.randint(-30, 31, (2, 4), generator=g, device=DEV).float())
    xs = torch.exp2(torch.randint(-30, 31, (M, 4), generator=g, device=DEV).float())
    y = Fp8Linear(w, ws)(x, xs, out_dtype=torch.float32)
    check_product(x, w, ws, y, "f32", xs)


def test_product_exact_sums():
    # whole numbers whose sums f32 holds: any order gives the same bits, in every kernel
    g = gen(9)
    for M, N, K in ((1, 200, 640), (20, 200, 640), (90, 200, 640), (400, 200, 640)):
        w = torch.randint(-8, 9, (N, K), generator=g, device=DEV).float().to(F8)
        x = torch.randint(-8, 9, (M, K), generator=g, device=DEV).float().to(F8)
        ws, xs = torch.ones((2, 5), device=DEV), torch.ones((M, 5), device=DEV)
        y = Fp8Linear(w, ws)(x, xs, out_dtype=torch.float32)
        same(np64(y), vals(x) @ vals(w).T)


def test_no_rows():
    g = gen(1)
    w, ws = weight(g, 20, 40)
    assert Fp8Linear(w, ws)(torch.empty((0, 40), device=DEV)).shape == (0, 20)
    q, s = fp8_quantize(torch.empty((0, 40), device=DEV))
    assert q.shape == (0, 40) and s.shape == (0, 1)
    m = moe(g, 4, 2, 40, 30)[0]
    out, ids, wt = m(torch.empty((0, 40), device=DEV), torch.empty((0, 4), device=DEV))
    assert out.shape == (0, 40) and ids.shape == (0, 2) and wt.shape == (0, 2)


# ---- the layer ------------------------------------------------------------------
def moe(g, E, K, H, I, **rule):
    up, gate, down = weight(g, E, I, H), weight(g, E, I, H), weight(g, E, H, I)
    router = ScoredRouter(E, K, **rule) if K else None
    return Fp8Moe(up[0], gate[0], down[0], up[1], gate[1], down[1], router=router), up, gate, down


def check_layer(x, ids, w, up, gate, down, out, dt):
    f = lambda m: (vals(m[0]), np64(m[1]))
    want, err = R.layer(np64(x), ids.cpu().numpy(), np64(w), f(gate), f(up), f(down), cut=(False, dt != "f32"))
    within(np64(out), want, R.out_bound(want, err, dt))


LAYERS = [(1, 8, 2, 256, 128), (1, 1, 1, 16, 16), (2, 5, 3, 130, 70), (4, 16, 4, 384, 256), (7, 60, 6, 1000, 200), (16, 32, 8, 512, 256),
          (17, 128, 8, 256, 128), (33, 9, 2, 300, 129), (64, 16, 4, 256, 384), (65, 8, 8, 128, 128), (130, 4, 1, 257, 100), (300, 6, 3, 512, 256),
          (700, 3, 2, 256, 640), (90, 16, 4, 384, 256), (100, 10, 4, 256, 384), (40, 8, 6, 512, 512), (1, 256, 10, 2048, 512), (5, 256, 8, 512, 64), (1100, 40, 4, 256, 256)]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T, E, K, H, I", LAYERS)
def test_layer(T, E, K, H, I, dt):
    g = gen(T + 10 * E + H)
    m, up, gate, down = moe(g, E, K, H, I)
    x, logits = randn(g, T, H).to(DT[dt]), randn(g, T, E)
    out, ids, w = m(x, logits)
    assert out.dtype is DT[dt]
    rid, rw = ScoredRouter(E, K)(logits)
    same(ids.cpu().numpy(), rid.cpu().numpy())
    same(np64(w), np64(rw))
    check_layer(x, ids, w, up, gate, down, out, dt)


@pytest.mark.parametrize("T", [1, 3, 20, 300])
def test_layer_rule(T):
    # sigmoid scores, a bias, groups, a scale, 16-bit logits in rows of a wider buffer
    g = gen(T)
    bias = 0.1 * randn(g, 64)
    rule = dict(score="sigmoid", bias=bias, n_groups=8, top_groups=4, group_best=2, scale=2.5)
    m, up, gate, down = moe(g, 64, 8, 256, 128, **rule)
    x, logits = randn(g, T, 256), randn(g, T, 70).to(torch.bfloat16)[:, 3:67]
    out, ids, w = m(x, logits, out_dtype=torch.float32)
    rid, rw = ScoredRouter(64, 8, **rule)(logits)
    same(ids.cpu().numpy(), rid.cpu().numpy())
    same(np64(w), np64(rw))
    check_layer(x, ids, w, up, gate, down, out, "f32")


@pytest.mark.parametrize("T", [1, 2, 16, 40, 64, 65, 200, 500])
@pytest.mark.parametrize("mode", ["one", "twice", "outside", "none", "some"])
def test_layer_given(T, mode):
    # every pair on one expert; an expert twice for a token; ids outside the experts; none inside
    g = gen(T)
    E, K, H, I = 12, 3, 272, 144
    m, up, gate, down = moe(g, E, 0, H, I)
    x = randn(g, T, H)
    ids = torch.randint(0, E, (T, K), generator=g, device=DEV, dtype=torch.int32)
    w = randn(g, T, K)
    if mode == "one":
        ids[:] = 7
    elif mode == "twice":
        ids[:, 1] = ids[:, 0]
    elif mode == "outside":
        ids[::2, 0], ids[1::2, 2], ids[0] = -1, E, torch.tensor([2 ** 31 - 1, -2 ** 31, 3], dtype=torch.int32)
    elif mode == "none":
        ids[:] = -1
    else:
        w[:, 1] = 0.0
    out, i, wt = m(x, ids=ids, w=w)
    assert i is ids and wt is w
    check_layer(x, ids, w, up, gate, down, out, "f32")
    if mode == "none":
        assert bool((out == 0).all())


@pytest.mark.parametrize("T", [2, 30, 260])
def test_layer_strides_and_views(T):
    # gate and up views of one tensor, experts apart, rows of x and out in wider buffers
    g = gen(T)
    E, K, H, I = 6, 2, 320, 128
    both, bs = weight(g, E, 2 * I, H + 16)
    both, bs = both[:, :, :H], bs[:, :, :3]
    wide, ds = weight(g, E, H + 5, I + 32)
    down, ds = wide[:, 5:, 7:7 + I], ds[:, :3, :1]
    m = Fp8Moe(both[:, I:], both[:, :I], down, bs[:, 1:], bs[:, :1], ds)
    xb, ob = randn(g, T, H + 13).to(torch.bfloat16), torch.full((T + 2, H + 9), -7.0, device=DEV)
    x, out = xb[:, 9:H + 9], ob[1:T + 1, 4:H + 4]
    ids = torch.randint(0, E, (T, K), generator=g, device=DEV, dtype=torch.int32)
    w = randn(g, T, K)
    assert m(x, ids=ids, w=w, out=out)[0] is out
    check_layer(x, ids, w, (both[:, I:], bs[:, 1:]), (both[:, :I], bs[:, :1]), (down, ds), out, "f32")
    out.fill_(-7.0)
    assert bool((ob == -7.0).all())


@pytest.mark.parametrize("T", [3, 40, 300])
def test_layer_row_of_nan(T):
    g = gen(T)
    m, up, gate, down = moe(g, 8, 2, 256, 160)
    x, logits = randn(g, T, 256), randn(g, T, 8)
    x[1, 100] = math.inf
    x[2] = 0.0
    out, ids, w = m(x, logits)
    y = np64(out)
    assert np.isnan(y[1]).all() and (y[2] == 0).all()
    x[1] = 1.0
    keep = [t for t in range(T) if t != 1]
    check_layer(x[keep], ids[keep], w[keep], up, gate, down, out[keep], "f32")


@pytest.mark.parametrize("T", [2, 50, 200])
def test_layer_far_experts(T):
    # experts 2^31 bytes apart: offsets pass 32 bits
    g = gen(T)
    E, K, H, I = 3, 2, 256, 128
    step = 2 ** 31 + 256
    n = I * H
    buf = torch.zeros(2 * step + 3 * n, dtype=torch.uint8, device=DEV)
    up, gate, down = weight(g, E, I, H), weight(g, E, I, H), weight(g, E, H, I)
    far = []
    for j, (q, rows, cols) in enumerate(((up[0], I, H), (gate[0], I, H), (down[0], H, I))):
        v = torch.as_strided(buf, (E, rows, cols), (step, cols, 1), j * n)
        v.copy_(q.view(torch.uint8))
        far.append(v.view(F8))
    m = Fp8Moe(*far, up[1], gate[1], down[1])
    x = randn(g, T, H)
    ids = torch.randint(0, E, (T, K), generator=g, device=DEV, dtype=torch.int32)
    w = randn(g, T, K)
    out = m(x, ids=ids, w=w)[0]
    check_layer(x, ids, w, up, gate, down, out, "f32")


# ---- as a step uses them -----------------------------------------------------------
@pytest.mark.parametrize("T", [1, 8, 30, 90, 400])
def test_together_captured_and_on_a_stream(T):
    # codes made of a 16-bit model's weights, a projection, a layer, a projection of codes; eager, on a stream, in two graphs
    # whose replays are mixed with eager work, on inputs that change
    g = gen(T)
    E, K, H, I = 16, 4, 384, 256
    q = [fp8_quantize(0.05 * randn(g, n, k), rows=128) for n, k in ((H, H), (200, H))]
    first, last = Fp8Linear(*q[0]), Fp8Linear(*q[1])
    up, gate, down = ([fp8_quantize(0.05 * randn(g, *shape), rows=128) for _ in range(E)] for shape in ((I, H), (I, H), (H, I)))
    m = Fp8Moe(*(torch.stack([c.view(torch.uint8) for c, _ in t]).view(F8) for t in (up, gate, down)),
               *(torch.stack([s for _, s in t]) for t in (up, gate, down)), router=ScoredRouter(E, K))
    router = 0.1 * randn(g, E, H)

    def step(x):
        h = first(x)
        out, ids, w = m(h, h.float() @ router.t())
        return last(*fp8_quantize(out), out_dtype=torch.float32), out, ids, w

    xs = [randn(g, T, H).to(torch.bfloat16) for _ in range(4)]
    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x, e in zip(xs, want):
            for a, b in zip(step(x), e):
                assert torch.equal(a, b)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        x = xs[0].clone()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            y = step(x)
        graphs.append((gr, x, y))
    for i in range(6):
        for k, (gr, x, y) in enumerate(graphs):
            x.copy_(xs[(i + k) % 4])
            gr.replay()
        again = step(xs[i % 4])
        torch.cuda.synchronize()
        for k, (gr, x, y) in enumerate(graphs):
            for a, b in zip(y, want[(i + k) % 4]):
                assert torch.equal(a, b), (i, k)
        for a, b in zip(again, want[i % 4]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T, E, K", [(90, 16, 4), (34, 4, 4), (150, 5, 2), (6, 8, 4)])
def test_the_same_bits_each_time(T, E, K):
    # experts whose last group of rows is not whole; several inputs in turn, so that nothing left behind is the call's own
    g = gen(90)
    m, up, gate, down = moe(g, E, K, 384, 256)
    xs = [(randn(g, T, 384).to(torch.bfloat16), randn(g, T, E)) for _ in range(5)]
    want = [m(*x) for x in xs]
    for x, (out, ids, w) in zip(xs, want):
        check_layer(x[0], ids, w, up, gate, down, out, "bf16")
    for i in range(60):
        for a, b in zip(m(*xs[7 * i % 5]), want[7 * i % 5]):
            assert torch.equal(a, b), i


def test_given_stream():
    g = gen(2)
    w, ws = weight(g, 300, 512)
    x = randn(g, 70, 512)
    want = Fp8Linear(w, ws)(x)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for stream in (s, s.cuda_stream):
        q, sc = fp8_quantize(x, stream=stream)
        y = Fp8Linear(w, ws)(q, sc, out_dtype=torch.float32, stream=stream)
        s.synchronize()
        assert torch.equal(y, want)


def test_the_same_rows_in_any_order():
    # a row's result does not depend on the rows beside it, for one kernel's sizes
    g = gen(5)
    w, ws = weight(g, 260, 640)
    x = randn(g, 48, 640)
    lin = Fp8Linear(w, ws)
    y = lin(x)
    p = torch.randperm(48, generator=g, device=DEV)
    assert torch.equal(lin(x[p]), y[p])
    m, *_ = moe(g, 16, 4, 256, 128)
    x, logits = randn(g, 48, 256), randn(g, 48, 16)
    out = m(x, logits)[0]
    assert torch.equal(m(x[p], logits[p])[0], out[p])
