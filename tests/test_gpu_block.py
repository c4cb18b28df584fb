"""moe_route_scored, moe_block_norm and moe_sample against their definitions in 64 bits (tests/block_ref.py).

Chosen ids and tokens are equal.  Weights and probabilities are rounded to f32 once: half a step (2^-24, a 64-bit
remainder beside it).  y and r are within the bound that block_ref derives from the f32 arithmetic, and half a step
of their type."""
import math

import numpy as np
import pytest
import torch

import block_ref as R
from moe_prefetch import _lib
from moe_prefetch.block import BlockNorm, Sampler, ScoredRouter

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
INF, NAN = math.inf, math.nan


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def np64(t):
    return None if t is None else t.double().cpu().numpy()


# ---- routing --------------------------------------------------------------------
def check_route(logits, got, scores=None, **rule):
    ids, w, s = R.route(np64(logits), **rule)
    np.testing.assert_array_equal(got[0].cpu().numpy(), ids)
    np.testing.assert_allclose(np64(got[1]), w, rtol=R.U * 1.001, atol=2.0 ** -149)
    if scores is not None:
        np.testing.assert_allclose(np64(scores), s, rtol=R.U * 1.001, atol=2.0 ** -149)


RULES = [dict(score="softmax"), dict(score="softmax", renormalize=False, scale=1.7),
         dict(score="sigmoid", bias=True, scale=2.5),
         dict(score="sigmoid", bias=True, n_groups=8, top_groups=4, group_best=2, scale=2.5),
         dict(score="softmax", n_groups=4, top_groups=2, group_best=1, renormalize=False)]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T, E, K", [(1, 256, 8), (3, 64, 6), (7, 8, 8), (65, 128, 8), (5, 160, 6), (130, 256, 8),
                                     (9, 512, 22), (2, 1024, 64), (33, 72, 1)])
@pytest.mark.parametrize("rule", RULES)
def test_route(rule, T, E, K, dt):
    g = gen(T * 1000 + E)
    rule = dict(rule)
    logits = (1.5 * randn(g, T, E)).to(DT[dt])
    bias = 0.1 * randn(g, E) if rule.pop("bias", False) else None
    if rule.get("n_groups", 1) > 1:
        m = E // rule["n_groups"]
        rule["top_groups"] = max(rule["top_groups"], -(-K // m))
        rule["group_best"] = min(rule["group_best"], m)
    scores = torch.empty((T, E), dtype=torch.float32, device=DEV)
    got = ScoredRouter(E, K, bias=bias, **rule)(logits, scores=scores)
    check_route(logits, got, scores, K=K, bias=None if bias is None else np64(bias), **rule)


@pytest.mark.parametrize("E, K, n_groups, top_groups, group_best", [
    (1, 1, 1, 1, 1), (2, 2, 2, 2, 1), (65, 7, 5, 2, 2), (63, 9, 7, 3, 2), (64, 4, 64, 5, 1), (192, 16, 3, 1, 2),
    (96, 3, 12, 1, 2), (1000, 10, 8, 3, 2), (576, 64, 64, 8, 1)])
def test_route_odd_groups(E, K, n_groups, top_groups, group_best):
    g = gen(E)
    logits = randn(g, 21, E)
    bias = 0.2 * randn(g, E)
    rule = dict(score="sigmoid", n_groups=n_groups, top_groups=top_groups, group_best=group_best)
    check_route(logits, ScoredRouter(E, K, bias=bias, **rule)(logits), K=K, bias=np64(bias), **rule)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_equal_scores_take_the_lower_id(score, groups):
    logits = torch.randint(-1, 2, (40, 128), generator=gen(3), device=DEV).float()
    logits[0] = 0.5
    rule = dict(score=score, n_groups=groups, top_groups=max(1, groups // 2), group_best=2)
    got = ScoredRouter(128, 8, **rule)(logits)
    check_route(logits, got, K=8, **rule)
    assert got[0][0].tolist() == list(range(8))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 8])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_route_switched_off_and_extreme_logits(score, groups, dt):
    E, K = 64, 8
    l = randn(gen(5), 16, E)
    l[0] = -INF                                       # nothing is on
    l[1] = NAN
    l[2, 3:] = -INF                                   # fewer than K
    l[3, ::2] = NAN
    l[4, 7] = INF
    l[5, [9, 30, 31]] = INF
    l[6] = INF
    l[7, 8:16] = -INF                                 # a group of eight off
    l[8, 17:24] = -INF                                # a group of one
    l[9] = torch.finfo(DT[dt]).min                    # the type's lowest value is a number
    l[10] = torch.finfo(DT[dt]).max
    l[11, 5] = torch.finfo(DT[dt]).max
    l[12] = -0.0
    l[13] = -800.0 if dt != "f16" else -60000.0       # sigmoid scores that leave nothing
    l = l.to(DT[dt])
    rule = dict(score=score, n_groups=groups, top_groups=max(1, groups // 2), group_best=2)
    scores = torch.empty((16, E), dtype=torch.float32, device=DEV)
    got = ScoredRouter(E, K, **rule)(l, scores=scores)
    check_route(l, got, scores, K=K, **rule)
    assert all(len(set(r)) == K for r in got[0].tolist())
    assert not got[1].isnan().any()


def test_route_bias_switches_off_and_forces():
    E, K = 32, 4
    l = randn(gen(6), 9, E)
    bias = torch.zeros(E, device=DEV)
    bias[3], bias[4], bias[9] = -INF, NAN, INF
    for groups in (1, 4):
        rule = dict(score="sigmoid", n_groups=groups, top_groups=max(1, groups // 2))
        got = ScoredRouter(E, K, bias=bias, **rule)(l)
        check_route(l, got, K=K, bias=np64(bias), **rule)
        assert (got[0] == 9).any(1).all() and not ((got[0] == 3) | (got[0] == 4)).any()
    # a balancing step changes the bias in place between calls
    r = ScoredRouter(E, K, bias=bias)
    bias.zero_()
    check_route(l, r(l), K=K, bias=np64(bias))


def test_route_slots_strides_and_rows_left_alone():
    E, K, T = 64, 6, 11
    buf = randn(gen(7), T, 3 * E + 1)
    for logits in (buf[:, 1:E + 1], buf[:, 5:E + 5].to(torch.bfloat16), buf.to(torch.float16)[:, 3:E + 3]):
        table = torch.randperm(E, generator=gen(8), device=DEV).to(torch.int32)
        ids = torch.full((T + 2, K), -7, dtype=torch.int32, device=DEV)
        w = torch.full((T + 2, K), 5.0, device=DEV)
        slots = torch.full((T + 2, K), -9, dtype=torch.int32, device=DEV)
        got = ScoredRouter(E, K)(logits, ids=ids[:T], w=w[:T], table=table, slots=slots[:T])
        check_route(logits, got, K=K)
        assert torch.equal(slots[:T], table[ids[:T].long()])
        assert (ids[T:] == -7).all() and (w[T:] == 5.0).all() and (slots[T:] == -9).all()
        ScoredRouter(E, K)(logits, slots=slots[:T])
        assert (slots[:T] == E).all()


def test_route_matches_moe_route():
    # where both apply the ids are those of moe_route, and the weights within its f32 arithmetic
    from moe_prefetch.batched import BatchedMoe
    logits = 2.0 * randn(gen(9), 50, 128)
    m = BatchedMoe(50)
    ids, w = m.route(50, logits=logits)
    ids2, w2 = ScoredRouter(128, 8)(logits)
    torch.cuda.synchronize()
    assert torch.equal(ids, ids2)
    assert torch.allclose(w, w2, rtol=2e-6, atol=0)


def exact_product(g, T, E):
    """W, x whose product is exact in f32 in any order (small whole numbers, W over 64), and the product."""
    W = torch.randint(-3, 4, (E, 2048), generator=g, device=DEV).float() / 64.0
    x = torch.randint(-2, 3, (T, 2048), generator=g, device=DEV).float()
    return W, x, (x.double() @ W.double().t())


@pytest.mark.parametrize("T, E, K", [(1, 64, 6), (3, 256, 8), (37, 128, 8), (300, 256, 10), (1000, 128, 1)])
def test_route_from_the_routers_product(T, E, K):
    from moe_prefetch.batched import BatchedMoe
    g = gen(40 + T)
    W, x, logits = exact_product(g, T, E)
    bias = 0.1 * randn(g, E)
    rule = dict(score="sigmoid", n_groups=8, top_groups=4, group_best=2, scale=2.5)
    m = BatchedMoe(T + 2, n_experts=E, n_expert_used=K)
    m.ids.fill_(-3)
    torch.cuda.synchronize()
    got = m.route(T, W=W, x=x, router=ScoredRouter(E, K, bias=bias, **rule))
    torch.cuda.synchronize()
    check_route(logits, got, K=K, bias=np64(bias), **rule)
    assert (m.ids[T:] == -3).all()
    # and from given logits
    got = m.route(T, logits=logits.float(), router=ScoredRouter(E, K, bias=bias, **rule))
    torch.cuda.synchronize()
    check_route(logits, got, K=K, bias=np64(bias), **rule)
    for bad in (dict(router=ScoredRouter(E, K + 1)), dict(router=ScoredRouter(E, K), table=m.ids),
                dict(router=ScoredRouter(E, K), logits=logits.float()[:0])):
        with pytest.raises(ValueError):
            m.route(T, **{"W": W, "x": x, **bad})


# ---- block norm -----------------------------------------------------------------
def check_norm(dt, x, got, y_dt=None, **kw):
    y, r, e_y, e_r = R.block_norm(np64(x), **{k: np64(v) if torch.is_tensor(v) else v for k, v in kw.items()})
    for name, t, want, err, half in (("y", got[0], y, e_y, R.HALF[y_dt or dt]), ("r", got[1], r, e_r, R.HALF[dt])):
        if t is None:
            continue
        tiny = {"f32": 0.0, "bf16": 0.0, "f16": 2.0 ** -25}[y_dt or dt if name == "y" else dt]   # half a subnormal step
        lim = err + half * (np.abs(want) + err) + tiny
        d = np.abs(np64(t) - want)
        assert (d <= lim).all(), (name, float((d / np.maximum(lim, 1e-300)).max()))


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T, H", [(1, 2048), (5, 2048), (1, 1), (3, 7), (2, 63), (4, 64), (3, 65), (2, 513), (9, 1024),
                                  (2, 1537), (2, 4096), (3, 5120), (2, 8191), (1, 8192), (2, 16383), (1, 16384)])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_norm_sizes(kind, T, H, dt):
    g = gen(H + T)
    x = (2.0 * randn(g, T, H) + 0.3).to(DT[dt])
    b = randn(g, T, 3, H)
    wt = lambda: (1.0 + 0.2 * randn(g, H)).to(DT[dt])
    kw = dict(weight=wt(), bias=wt(), post_weight=wt(), post_bias=wt(), kind=kind)
    got = BlockNorm(H, scale=0.3, **kw)(x, b)
    check_norm(dt, x, got, branch=b, post=True, scale=0.3, **kw)


@pytest.mark.parametrize("dt, y_dt, b_dt, w_dt", [("bf16", "bf16", "bf16", "bf16"), ("bf16", "f32", "f32", "f32"),
                                                  ("f16", "f32", "f16", "f32"), ("f16", "f16", "f32", "f16"),
                                                  ("f32", "f32", "f32", "f32"), ("bf16", "f32", "bf16", "f32")])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", [None, "token", "channel", "full", "row"])
@pytest.mark.parametrize("pairs", [0, 1, 8])
def test_norm_forms(pairs, gate, post, dt, y_dt, b_dt, w_dt):
    T, H = 6, 520
    g = gen(11)
    x = randn(g, T, H).to(DT[dt])
    b = (randn(g, T, pairs, H) if pairs else randn(g, T, H)).to(DT[b_dt])
    gt = {None: None, "token": (T,), "channel": (H,), "full": (T, H), "row": (T, 1)}[gate]
    act = "sigmoid" if gate in ("token", "full") else None
    gt = None if gt is None else randn(g, *gt).to(DT[dt] if gate == "full" else torch.float32)
    w = (randn(g, H) * 0.2).to(DT[w_dt])
    pw = (randn(g, H) * 0.2).to(DT[w_dt]) if post else None
    kw = dict(weight=w, post_weight=pw, weight_offset=1.0, scale=0.22, gate_act=act, post_eps=1e-3)
    got = BlockNorm(H, **kw)(x, b, gt, out_dtype=DT[y_dt])
    assert got[0].dtype == DT[y_dt] and got[1].dtype == DT[dt]
    check_norm(dt, x, got, y_dt, branch=b, gate=gt, post=post, **kw)


def test_norm_without_branch_weights_or_outputs():
    T, H = 5, 2048
    x = randn(gen(12), T, H).to(torch.bfloat16)
    y, r = BlockNorm(H)(x)
    assert r is x
    check_norm("bf16", x, (y, None))
    r = torch.empty_like(x)
    BlockNorm(H)(x, residual=r)
    assert torch.equal(r, x)
    # a post-norm without weights
    b = randn(gen(13), T, H)
    check_norm("bf16", x, BlockNorm(H, post=True)(x, b), branch=b, post=True)


@pytest.mark.parametrize("H", [2048, 1537, 9, 5, 3, 1, 4095, 9001])
def test_norm_in_place_and_strides(H):
    T, g = 7, gen(14)
    buf = randn(g, T + 2, H + 37).to(torch.bfloat16)
    for off in (0, 1, 8):
        x = buf[1:T + 1, off:off + H]
        b = randn(g, T, H + 5)[:, 3:H + 3]
        was, keep = x.clone(), buf.clone()
        y, r = BlockNorm(H, scale=0.5)(x, b, residual=x, out=torch.empty_like(buf)[1:T + 1, off:off + H])
        check_norm("bf16", was, (y, r), branch=b, scale=0.5)
        assert r.data_ptr() == x.data_ptr()
        keep[1:T + 1, off:off + H] = r
        assert torch.equal(buf, keep)                 # nothing beside the rows was written
    x = buf[1:T + 1, :H]
    was = x.clone()
    check_norm("bf16", was, (BlockNorm(H)(x, out=x)[0], None))


def test_norm_of_zeros_large_values_and_nan():
    H = 2048
    x = torch.zeros(4, H, device=DEV)
    x[1] = 1e17
    x[2, 5] = NAN
    y, _ = BlockNorm(H)(x)
    assert (y[0] == 0).all() and torch.allclose(y[1], torch.ones(H, device=DEV), rtol=1e-5)
    assert y[2].isnan().all() and (y[3] == 0).all()
    # rows are apart: a NaN in one stays there
    y, _ = BlockNorm(H, kind="layer", bias=torch.ones(H, device=DEV))(x)
    assert (y[0] == 1).all() and y[2].isnan().all() and (y[3] == 1).all()


# ---- sampling -------------------------------------------------------------------
def check_sample(logits, u, got, **kw):
    tokens, probs = R.sample(np64(logits), np64(u), **{k: np64(v) if torch.is_tensor(v) else v for k, v in kw.items()})
    np.testing.assert_array_equal(got[0].cpu().numpy(), tokens)
    # a mass is off by at most 2^-(63 - ceil(log2 V)), so V of them by V^2 2^-62 beside a total of at least 1
    V = logits.shape[1]
    np.testing.assert_allclose(np64(got[1]), probs, rtol=R.U * 1.000001 + V * V * 2.0 ** -62, atol=2.0 ** -149)


CUTS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=40, temperature=0.8), dict(top_p=0.9),
        dict(min_p=0.05), dict(top_k=50, top_p=0.95, min_p=0.02, temperature=1.1), dict(top_k=1500, top_p=0.999),
        dict(temperature=3.0, top_p=0.97), dict(temperature=0.0), dict(top_k=5, min_p=0.9), dict(temperature=1e38)]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T, V", [(1, 151936), (4, 32003), (17, 1000), (3, 8192), (5, 4097), (2, 65), (2, 64), (3, 2),
                                  (2, 1), (40, 257)])
@pytest.mark.parametrize("cut", CUTS)
def test_sample(cut, T, V, dt):
    g = gen(V + T)
    logits = 2.0 * randn(g, T, V)
    logits[:, ::max(1, V // 9)] += 6.0
    logits = logits.to(DT[dt])
    u = torch.rand(T, generator=g, device=DEV)
    check_sample(logits, u, Sampler(V)(logits, u, **cut), **cut)


@pytest.mark.parametrize("spread", [0.0, 1e-3, 30.0])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_sample_flat_and_peaked_rows(spread, dt):
    T, V, g = 12, 70001, gen(21)
    logits = (spread * randn(g, T, V)).to(DT[dt])
    u = torch.rand(T, generator=g, device=DEV)
    for cut in (dict(), dict(top_p=0.5), dict(top_k=60000), dict(min_p=0.999, top_p=0.25), dict(top_k=7, top_p=0.3)):
        check_sample(logits, u, Sampler(V)(logits, u, **cut), **cut)


def test_sample_rows_of_their_own():
    T, V, g = 64, 50257, gen(22)
    logits = 3.0 * randn(g, T, V)
    r = lambda: torch.rand(T, generator=g, device=DEV)
    temperature = torch.where(r() < 0.2, torch.zeros(T, device=DEV), 0.2 + 2.0 * r())
    kw = dict(temperature=temperature, top_k=torch.randint(-2, 300, (T,), generator=g, device=DEV, dtype=torch.int32),
              top_p=1.1 * r(), min_p=torch.where(r() < 0.5, torch.zeros(T, device=DEV), 0.2 * r()))
    u = r()
    check_sample(logits, u, Sampler(V)(logits, u, **kw), **kw)
    # the same row gives the same token in any batch
    for t in (0, 13, 63):
        one = Sampler(V)(logits[t:t + 1], u[t:t + 1], **{k: v[t:t + 1] for k, v in kw.items()})
        all_ = Sampler(V)(logits, u, **kw)
        assert one[0][0] == all_[0][t] and one[1][0] == all_[1][t]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("levels", [1, 3, 200])
def test_sample_equal_logits(levels, dt):
    # many equal logits: borders inside runs of equal tokens, sums that are whole numbers
    T, V, g = 24, 5000, gen(23)
    logits = torch.randint(0, levels, (T, V), generator=g, device=DEV).to(DT[dt])
    u = torch.arange(T, device=DEV).float() / T
    for cut in (dict(), dict(top_k=777), dict(top_p=0.5), dict(top_k=3000, top_p=0.75), dict(min_p=1.0)):
        check_sample(logits, u, Sampler(V)(logits, u, **cut), **cut)


def test_sample_ends_of_u_and_parameters_out_of_range():
    V = 3000
    logits = randn(gen(24), 8, V)
    u = torch.tensor([0.0, 1.0, 2.0, -1.0, NAN, 1.0 - 2.0 ** -24, INF, 0.5], device=DEV)
    for cut in (dict(), dict(top_k=9), dict(top_p=0.6)):
        check_sample(logits, u, Sampler(V)(logits, u, **cut), **cut)
    for cut in (dict(top_p=0.0), dict(top_p=-1.0), dict(top_k=-5), dict(top_k=V), dict(top_k=V + 1), dict(min_p=-1.0),
                dict(min_p=2.0), dict(top_p=NAN), dict(min_p=NAN), dict(temperature=NAN), dict(temperature=-1.0),
                dict(temperature=1e-30), dict(temperature=1e30), dict(temperature=INF)):
        if cut.get("top_p") != cut.get("top_p") or cut.get("min_p") != cut.get("min_p"):
            check_sample(logits, u, Sampler(V)(logits, u, **cut))           # cuts nothing
        else:
            check_sample(logits, u, Sampler(V)(logits, u, **cut), **cut)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_sample_switched_off_and_extreme_logits(dt):
    V, big = 2500, torch.finfo(DT[dt]).max
    l = randn(gen(25), 12, V)
    l[0] = -INF
    l[1] = NAN
    l[2, 1:] = -INF
    l[3, :-1] = NAN
    l[4, 100:] = -INF
    l[5, ::3] = NAN
    l[6, 77] = INF
    l[7, [5, 600, 2499]] = INF
    l[8] = -big
    l[9, 3] = big
    l[10, 10:] = -big                                 # a mask of the type's lowest value
    l[11, :] = -0.0
    l[11, 1::2] = 0.0
    l = l.to(DT[dt])
    for s in (0.0, 0.3, 0.7, 0.999):
        u = torch.full((12,), s, device=DEV)
        for cut in (dict(), dict(top_k=50), dict(top_p=0.9), dict(min_p=0.1), dict(temperature=0.0),
                    dict(top_k=200, top_p=0.5, temperature=2.0)):
            got = Sampler(V)(l, u, **cut)
            check_sample(l, u, got, **cut)
            assert got[0][:2].tolist() == [-1, -1] and got[1][:2].tolist() == [0.0, 0.0]


def test_sample_strides_and_rows_left_alone():
    T, V = 6, 4001
    buf = 2.0 * randn(gen(26), T, V + 77)
    u = torch.rand(T, generator=gen(27), device=DEV)
    for dt in DT.values():
        for off in (0, 1, 3, 8):
            logits = buf.to(dt)[:, off:off + V]
            tokens = torch.full((T + 3,), -5, dtype=torch.int32, device=DEV)
            probs = torch.full((T + 3,), 9.0, device=DEV)
            got = Sampler(V)(logits, u, top_k=30, top_p=0.9, tokens=tokens[:T], probs=probs[:T])
            check_sample(logits, u, got, top_k=30, top_p=0.9)
            assert (tokens[T:] == -5).all() and (probs[T:] == 9.0).all()


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_sample_of_a_long_tail(dt, sign):
    # the draw falls among tokens far below the first (the last, open bin of the undecided rows' histogram) beside many
    # that are switched off; and among equal 16-bit logits next to the bin that is gathered
    V, g = 100000, gen(60)
    l = torch.full((6, V), -INF, device=DEV)
    top = 30.0 if sign > 0 else -1.0
    for t in range(3):
        at = torch.randperm(V, generator=g, device=DEV)[:1500]
        l[t, at] = top - 23.5 - 0.2 * torch.rand(1500, generator=g, device=DEV)
        l[t, at[0]] = top
    for t in range(3, 6):                             # thousands of equal logits, the cut among their neighbours
        l[t] = top - 3.0 - torch.randint(0, 400, (V,), generator=g, device=DEV) / 100.0
    l = l.to(DT[dt])
    for s in (1.0 - 2.0 ** -24, 1.0 - 2.0 ** -23, 0.999, 0.5):
        u = torch.full((6,), s, device=DEV)
        for cut in (dict(), dict(top_p=0.9), dict(top_k=1400), dict(min_p=1e-12), dict(top_p=0.99999988, min_p=1e-11)):
            check_sample(l, u, Sampler(V)(l, u, **cut), **cut)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [999, 1001, 4088, 4089, 4095, 8184, 8185, 98295, 102400])
def test_sample_sizes_next_to_the_slices(dt, V):
    # rows at every alignment of their type, the likely tokens in one run of neighbours or at both ends
    size = 4 if dt == "f32" else 2
    for m in range(16 // size):
        g = gen(70 + m)
        wide = torch.full((4, V + 16), 50.0, device=DEV).to(DT[dt])
        rows = wide[:, m:m + V] if (V + 16) * size % 16 == 0 else wide.flatten()[m:m + 4 * V].view(4, V)
        l = randn(g, 4, V)
        l[0, V // 3:V // 3 + 700] += 9.0
        l[1, :8] += 9.0
        l[1, -8:] += 9.0
        l[2] *= 0.01
        l[3] -= 40.0
        rows.copy_(l)
        u = torch.rand(4, generator=g, device=DEV)
        for cut in (dict(), dict(top_k=300), dict(top_p=0.95, temperature=1.5), dict(min_p=0.3), dict(top_k=9, top_p=0.5)):
            check_sample(rows, u, Sampler(V)(rows, u, **cut), **cut)


def test_sample_the_same_bits_each_time():
    # whatever order workgroups and waves take their turns in
    V, T, g = 30011, 200, gen(62)
    logits = (0.3 + 2.0 * torch.rand(T, 1, generator=g, device=DEV)) * randn(g, T, V)
    u = torch.rand(T, generator=g, device=DEV)
    for cut in (dict(), dict(top_k=300), dict(top_k=1000, top_p=0.7), dict(top_k=20000, min_p=0.01), dict(top_p=0.9)):
        want = Sampler(V)(logits, u, **cut)
        for _ in range(20):
            got = Sampler(V)(logits, u, **cut)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        for t in (0, 77, 199):
            one = Sampler(V)(logits[t:t + 1].clone(), u[t:t + 1], **cut)
            if logits[t].data_ptr() % 16 == 0:
                assert one[0][0] == want[0][t] and one[1][0] == want[1][t]


def test_sample_more_rows_than_a_launch():
    V, T = 300, 4096 + 77
    g = gen(61)
    logits = 3.0 * randn(g, T, V + 5)[:, 2:V + 2]
    u = torch.rand(T, generator=g, device=DEV)
    kw = dict(temperature=0.5 + torch.rand(T, generator=g, device=DEV),
              top_k=torch.randint(0, 60, (T,), generator=g, device=DEV, dtype=torch.int32),
              top_p=0.3 + torch.rand(T, generator=g, device=DEV), min_p=0.01 * torch.rand(T, generator=g, device=DEV))
    check_sample(logits, u, Sampler(V)(logits, u, **kw), **kw)


def test_sample_largest_vocabulary():
    V = 1000000
    logits = randn(gen(28), 2, V)
    u = torch.tensor([0.4, 0.9], device=DEV)
    for cut in (dict(), dict(top_k=100), dict(top_p=0.7)):
        check_sample(logits, u, Sampler(V)(logits, u, **cut), **cut)


# ---- all three ------------------------------------------------------------------
def test_rows_past_32_bit_offsets():
    n = (1 << 31) + 64                                # elements between the rows: two rows pass 2^32 bytes
    buf = torch.empty(2 * n + 4096, dtype=torch.bfloat16, device=DEV)
    rows = torch.as_strided(buf, (3, 2048), (n, 1))
    src = randn(gen(30), 3, 2048).to(torch.bfloat16)
    rows.copy_(src)
    for a, b in zip(ScoredRouter(256, 8)(rows[:, :256]), ScoredRouter(256, 8)(src[:, :256].contiguous())):
        assert torch.equal(a, b)
    for a, b in zip(BlockNorm(2048)(rows, rows), BlockNorm(2048)(src, src)):
        assert torch.equal(a, b)
    u = torch.rand(3, generator=gen(31), device=DEV)
    for a, b in zip(Sampler(2048)(rows, u, top_p=0.9), Sampler(2048)(src, u, top_p=0.9)):
        assert torch.equal(a, b)
    out = torch.empty_like(src)
    BlockNorm(2048)(src, out=rows)
    BlockNorm(2048)(src, out=out)
    assert torch.equal(rows, out)


def test_no_tokens():
    e = lambda *s: torch.empty(s, device=DEV)
    assert ScoredRouter(64, 8)(e(0, 64))[0].shape == (0, 8)
    assert BlockNorm(64)(e(0, 64), e(0, 64))[0].shape == (0, 64)
    assert Sampler(64)(e(0, 64), e(0))[0].shape == (0,)


def test_python_refusals():
    x = torch.zeros(4, 64, device=DEV)
    r, n, s, u = ScoredRouter(64, 8), BlockNorm(64), Sampler(64), torch.zeros(4, device=DEV)
    for bad in (lambda: r(x[:, :63]), lambda: r(x.t()), lambda: r(x.double()), lambda: r(x[0]),
                lambda: r(x, ids=torch.zeros(4, 8, device=DEV)), lambda: r(x, w=torch.zeros(3, 8, device=DEV)),
                lambda: r(x, table=torch.zeros(63, dtype=torch.int32, device=DEV)),
                lambda: r(x[:1].expand(4, 64)), lambda: r(x, ids=torch.zeros(4, 8, dtype=torch.int32)),
                lambda: n(x, x[:3]), lambda: n(x, x.double()), lambda: n(x, gate=torch.zeros(5, device=DEV)),
                lambda: n(x, x, torch.zeros(4, 2, device=DEV)), lambda: n(x, x.view(4, 64, 1).expand(4, 64, 2)),
                lambda: n(x, residual=x.half()), lambda: n(x, out=x[:2]), lambda: n(x, out_dtype=torch.float64),
                lambda: n(x, out=x, out_dtype=torch.float16), lambda: n(x.cpu()),
                lambda: s(x, u[:3]), lambda: s(x, u.double()), lambda: s(x, u, top_k=u), lambda: s(x, u, top_p=u[:2]),
                lambda: s(x, u, top_k=1 << 40), lambda: s(x, u, min_p="0"),
                lambda: r(x, dummy=1 << 31), lambda: s(x, u, temperature=u.cpu()), lambda: s(x, u, tokens=u), lambda: s(x[:, ::2], u)):
        with pytest.raises((ValueError, _lib.MoeError)):
            bad()
    with pytest.raises(_lib.MoeError, match="branch"):
        n(x, gate=torch.zeros(64, device=DEV))
    with pytest.raises(_lib.MoeError, match="same memory"):
        n(x, x.clone(), out=x, residual=x)


@pytest.mark.parametrize("B", [1, 5, 80])
@pytest.mark.parametrize("cpu", [False, True])
def test_decode_batch_of_scored_layers(B, cpu):
    # a cache with one layer routed by scores and one by softmax: the same bits as the calls it is made of
    from gpu_rig import Rig
    from moe_prefetch.batched import BatchedMoe
    E, K = 128, 8
    rig = Rig([40, 128], [_lib.TYPE_Q4K, _lib.TYPE_Q6K], T=B, steer=False, admit="window", batch_tables=True)
    bias = 0.02 * randn(gen(41), E)
    router = ScoredRouter(E, K, score="sigmoid", bias=bias, n_groups=8, top_groups=4, group_best=2, scale=2.5)
    st = torch.cuda.current_stream().cuda_stream
    try:
        if cpu:
            rig.cache.set_sidecar(4, (1, 2))
        rig.cache.set_scoring(0, router)
        x = rig.x.transpose(0, 1).contiguous()
        out = torch.empty((2, B, 2048), device=DEV)
        with pytest.raises(_lib.MoeError, match="moe_decode_batch"):
            rig.cache.decode_token(x[:, 0].contiguous(), out[:, 0].contiguous(), stream=st)
        with pytest.raises(_lib.MoeError, match="moe_decode_batch"):
            rig.cache.decode_layer(1, x[1, 0], out[1, 0], stream=st)
        for rep in range(3):                          # the slots change between the steps, the outputs do not
            ids = rig.cache.decode_batch(x, out, stream=st)
            torch.cuda.synchronize()
            for l in range(2):
                m, want = BatchedMoe(B), torch.empty((B, 2048), device=DEV)
                m.forward(x[l], want, rig.stores[l].dev, rig.eb[l], E, rig.down_types[l], W=rig.W[l], xf32=x[l],
                          router=router if l == 0 else None, stream=st)
                torch.cuda.synchronize()
                assert np.array_equal(ids[l], m.ids[:B].cpu().numpy()), (rep, l)
                assert torch.equal(out[l], want), (rep, l)
            bias += 0.01 * randn(gen(42 + rep), E)    # balancing in place reaches the cache's next call
            torch.cuda.synchronize()
        rig.cache.set_scoring(0, None)
        rig.cache.decode_token(x[:, 0].contiguous(), out[:, 0].contiguous(), stream=st)
    finally:
        rig.close()


def test_a_decode_step_of_all_of_them():
    # two layers and the next token for a batch: norm, scored routing, expert products, the rows' sum with post-norm,
    # gate and residual, the next norm, logits, sampling; every step against its definition, then captured and replayed
    from gpu_rig import Pinned, synth_experts_dev
    from moe_prefetch.batched import BatchedMoe
    B, E, K, H, V, eb = 6, 64, 6, 2048, 5003, _lib.lib().moe_expert_bytes(2048, 256, _lib.TYPE_Q4K)
    g = gen(50)
    stores = [torch.empty(E * eb, dtype=torch.uint8, device=DEV) for _ in range(2)]
    for l in range(2):
        synth_experts_dev(7, l, 0, E, 256, _lib.TYPE_Q4K, stores[l].data_ptr(), eb)
    torch.cuda.synchronize()
    wt = lambda: (1.0 + 0.1 * randn(g, H)).to(torch.bfloat16)
    bf = torch.bfloat16
    Wr = [0.02 * randn(g, E, H) for _ in range(2)]
    head = (0.03 * randn(g, V, H)).to(bf)
    bias = 0.05 * randn(g, E)
    w_in, w_mid, w_post, w_out = wt(), wt(), wt(), wt()
    first = BlockNorm(H, weight=w_in)
    between = [BlockNorm(H, weight=w, post_weight=w_post, scale=0.5, gate_act="sigmoid") for w in (w_mid, w_out)]
    router = ScoredRouter(E, K, score="sigmoid", bias=bias, n_groups=4, top_groups=2, group_best=2, scale=2.0)
    sampler = Sampler(V)
    moe = BatchedMoe(B, n_experts=E, n_expert_used=K, intermediate=256)
    x = randn(g, B, H).to(bf)
    gate = randn(g, B)
    u = torch.rand(B, generator=g, device=DEV)
    pairs = [torch.empty(B, K, H, device=DEV) for _ in range(2)]
    scratch = torch.empty(B, H, device=DEV)

    def step(keep=None):
        r, (y, _) = x, first(x)
        for l in range(2):
            st = torch.cuda.current_stream().cuda_stream
            logits = y.float() @ Wr[l].t()
            moe.route(B, logits=logits, router=router, stream=st)
            moe.dispatch(B, stream=st)
            moe.experts(y, scratch, B, stores[l].data_ptr(), eb, E, _lib.TYPE_Q4K, pair_out=pairs[l], stream=st)
            was = r
            y, r = between[l](r, pairs[l], gate)
            if keep is not None:
                torch.cuda.synchronize()
                check_route(logits, (moe.ids, moe.w), K=K, score="sigmoid", bias=np64(bias), n_groups=4, top_groups=2,
                            group_best=2, scale=2.0)
                check_norm("bf16", was, (y, r), branch=pairs[l], gate=gate, weight=(w_mid, w_out)[l], post_weight=w_post,
                           post=True, scale=0.5, gate_act="sigmoid")
        lm = (y @ head.t()).float()
        tokens, probs = sampler(lm, u, temperature=0.8, top_k=50, top_p=0.9, min_p=0.02)
        if keep is not None:
            check_sample(lm, u, (tokens, probs), temperature=0.8, top_k=50, top_p=0.9, min_p=0.02)
        return tokens, probs, r

    step(keep=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        x.copy_(randn(g, B, H))
        u.copy_(torch.rand(B, generator=g, device=DEV))
        graph.replay()
        have = [t.clone() for t in got]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(have, want)), i


def test_streams_and_two_calls_at_once():
    g = gen(32)
    logits, x = randn(g, 300, 256), randn(g, 300, 2048)
    voc, u = randn(g, 300, 5000), torch.rand(300, generator=g, device=DEV)
    router, norm, sampler = ScoredRouter(256, 8, score="sigmoid"), BlockNorm(2048, scale=0.5), Sampler(5000)
    run = lambda **kw: (*router(logits, **kw), *norm(x, x, **kw), *sampler(voc, u, top_p=0.8, **kw))
    want = run()
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    outs = [run(stream=a), run(stream=b.cuda_stream), run(stream=a), run(stream=b), run(stream=0)]
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(p, q) for p, q in zip(o, want))


def test_graph_replays():
    g = gen(33)
    logits, x = randn(g, 33, 128), randn(g, 33, 2048).to(torch.bfloat16)
    voc, u = 2.0 * randn(g, 33, 32003), torch.rand(33, generator=g, device=DEV)
    rows = randn(g, 33, 8, 2048)
    router, norm, sampler = ScoredRouter(128, 8), BlockNorm(2048), Sampler(32003)
    run = lambda: (*router(logits), *norm(x, rows), *sampler(voc, u, temperature=0.9, top_k=64, top_p=0.95))
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for i in range(4):
        logits.copy_(randn(g, 33, 128))
        rows.copy_(randn(g, 33, 8, 2048))
        voc.copy_(2.0 * randn(g, 33, 32003))
        u.copy_(torch.rand(33, generator=g, device=DEV))
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(outs, want)), i


def test_two_graphs_of_the_same_objects():
    g = gen(34)
    logits, x, voc = randn(g, 9, 128), randn(g, 9, 2048), randn(g, 9, 32003)
    u = torch.rand(9, generator=g, device=DEV)
    router, norm, sampler = ScoredRouter(128, 8), BlockNorm(2048), Sampler(32003)
    runs = [lambda: (*router(logits), *norm(x, x), *sampler(voc, u, top_p=0.95)),
            lambda: (*router(logits[:5]), *norm(x[:5]), *sampler(voc[:5], u[:5], top_k=500))]
    graphs, outs = [], []
    for r in runs:
        r()
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(r())
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for i in range(4):
        logits.copy_(randn(g, 9, 128))
        voc.copy_(randn(g, 9, 32003))
        torch.cuda.synchronize()
        with torch.cuda.stream(a):
            graphs[0].replay()
        with torch.cuda.stream(b):
            graphs[1].replay()
        torch.cuda.synchronize()
        for r, o in zip(runs, outs):
            assert all(torch.equal(p, q) for p, q in zip(o, r())), i
