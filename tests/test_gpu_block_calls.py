"""Calls of moe_route_scored, moe_block_norm, moe_sample and of the paths around them that tests/test_gpu_block.py
does not make."""
import ctypes

import numpy as np
import pytest
import torch

import block_examples as X
import block_ref as R
from moe_prefetch import MoeCache, _lib
from moe_prefetch.block import BlockNorm, Sampler, ScoredRouter

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def np64(t):
    return t.double().cpu().numpy()


def f32(v):
    return None if v is None else torch.tensor(v, dtype=torch.float32, device=DEV)


# ---- examples worked by hand ----------------------------------------------------------
# The logits are logarithms below 2.1 in size, rounded to f32 (2^-24 of that, twice as much at temperature 1/2): a mass is
# off by 5 x 2^-24 of itself at most, a ratio of two sums of them by 10 x 2^-24, and the result is rounded once.
@pytest.mark.parametrize("logits, K, rule, ids, w", X.ROUTE)
def test_route_examples(logits, K, rule, ids, w):
    got = ScoredRouter(len(logits), K, **{**rule, "bias": f32(rule.get("bias"))})(f32([logits]))
    assert got[0][0].tolist() == ids
    np.testing.assert_allclose(np64(got[1][0]), w, rtol=11 * 2.0 ** -24, atol=0)


# (at most six roundings on the way from the inputs, which are exact, to r; twelve more to y, whose difference from the
# mean may be an eighth of r: 8 x 6 + 12)
@pytest.mark.parametrize("x, rows, gate, rule, y, r", X.NORM)
def test_norm_examples(x, rows, gate, rule, y, r):
    weights = {k: f32(rule.get(k)) for k in ("weight", "bias", "post_weight", "post_bias")}
    got = BlockNorm(len(x), **{**rule, **weights, "eps": 0.0})(f32([x]), None if rows is None else f32([rows]), f32(gate)
                                                               if rows is not None else None)
    np.testing.assert_allclose(np64(got[0][0]), y, rtol=60 * 2.0 ** -24, atol=0)
    np.testing.assert_allclose(np64(got[1][0]), x if r is None else r, rtol=6 * 2.0 ** -24, atol=0)


@pytest.mark.parametrize("logits, u, rule, token, prob", X.SAMPLE)
def test_sample_examples(logits, u, rule, token, prob):
    got = Sampler(len(logits))(f32([logits]), f32([u]), **rule)
    assert got[0].item() == token
    np.testing.assert_allclose(got[1].item(), prob, rtol=11 * 2.0 ** -24, atol=0)


# ---- a cache's scoring rule ---------------------------------------------------------
def test_a_cache_refuses_a_bias_that_its_gpu_cannot_read():
    c = MoeCache(1, n_experts=128, intermediate=768, n_slots=16)
    try:
        router = ScoredRouter(128, 8, score="sigmoid", bias=torch.zeros(128, device=DEV))
        c.set_scoring(0, router)
        on_host = np.zeros(128, np.float32)
        rule = router.rule()
        rule.bias = on_host.ctypes.data
        assert _lib.lib().moe_cache_set_scoring(c.h, 0, ctypes.byref(rule)) == _lib.MOE_ERR_ARG
        assert b"moe_cache_set_scoring" in _lib.lib().moe_last_error()
        with pytest.raises(ValueError, match="bias"):
            router.bias = torch.zeros(128)
            c.set_scoring(0, router)
        # the refusal leaves nothing behind for the next launch to report
        router.bias = torch.zeros(128, device=DEV)
        logits = randn(gen(1), 5, 128)
        ids, w = router(logits)
        want = R.route(np64(logits), 8, score="sigmoid", bias=np.zeros(128))
        assert np.array_equal(ids.cpu().numpy(), want[0])
    finally:
        c.close()


def test_a_cache_reads_the_bias_it_was_given():
    # the router gets another bias, and the first one's memory is offered to others: the cache still reads the first
    from gpu_rig import Rig
    from moe_prefetch.batched import BatchedMoe
    B, E = 5, 128
    rig = Rig([40], [_lib.TYPE_Q4K], T=B, steer=False, admit="window", batch_tables=True)
    try:
        bias = 0.05 * randn(gen(2), E)
        router = ScoredRouter(E, 8, score="sigmoid", bias=bias.clone())
        rig.cache.set_scoring(0, router)
        router.bias = torch.zeros(E, device=DEV)
        others = [torch.full((E,), 9.0 - i, device=DEV) for i in range(64)]
        x = rig.x.transpose(0, 1).contiguous()
        out = torch.empty((1, B, 2048), device=DEV)
        torch.cuda.synchronize()
        ids = rig.cache.decode_batch(x, out, stream=torch.cuda.current_stream().cuda_stream)
        m = BatchedMoe(B)
        m.route(B, W=rig.W[0], x=x[0], router=ScoredRouter(E, 8, score="sigmoid", bias=bias))
        torch.cuda.synchronize()
        assert np.array_equal(ids[0], m.ids.cpu().numpy())
        del others
    finally:
        rig.close()


def test_the_one_token_paths_come_back_with_the_last_scored_layer():
    from gpu_rig import Rig
    rig = Rig([40, 40], [_lib.TYPE_Q4K, _lib.TYPE_Q4K], T=1, steer=False, admit="window")
    st = torch.cuda.current_stream().cuda_stream
    x = rig.x.transpose(0, 1)[:, 0].contiguous()
    out, want = torch.empty_like(x), torch.empty_like(x)
    router = ScoredRouter(128, 8)
    try:
        def decodes():
            try:
                rig.cache.decode_token(x, out, stream=st)
            except _lib.MoeError as e:
                assert "moe_decode_batch" in str(e)
                with pytest.raises(_lib.MoeError, match="moe_decode_batch"):
                    rig.cache.decode_layer(0, x[0], out[0], stream=st)
                return False
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            return True
        rig.cache.decode_token(x, want, stream=st)
        torch.cuda.synchronize()
        for layer, rule, scored in ((0, None, 0), (0, router, 1), (0, router, 1), (1, router, 2), (0, None, 1), (0, None, 1),
                                    (1, router, 1), (1, None, 0), (1, None, 0), (1, router, 1), (1, None, 0)):
            rig.cache.set_scoring(layer, rule)
            assert decodes() == (scored == 0), (layer, rule is not None)
        with pytest.raises(_lib.MoeError):
            rig.cache.set_scoring(0, ScoredRouter(128, 6))            # refused: counts for nothing
        assert decodes()
    finally:
        rig.close()


# ---- a row and its batch ------------------------------------------------------------
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [30011, 901])
def test_a_row_gives_the_same_bits_in_any_batch(V, dt):
    # a row copied to the same place in 16 bytes, alone and among others: odd rows next to each other begin at every place
    T, g = 64, gen(3)
    logits = ((0.3 + 2.0 * torch.rand(T, 1, generator=g, device=DEV)) * randn(g, T, V)).to(dt)
    u = torch.rand(T, generator=g, device=DEV)
    rows = list(range(0, T, 5)) + [T - 1]
    where = [logits[t].data_ptr() % 16 // logits.element_size() for t in rows]
    assert len(set(where)) == 16 // logits.element_size()
    for cut in (dict(), dict(top_k=300), dict(top_k=1000, top_p=0.7), dict(top_k=20000, min_p=0.01), dict(top_p=0.9),
                dict(temperature=3.0), dict(temperature=0.0)):
        want = Sampler(V)(logits, u, **cut)
        for t, m in zip(rows, where):
            for n, i in ((1, 0), (7, 3)):
                ld = (V + 31) // 16 * 16
                batch = randn(g, n, ld).to(dt)[:, m:m + V]
                batch[i] = logits[t]
                assert batch[i].data_ptr() % 16 == logits[t].data_ptr() % 16
                got = Sampler(V)(batch, u[t:t + 1].expand(n).contiguous(), **cut)
                assert got[0][i] == want[0][t] and got[1][i] == want[1][t], (cut, t, n)


# ---- bounds of the kernels' own arithmetic ----------------------------------------------
@pytest.mark.parametrize("H", [2048, 2047, 8192, 8191, 16384, 16383])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_norm_within_the_kernels_own_sums(kind, H, monkeypatch):
    # a sum over a row is a chain of at most 16 terms a thread, six steps of a wave and 16 waves: 38 roundings
    unit = R._unit
    monkeypatch.setattr(R, "_unit", lambda *a: unit(*a[:-1], 38))
    g = gen(4)
    x, b = 2.0 * randn(g, 3, H) + 0.3, randn(g, 3, 2, H)
    kw = dict(weight=1.0 + 0.2 * randn(g, H), bias=randn(g, H), post_weight=1.0 + 0.2 * randn(g, H), post_bias=randn(g, H),
              kind=kind, scale=0.3)
    got = BlockNorm(H, **kw)(x, b)
    y, r, e_y, e_r = R.block_norm(np64(x), np64(b), post=True, **{k: np64(v) if torch.is_tensor(v) else v for k, v in kw.items()})
    for t, want, err in ((got[0], y, e_y), (got[1], r, e_r)):
        assert (np.abs(np64(t) - want) <= err + R.U * (np.abs(want) + err)).all()


@pytest.mark.parametrize("T, V", [(3, 1000000), (5, 151936), (9, 32003), (9, 1000)])
@pytest.mark.parametrize("spread", [0.3, 2.0])
def test_sample_probabilities_to_half_a_step(T, V, spread):
    # a mass is a 64-bit number, or an integer of which the row's whole has 62 bits: half of one a token, V 2^-62 of the
    # sum (kept tokens are the largest).  Sums in 64 bits, here and in the reference, V 2^-53 each.  The result is rounded once.
    g = gen(V + T)
    logits = spread * randn(g, T, V)
    u = torch.rand(T, generator=g, device=DEV)
    for cut in (dict(), dict(top_p=0.9), dict(min_p=0.2), dict(temperature=2.0, top_p=0.5), dict(top_k=60)):
        tokens, probs = R.sample(np64(logits), np64(u), **cut)
        got = Sampler(V)(logits, u, **cut)
        np.testing.assert_array_equal(got[0].cpu().numpy(), tokens)
        np.testing.assert_allclose(np64(got[1]), probs, rtol=R.U * 1.001 + V * (2.0 ** -62 + 2.0 ** -52), atol=0)


def test_a_norm_reads_the_memory_it_was_given():
    # a parameter's data is exchanged and its first memory offered to others: the norm still reads that
    H, g = 2048, gen(5)
    first = 1.0 + 0.2 * randn(g, H)
    p = torch.nn.Parameter(first.clone())
    norm = BlockNorm(H, weight=p)
    p.data = torch.zeros(H, device=DEV)
    others = [torch.full((H,), 9.0 - i, device=DEV) for i in range(64)]
    x = randn(g, 7, H)
    assert torch.equal(norm(x)[0], BlockNorm(H, weight=first)(x)[0])
    norm.weights[0].zero_()                           # a change in place reaches it
    assert (norm(x)[0] == 0).all()
    del others
