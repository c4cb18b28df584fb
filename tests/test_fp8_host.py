"""Refusals and empty calls of moe_fp8_quantize, moe_fp8_product and moe_fp8_layer and of their Python classes, and what these
hand to the library: host code only, no GPU.  OnGpu stands for a tensor of a GPU: its address is never read."""
import ctypes

import pytest
import torch

import moe_prefetch
from moe_prefetch import MoeError, _lib
from moe_prefetch import fp8 as M
from moe_prefetch.block import ScoredRouter
from moe_prefetch.fp8 import Fp8Linear, Fp8Moe, fp8_quantize
from test_block_calls_host import OnGpu

L = moe_prefetch.lib()
PTR = 4096                                            # an aligned address that no refused call reads
F8, F32, BF16, I32 = torch.float8_e4m3fn, torch.float32, torch.bfloat16, torch.int32


def quantize(**kw):
    d = dict(x=PTR, x_stride=300, x_type=1, rows=1, n_tok=2, K=300, q=PTR + 1, q_stride=300, scale=PTR, scale_stride=3)
    d.update(kw)
    return L.moe_fp8_quantize(ctypes.byref(_lib.Fp8QuantizeDesc(**d)), None)


@pytest.mark.parametrize("bad", [
    dict(n_tok=-1), dict(n_tok=(1 << 20) + 1), dict(K=0), dict(K=(1 << 18) + 1), dict(x_type=3), dict(x_type=-1), dict(rows=0),
    dict(rows=64), dict(x=None), dict(q=None), dict(scale=None), dict(x_stride=299), dict(q_stride=299), dict(scale_stride=2),
    dict(x=PTR + 1), dict(x_type=0, x=PTR + 2), dict(scale=PTR + 2)])
def test_quantize_refusals(bad):
    assert quantize(**bad) == _lib.MOE_ERR_ARG
    assert b"moe_fp8_quantize" in L.moe_last_error()


def weight(name, n, k, **kw):
    d = {name: PTR + 3, name + "_stride": k, name + "_expert": n * k, name + "_scale": PTR, name + "_scale_stride": -(-k // 128),
         name + "_scale_expert": 64}
    d.update({name + key: v for key, v in kw.items()})
    return d


def product(**kw):
    d = dict(x=PTR, x_stride=300, x_type=1, n_tok=20, N=200, K=300, y=PTR, y_stride=200, y_type=1, workspace=PTR)
    d.update(weight("weight", 200, 300))
    d.update(kw)
    return L.moe_fp8_product(ctypes.byref(_lib.Fp8ProductDesc(**d)), None)


@pytest.mark.parametrize("bad", [
    dict(n_tok=-1), dict(n_tok=(1 << 20) + 1), dict(N=0), dict(N=(1 << 18) + 1), dict(K=0), dict(K=(1 << 18) + 1), dict(x_type=4),
    dict(y_type=3), dict(x=None), dict(y=None), dict(weight=None), dict(weight_scale=None), dict(weight_stride=299),
    dict(weight_stride=-300), dict(weight_scale_stride=2), dict(weight_scale_stride=-3), dict(weight_scale=PTR + 2), dict(x_stride=299),
    dict(y_stride=199), dict(x=PTR + 1), dict(y=PTR + 1), dict(y_type=0, y=PTR + 2), dict(workspace=None), dict(workspace=PTR + 8),
    dict(x_type=3), dict(x_type=3, x_scale=PTR, x_scale_stride=2), dict(x_type=3, x_scale=PTR + 1, x_scale_stride=3)])
def test_product_refusals(bad):
    assert product(**bad) == _lib.MOE_ERR_ARG
    assert b"moe_fp8_product" in L.moe_last_error()


def layer(route=None, **kw):
    d = dict(x=PTR, x_stride=256, x_type=1, n_tok=2, E=8, K=2, H=256, I=200, ids=PTR, w=PTR, out=PTR, out_stride=256, out_type=1,
             workspace=PTR)
    for name, n, k in (("gate", 200, 256), ("up", 200, 256), ("down", 256, 200)):
        d.update(weight(name, n, k))
    d.update(kw)
    desc = _lib.Fp8LayerDesc(**d)
    for k, v in (route or {}).items():
        setattr(desc.route, k, v)
    return L.moe_fp8_layer(ctypes.byref(desc), None)


LOGITS = dict(logits=PTR, logits_stride=8, n_groups=1, top_groups=1, group_best=1, scale=1.0)


@pytest.mark.parametrize("bad", [
    dict(n_tok=-1), dict(n_tok=32768), dict(E=0), dict(E=257), dict(K=0), dict(K=65), dict(H=0), dict(I=0), dict(H=(1 << 18) + 1),
    dict(I=(1 << 18) + 1), dict(x_type=3), dict(out_type=3), dict(gate=None), dict(up_scale=None), dict(down=None), dict(down_stride=199),
    dict(gate_stride=255), dict(up_scale_stride=1), dict(gate_expert=-1), dict(down_scale_expert=-4), dict(up_scale=PTR + 1), dict(x=None),
    dict(ids=None), dict(w=None), dict(out=None), dict(workspace=None), dict(workspace=PTR + 4), dict(x_stride=255), dict(out_stride=255),
    dict(x=PTR + 1), dict(out=PTR + 1), dict(ids=PTR + 2), dict(w=PTR + 1)])
def test_layer_refusals(bad):
    assert layer(**bad) == _lib.MOE_ERR_ARG
    assert b"moe_fp8_layer" in L.moe_last_error()


@pytest.mark.parametrize("bad", [
    dict(score=2), dict(n_groups=3), dict(n_groups=0), dict(top_groups=2), dict(group_best=3), dict(scale=float("nan")), dict(logits_type=3),
    dict(logits_stride=7), dict(logits=PTR + 2), dict(bias=PTR + 2)])
def test_layer_rule_refusals(bad):
    assert layer({**LOGITS, **bad}) == _lib.MOE_ERR_ARG
    assert b"moe_route_scored" in L.moe_last_error()


def test_more_experts_a_token_than_there_are():
    # chosen: refused by the rule; given: an id may stand twice
    assert layer(LOGITS, K=9) == _lib.MOE_ERR_ARG
    assert layer(K=9, n_tok=0) == _lib.MOE_OK


def test_calls_without_rows():
    assert quantize(n_tok=0, x=None, q=None, scale=None) == _lib.MOE_OK
    assert product(n_tok=0, x=None, y=None, workspace=None) == _lib.MOE_OK
    assert layer(n_tok=0, x=None, ids=None, w=None, out=None, workspace=None) == _lib.MOE_OK
    assert layer(LOGITS, n_tok=0, x=None, ids=None, w=None, out=None, workspace=None) == _lib.MOE_OK


def test_null_descriptors():
    for call in (L.moe_fp8_quantize, L.moe_fp8_product, L.moe_fp8_layer):
        assert call(None, None) == _lib.MOE_ERR_ARG


def test_workspaces():
    assert L.moe_fp8_product_workspace_bytes(4, 100, 300, 3) == 0
    assert L.moe_fp8_product_workspace_bytes(0, 100, 300, 1) == 0
    assert L.moe_fp8_product_workspace_bytes(4, 0, 300, 1) == 0
    assert L.moe_fp8_product_workspace_bytes(16, 100, 300, 1) == 0 < L.moe_fp8_product_workspace_bytes(16, 100, 1 << 18, 1)
    assert L.moe_fp8_product_workspace_bytes(1000, 100, 300, 1) >= 1000 * (300 + 12)
    assert L.moe_fp8_layer_workspace_bytes(0, 8, 2, 256, 128) == 0
    assert L.moe_fp8_layer_workspace_bytes(32768, 8, 2, 256, 128) == 0
    assert L.moe_fp8_layer_workspace_bytes(100, 257, 2, 256, 128) == 0
    a, b = (L.moe_fp8_layer_workspace_bytes(n, 8, 2, 256, 128) for n in (1000, 2000))
    assert 0 < a < b


def test_descriptor_sizes_match_the_header():
    import os
    import subprocess
    import tempfile
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with tempfile.TemporaryDirectory() as d:
        src = os.path.join(d, "s.c")
        with open(src, "w") as f:
            f.write('#include "moe_prefetch.h"\n#include <stdio.h>\nint main(void) { printf("%zu %zu %zu %zu\\n", '
                    "sizeof(moe_fp8_quantize_desc), sizeof(moe_fp8_product_desc), sizeof(moe_fp8_layer_desc), "
                    "offsetof(moe_fp8_layer_desc, route)); }\n")
        subprocess.run(["gcc", "-I", os.path.join(root, "include"), src, "-o", os.path.join(d, "s")], check=True)
        got = [int(v) for v in subprocess.run([os.path.join(d, "s")], capture_output=True, text=True, check=True).stdout.split()]
    S = ctypes.sizeof
    assert got == [S(_lib.Fp8QuantizeDesc), S(_lib.Fp8ProductDesc), S(_lib.Fp8LayerDesc), S(_lib.Fp8LayerHead)]


# ---- the classes --------------------------------------------------------------------
def given(cls, desc):
    """The fields that the class's next calls hand to the library."""
    seen = []

    def fn(raw, stream):
        if isinstance(raw, bytes):
            seen.append((desc.from_buffer_copy(raw), stream))
        return 0
    return seen, fn


@pytest.fixture(autouse=True)
def no_gpu(monkeypatch):
    monkeypatch.setattr("moe_prefetch.block._raw_stream", lambda dev: 77)
    monkeypatch.setattr("moe_prefetch.block._device", lambda: 0)
    monkeypatch.setattr(M, "_empty", lambda shape, dtype, dev, stream: OnGpu(*shape, dtype=dtype, at=1 << 20))


def test_quantize_hands_on(monkeypatch):
    seen, fn = given(None, _lib.Fp8QuantizeDesc)
    monkeypatch.setattr(M, "_quantize", (_lib.packed(_lib.Fp8QuantizeDesc)[0], fn))
    q, s = fp8_quantize(OnGpu(5, 300, dtype=BF16))
    d, stream = seen[0]
    assert (d.x, d.x_stride, d.x_type, d.rows, d.n_tok, d.K, d.q_stride, d.scale_stride, stream) == (4096, 300, 1, 1, 5, 300, 300, 3, 77)
    assert q.shape == (5, 300) and q.dtype is F8 and s.shape == (5, 3)
    fp8_quantize(OnGpu(300, 400)[:, :130], rows=128, stream=5)
    d, stream = seen[1]
    assert (d.x_stride, d.x_type, d.rows, d.n_tok, d.K, stream) == (400, 0, 128, 300, 130, 5)
    for bad, kw in ((OnGpu(5), {}), (OnGpu(5, 6, dtype=torch.float64), {}), (OnGpu(5, 6, dtype=F8), {}), (torch.zeros(5, 6), {}),
                    (OnGpu(5, 6), dict(rows=2)), (OnGpu(5, 6), dict(q=OnGpu(5, 6))), (OnGpu(5, 6), dict(q=OnGpu(5, 5, dtype=F8))),
                    (OnGpu(5, 6), dict(scale=OnGpu(5, 2))), (OnGpu(5, 6), dict(scale=OnGpu(5, 1, dtype=BF16))),
                    (OnGpu(5, 6), dict(scale=OnGpu(5, 1, device=1))), (OnGpu(5, 12)[:, ::2], {})):
        with pytest.raises(ValueError):
            fp8_quantize(bad, **kw)
    assert len(seen) == 2


def test_linear_hands_on():
    lin = Fp8Linear(OnGpu(200, 320, dtype=F8, at=99)[:, :300], OnGpu(2, 5)[:, :3])
    seen, lin._fn = given(lin, _lib.Fp8ProductDesc)
    y = lin(OnGpu(40, 300, dtype=BF16))
    d, stream = seen[0]
    assert (d.weight, d.weight_stride, d.weight_scale_stride, d.N, d.K, d.n_tok) == (99, 320, 5, 200, 300, 40)
    assert (d.x_type, d.y_type, d.y_stride, d.workspace, stream, y.dtype) == (1, 1, 200, 1 << 20, 77, BF16)
    y = lin(OnGpu(4, 300, dtype=F8), OnGpu(4, 3, at=555))
    d = seen[1][0]
    assert (d.x_type, d.x_scale, d.x_scale_stride, d.y_type, d.workspace, y.dtype) == (3, 555, 3, 1, None, BF16)
    assert lin(OnGpu(4, 300, dtype=F8), OnGpu(4, 3), out_dtype=F32).dtype is F32
    bad = [(OnGpu(4, 299), {}), (OnGpu(4, 300, dtype=F8), {}), (OnGpu(4, 300), dict(x_scale=OnGpu(4, 3))),
           (OnGpu(4, 300, dtype=F8), dict(x_scale=OnGpu(4, 2))), (OnGpu(4, 300, dtype=F8), dict(x_scale=OnGpu(4, 3, dtype=BF16))),
           (OnGpu(4, 300, device=1), {}), (OnGpu(4, 300), dict(out=OnGpu(4, 199))), (OnGpu(4, 300), dict(out=OnGpu(4, 200, dtype=F8))),
           (OnGpu(4, 300), dict(out_dtype=F8)), (OnGpu(4, 300), dict(out=OnGpu(4, 200), out_dtype=BF16)),
           (OnGpu(4, 300, dtype=torch.int32), {}), (torch.zeros(4, 300), {})]
    for x, kw in bad:
        with pytest.raises(ValueError):
            lin(x, **kw)
    assert len(seen) == 3


@pytest.mark.parametrize("w, s", [
    (OnGpu(200, 300), OnGpu(2, 3)), (OnGpu(200, 300, dtype=F8), OnGpu(2, 2)), (OnGpu(200, 300, dtype=F8), OnGpu(2, 3, dtype=BF16)),
    (OnGpu(200, 300, dtype=F8), OnGpu(2, 3, device=1)), (OnGpu(200, 300, dtype=F8)[0], OnGpu(2, 3)),
    (OnGpu(200, 600, dtype=F8)[:, ::2], OnGpu(2, 3)), (torch.zeros(200, 300).to(F8), OnGpu(2, 3))])
def test_linear_refusals(w, s):
    with pytest.raises(ValueError):
        Fp8Linear(w, s)


def test_a_weight_too_wide_is_refused():
    with pytest.raises(MoeError, match="moe_fp8_product"):
        Fp8Linear(OnGpu(1, (1 << 18) + 1, dtype=F8), OnGpu(1, 2049))


def experts(E=8, I=200, H=256, device=0):
    return [OnGpu(*s, dtype=F8, device=device) for s in ((E, I, H), (E, I, H), (E, H, I))] + [
        OnGpu(*s, device=device) for s in ((E, 2, 2), (E, 2, 2), (E, 2, 2))]


def test_moe_hands_on():
    m = Fp8Moe(*experts(), router=ScoredRouter(8, 2, score="sigmoid", bias=OnGpu(8, at=333), scale=2.5))
    seen, m._fn = given(m, _lib.Fp8LayerDesc)
    out, ids, w = m(OnGpu(5, 256, dtype=BF16), OnGpu(5, 9, at=777)[:, :8])
    d, stream = seen[0]
    assert (d.n_tok, d.E, d.K, d.H, d.I, d.x_type, d.out_type, stream) == (5, 8, 2, 256, 200, 1, 1, 77)
    assert (d.gate_stride, d.gate_expert, d.down_stride, d.down_expert, d.up_scale_expert) == (256, 200 * 256, 200, 256 * 200, 4)
    r = d.route
    assert (r.logits, r.logits_stride, r.logits_type, r.score, r.bias, r.scale, r.renormalize) == (777, 9, 0, 1, 333, 2.5, 1)
    assert out.dtype is BF16 and ids.shape == (5, 2) and ids.dtype is I32 and w.shape == (5, 2)
    out, ids, w = m(OnGpu(5, 256), ids=OnGpu(5, 3, dtype=I32, at=11), w=OnGpu(5, 3, at=12), out_dtype=BF16)
    d = seen[1][0]
    assert (d.K, d.ids, d.w, d.route.logits, d.x_type, d.out_type) == (3, 11, 12, None, 0, 1)
    bad = [((OnGpu(5, 255), OnGpu(5, 8)), {}), ((OnGpu(5, 256), OnGpu(4, 8)), {}), ((OnGpu(5, 256), OnGpu(5, 7)), {}), ((OnGpu(5, 256),), {}),
           ((OnGpu(5, 256),), dict(ids=OnGpu(5, 2, dtype=I32))), ((OnGpu(5, 256),), dict(ids=OnGpu(5, 2), w=OnGpu(5, 2))),
           ((OnGpu(5, 256),), dict(ids=OnGpu(5, 2, dtype=I32), w=OnGpu(5, 3))), ((OnGpu(5, 256, dtype=F8), OnGpu(5, 8)), {}),
           ((OnGpu(5, 256, device=1), OnGpu(5, 8)), {}), ((OnGpu(5, 256), OnGpu(5, 8)), dict(ids=OnGpu(5, 3, dtype=I32))),
           ((OnGpu(5, 256), OnGpu(5, 8)), dict(out=OnGpu(5, 255))), ((OnGpu(5, 256), OnGpu(5, 8, dtype=torch.int32)), {}),
           ((OnGpu(5, 256), OnGpu(5, 8)), dict(out_dtype=torch.float64)), ((OnGpu(5, 256), OnGpu(8)), {})]
    for a, kw in bad:
        with pytest.raises(ValueError):
            m(*a, **kw)
    assert len(seen) == 2
    m.router = None
    with pytest.raises(ValueError, match="router"):
        m(OnGpu(5, 256), OnGpu(5, 8))


@pytest.mark.parametrize("change", [
    {0: OnGpu(8, 200, 255, dtype=F8)}, {1: OnGpu(8, 200, 256)}, {2: OnGpu(8, 200, 256, dtype=F8)}, {3: OnGpu(8, 2, 3)},
    {4: OnGpu(8, 2, 2, dtype=BF16)}, {5: OnGpu(8, 2, 2, device=1)}, {0: OnGpu(200, 256, dtype=F8)}, {1: OnGpu(7, 200, 256, dtype=F8)},
    {2: OnGpu(8, 256, 400, dtype=F8)[:, :, ::2]}])
def test_moe_refusals(change):
    t = experts()
    for i, v in change.items():
        t[i] = v
    with pytest.raises(ValueError):
        Fp8Moe(*t)


def test_moe_refuses_another_router_and_too_many_experts():
    with pytest.raises(ValueError, match="router"):
        Fp8Moe(*experts(), router=ScoredRouter(9, 2))
    with pytest.raises(MoeError, match="at most 256 experts"):
        Fp8Moe(*experts(E=257))


def test_the_names_are_the_packages():
    assert {"Fp8Linear", "Fp8Moe", "fp8_quantize"} <= set(dir(moe_prefetch))
    assert moe_prefetch.Fp8Linear is Fp8Linear and moe_prefetch.Fp8Moe is Fp8Moe and moe_prefetch.fp8_quantize is fp8_quantize
