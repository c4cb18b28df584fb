"""Refusals and empty calls of moe_route_scored, moe_block_norm and moe_sample and of their Python classes: host code
only, no GPU."""
import ctypes
import os
import subprocess

import pytest
import torch

import moe_prefetch
from moe_prefetch import MoeError, _lib
from moe_prefetch.block import BlockNorm, Sampler, ScoredRouter

L = moe_prefetch.lib()
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PTR = 4096                                            # an aligned address that no refused call reads


def scored(**kw):
    d = dict(logits=PTR, logits_stride=64, logits_type=0, n_tok=2, E=64, K=6, score=0, renormalize=1, n_groups=1,
             top_groups=1, group_best=1, scale=1.0, ids=PTR, w=PTR)
    d.update(kw)
    return L.moe_route_scored(ctypes.byref(_lib.RouteScoredDesc(**d)), None)


@pytest.mark.parametrize("bad", [
    dict(E=0), dict(E=1025), dict(K=0), dict(K=65), dict(E=5, K=6), dict(score=2), dict(n_groups=0), dict(n_groups=65),
    dict(n_groups=5), dict(top_groups=0), dict(top_groups=2), dict(n_groups=16, top_groups=1), dict(group_best=0),
    dict(group_best=3), dict(n_groups=64, top_groups=64, group_best=2), dict(scale=float("inf")),
    dict(scale=float("nan")), dict(n_tok=-1), dict(n_tok=(1 << 20) + 1), dict(logits_type=3), dict(logits=None), dict(ids=None),
    dict(logits=None, W=PTR, x=PTR, H=2048), dict(logits=None, W=PTR, x=PTR + 8, H=2048, workspace=PTR),
    dict(logits=None, W=PTR, x=PTR, H=1024, workspace=PTR), dict(logits=None, W=PTR, x=PTR, H=2048, workspace=PTR, E=72),
    dict(logits=None, W=PTR, x=PTR, H=2048, workspace=PTR, n_tok=65536), dict(w=None),
    dict(logits_stride=63), dict(logits=PTR + 2), dict(logits_type=1, logits=PTR + 1), dict(ids=PTR + 2),
    dict(bias=PTR + 1), dict(table=PTR + 2), dict(slots=PTR + 3), dict(scores=PTR + 1)])
def test_scored_refusals(bad):
    assert scored(**bad) == _lib.MOE_ERR_ARG
    assert any(w in L.moe_last_error() for w in (b"moe_route_scored", b"hidden size", b"n_experts"))


def norm(**kw):
    d = dict(n_tok=2, H=128, kind=0, x=PTR, x_stride=128, x_type=1, branch=2 * PTR, branch_stride=128, branch_type=0,
             n_sum=1, scale=1.0, eps=1e-6, post_eps=1e-6, residual=3 * PTR, residual_stride=128, y=4 * PTR,
             y_stride=128, y_type=1)
    d.update(kw)
    return L.moe_block_norm(ctypes.byref(_lib.BlockNormDesc(**d)), None)


@pytest.mark.parametrize("bad", [
    dict(n_tok=-1), dict(n_tok=(1 << 20) + 1), dict(H=0), dict(H=16385), dict(kind=2), dict(x_type=3), dict(branch_type=2), dict(gate_type=2),
    dict(weight_type=2), dict(y_type=2), dict(gate_act=2), dict(gate_col_stride=2), dict(eps=-1.0),
    dict(eps=float("nan")), dict(post_eps=-1.0), dict(scale=float("inf")), dict(weight_offset=float("nan")),
    dict(branch=None, gate=PTR), dict(branch=None, post=1), dict(n_sum=0), dict(n_sum=65), dict(post_weight=PTR),
    dict(x=None), dict(residual=None, y=None), dict(residual=4 * PTR), dict(residual=PTR, residual_stride=256),
    dict(y=PTR, y_type=0), dict(x_stride=127), dict(branch_stride=1), dict(residual_stride=127), dict(y_stride=0),
    dict(gate=PTR, gate_row_stride=-1), dict(gate=PTR, gate_row_stride=64, gate_col_stride=1), dict(x=PTR + 1),
    dict(branch=PTR + 2), dict(gate=PTR + 2), dict(weight=PTR + 2), dict(bias=PTR + 2),
    dict(post=1, post_weight=PTR + 2), dict(residual=PTR + 129), dict(y=PTR + 1)])
def test_norm_refusals(bad):
    assert norm(**bad) == _lib.MOE_ERR_ARG
    assert b"moe_block_norm" in L.moe_last_error()


def sample(**kw):
    d = dict(logits=PTR, logits_stride=100, logits_type=0, n_tok=2, V=100, u=PTR, temperature_all=1.0, top_p_all=1.0,
             tokens=PTR, workspace=PTR)
    d.update(kw)
    return L.moe_sample(ctypes.byref(_lib.SampleDesc(**d)), None)


@pytest.mark.parametrize("bad", [
    dict(n_tok=-1), dict(n_tok=65536), dict(V=0), dict(V=1000001), dict(logits_type=-1), dict(logits=None), dict(u=None),
    dict(tokens=None), dict(logits_stride=99), dict(logits=PTR + 2), dict(logits_type=2, logits=PTR + 1),
    dict(u=PTR + 1), dict(temperature=PTR + 2), dict(top_k=PTR + 2), dict(top_p=PTR + 2), dict(min_p=PTR + 2),
    dict(tokens=PTR + 2), dict(probs=PTR + 2), dict(workspace=None), dict(workspace=PTR + 4)])
def test_sample_refusals(bad):
    assert sample(**bad) == _lib.MOE_ERR_ARG
    assert b"moe_sample" in L.moe_last_error()


def test_null_descriptors():
    assert L.moe_route_scored(None, None) == L.moe_block_norm(None, None) == L.moe_sample(None, None) == _lib.MOE_ERR_ARG


def test_no_tokens_is_done_without_a_gpu():
    assert scored(n_tok=0, logits=None, ids=None, w=None) == _lib.MOE_OK
    assert norm(n_tok=0, x=None, residual=None, y=None) == _lib.MOE_OK
    assert sample(n_tok=0, logits=None, u=None, tokens=None) == _lib.MOE_OK


@pytest.mark.parametrize("name, struct", [("moe_route_scored_desc", _lib.RouteScoredDesc),
                                          ("moe_block_norm_desc", _lib.BlockNormDesc),
                                          ("moe_sample_desc", _lib.SampleDesc)])
def test_descriptors_match_the_header(tmp_path, name, struct):
    fields = [f for f, _ in struct._fields_]
    src = tmp_path / "offsets.c"
    src.write_text('#include <stdio.h>\n#include "moe_prefetch.h"\nint main(void) {\n' +
                   "".join(f'    printf("%zu ", offsetof({name}, {f}));\n' for f in fields) +
                   f'    printf("%zu", sizeof({name}));\n    return 0;\n}}\n')
    exe = str(tmp_path / "offsets")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    want = [int(v) for v in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    assert [getattr(struct, f).offset for f in fields] + [ctypes.sizeof(struct)] == want


@pytest.mark.parametrize("struct", [_lib.RouteScoredDesc, _lib.BlockNormDesc, _lib.SampleDesc])
def test_packed_descriptors(struct):
    pack, place = _lib.packed(struct)
    values = [7 * i + 3 for i in range(len(place))]
    d = struct.from_buffer_copy(pack(*values))
    assert [getattr(d, n) for n in place] == values


def test_rules_are_refused_where_they_are_made():
    with pytest.raises(MoeError, match="n_experts"):
        ScoredRouter(2000, 8)
    with pytest.raises(MoeError, match="n_groups"):
        ScoredRouter(64, 8, n_groups=7)
    with pytest.raises(MoeError, match="top_groups"):
        ScoredRouter(64, 9, n_groups=8, top_groups=1)
    with pytest.raises(ValueError, match="score"):
        ScoredRouter(64, 8, score="tanh")
    with pytest.raises(ValueError, match="bias"):
        ScoredRouter(64, 8, bias=torch.zeros(63))
    with pytest.raises(MoeError, match="hidden"):
        BlockNorm(20000)
    with pytest.raises(ValueError, match="kind"):
        BlockNorm(64, kind="batch")
    with pytest.raises(ValueError, match="gate_act"):
        BlockNorm(64, gate_act="relu")
    with pytest.raises(ValueError, match="dtype"):
        BlockNorm(64, weight=torch.ones(64), post_weight=torch.ones(64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="post-norm"):
        BlockNorm(64, post_weight=torch.ones(64), post=False)
    with pytest.raises(MoeError, match="vocabulary"):
        Sampler(1 << 21)


def test_scoring_of_a_cache():
    from moe_prefetch import MoeCache
    c = MoeCache(2, n_experts=128, intermediate=768, n_slots=16, device=-1)
    try:
        rule = ScoredRouter(128, 8, score="sigmoid", n_groups=8, top_groups=4, group_best=2, scale=2.5)
        c.set_scoring(1, rule)
        c.set_scoring(1, None)
        with pytest.raises(MoeError, match="the cache 8 of 128"):
            c.set_scoring(0, ScoredRouter(64, 8))
        with pytest.raises(MoeError, match="the cache 8 of 128"):
            c.set_scoring(0, ScoredRouter(128, 6))
        with pytest.raises(MoeError, match="bad arguments"):
            c.set_scoring(2, rule)
        bad = rule.rule()
        bad.n_groups = 7
        assert L.moe_cache_set_scoring(c.h, 0, ctypes.byref(bad)) == _lib.MOE_ERR_ARG
        bad = rule.rule()
        bad.bias = PTR + 2
        assert L.moe_cache_set_scoring(c.h, 0, ctypes.byref(bad)) == _lib.MOE_ERR_ARG
        assert L.moe_cache_set_scoring(None, 0, ctypes.byref(bad)) == _lib.MOE_ERR_ARG
    finally:
        c.close()
    c = MoeCache(1, n_experts=128, intermediate=768, n_slots=16, device=-1, cache_prior=0.01)
    try:
        with pytest.raises(MoeError, match="prior"):
            c.set_scoring(0, rule)
    finally:
        c.close()


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="GPU"):
        ScoredRouter(64, 8)(torch.zeros(2, 64))
    with pytest.raises(ValueError, match="GPU"):
        BlockNorm(64)(torch.zeros(2, 64))
    with pytest.raises(ValueError, match="GPU"):
        Sampler(64)(torch.zeros(2, 64), torch.zeros(2))
