"""moe_fp8_layer of up to nine pairs, where down and the sum over a token's experts are one launch for eight of them at most, and of 31 to 34, where
gate and up change their kernel; against 64 bits within tests/fp8_ref.py's bounds of f32 sums."""
import pytest
import torch

import fp8_ref as R
from test_gpu_fp8 import DEV, DT, gen, moe, np64, randn, vals, within

pytestmark = pytest.mark.gpu


def check(x, ids, w, up, gate, down, out, dt):
    f = lambda q: (vals(q[0]), np64(q[1]))
    want, err = R.layer(np64(x), ids.cpu().numpy(), np64(w), f(gate), f(up), f(down))
    within(np64(out), want, R.out_bound(want, err, dt))


@pytest.mark.parametrize("T, K", [(1, 3), (1, 5), (5, 1), (3, 2), (2, 3), (7, 1), (1, 7), (1, 8), (2, 4), (4, 2), (8, 1), (9, 1), (3, 3), (1, 9)])
@pytest.mark.parametrize("mode", ["any", "one", "twice", "outside", "none"])
@pytest.mark.parametrize("H, I, dt", [(272, 200, "f32"), (130, 1000, "bf16"), (300, 5120, "f16")])
def test_few_pairs(T, K, mode, H, I, dt):
    # every pair on one expert; an expert twice for a token; ids outside the experts; none inside.  Of 5,120 wide h LDS holds ten rows
    g = gen(10 * T + K + H)
    E = 11
    m, up, gate, down = moe(g, E, 0, H, I)
    x = randn(g, T, H).to(DT[dt])
    ids = torch.randint(0, E, (T, K), generator=g, device=DEV, dtype=torch.int32)
    w = randn(g, T, K)
    if mode == "one":
        ids[:] = E - 1
    elif mode == "twice":
        ids[:] = ids[:, :1]
    elif mode == "outside":
        ids.view(-1)[::2] = torch.tensor([-1, E, 2 ** 31 - 1, -2 ** 31, 256], dtype=torch.int32, device=DEV)[:(T * K + 1) // 2]
    elif mode == "none":
        ids[:] = -1
    out = m(x, ids=ids, w=w)[0]
    check(x, ids, w, up, gate, down, out, dt)
    if mode == "none":
        assert bool((out == 0).all())


@pytest.mark.parametrize("T, K", [(1, 8), (2, 4), (8, 1)])
def test_the_most_pairs_that_lds_holds(T, K):
    # rows of 6,400 fit eight times, of 6,800 seven
    for I in (6400, 6800):
        g = gen(T + I)
        m, up, gate, down = moe(g, 9, 0, 48, I)
        x, w = randn(g, T, 48), randn(g, T, K)
        ids = torch.randint(0, 9, (T, K), generator=g, device=DEV, dtype=torch.int32)
        check(x, ids, w, up, gate, down, m(x, ids=ids, w=w)[0], "f32")


@pytest.mark.parametrize("T, K", [(31, 1), (16, 2), (33, 1), (17, 2), (64, 1), (13, 5)])
@pytest.mark.parametrize("E", [3, 20, 100])
def test_gate_and_up_where_the_kernel_changes(T, K, E):
    g, K = gen(T + E), min(K, E)
    m, up, gate, down = moe(g, E, K, 400, 144)
    x, logits = randn(g, T, 400).to(torch.bfloat16), randn(g, T, E)
    out, ids, w = m(x, logits)
    check(x, ids, w, up, gate, down, out, "bf16")
