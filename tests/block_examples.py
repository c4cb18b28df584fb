"""Worked examples of moe_route_scored, moe_block_norm and moe_sample: inputs whose answers are found by hand, for the
references of tests/block_ref.py and for the operators alike."""
import math

INF, NAN = math.inf, math.nan
ln = lambda *v: [math.log(a) if a > 0 else -INF for a in v]
logit = lambda *s: [math.log(a / (1 - a)) for a in s]

# (logits of one token, K, rule, ids, weights)
ROUTE = [
    # softmax .5 .3 .2
    (ln(5, 3, 2), 2, dict(renormalize=False), [0, 1], [0.5, 0.3]),
    (ln(5, 3, 2), 2, dict(), [0, 1], [5 / 8, 3 / 8]),
    (ln(2, 3, 5), 2, dict(scale=4.0), [2, 1], [4 * 5 / 8, 4 * 3 / 8]),
    # the bias chooses, .8 .6 .9 .2, and does not weigh: .4 and .8
    (logit(0.8, 0.6, 0.4, 0.2), 2, dict(score="sigmoid", bias=[0, 0, 0.5, 0], scale=3.0), [2, 0], [1.0, 2.0]),
    # groups by their best two, 1.4 and 1.1; by their best, .8 and .9
    (logit(0.8, 0.6, 0.4, 0.2), 2, dict(score="sigmoid", bias=[0, 0, 0.5, 0], n_groups=2, top_groups=1, group_best=2),
     [0, 1], [0.8 / 1.4, 0.6 / 1.4]),
    (logit(0.8, 0.6, 0.4, 0.2), 2, dict(score="sigmoid", bias=[0, 0, 0.5, 0], n_groups=2, top_groups=1, group_best=1),
     [2, 3], [0.4 / 0.6, 0.2 / 0.6]),
    # equal ones by the lower id; switched-off ones last, with weight 0
    ([1.0, 2.0, 2.0, 1.0], 3, dict(score="sigmoid", renormalize=False), [1, 2, 0],
     [1 / (1 + math.exp(-2)), 1 / (1 + math.exp(-2)), 1 / (1 + math.exp(-1))]),
    ([-INF, 0.0, NAN, 0.0], 3, dict(), [1, 3, 0], [0.5, 0.5, 0.0]),
    ([-INF, NAN], 2, dict(), [0, 1], [0.0, 0.0]),
]

S = math.sqrt(12.5)                                   # the root of the mean square of 3 and 4
# (x of one token, branch rows, gate, rule, y, r)
NORM = [
    ([3.0, 4.0], None, None, dict(), [3 / S, 4 / S], None),
    ([3.0, 4.0], None, None, dict(weight=[2.0, 3.0], weight_offset=1.0), [9 / S, 16 / S], None),
    ([1.0, 3.0], None, None, dict(kind="layer", weight=[2.0, 3.0], bias=[0.5, 0.25]), [-1.5, 3.25], None),
    # 2 x sigmoid(0) x (rows' sum) = (3, 2)
    ([0.0, 2.0], [[1.0, 0.0], [2.0, 2.0]], [0.0], dict(scale=2.0, gate_act="sigmoid"), [3 / S, 4 / S], [3.0, 4.0]),
    # the branch's own norm: (1, -1), times (4, 2), times a gate of (0.5, 1.5)
    ([1.0, 7.0], [[5.0, 1.0]], [[0.5, 1.5]], dict(kind="layer", post_weight=[4.0, 2.0], post=True), [-1.0, 1.0], [3.0, 4.0]),
]

# (logits of one row, u, rule, token, its probability); masses 8 4 2 1 1 at temperature 1, and their powers at others
P = ln(8, 4, 2, 1, 1)
SAMPLE = [
    (P, 0.0, dict(), 0, 8 / 16), (P, 0.51, dict(), 1, 4 / 16), (P, 0.99, dict(), 4, 1 / 16),
    (P[::-1], 0.51, dict(), 3, 4 / 16), (P, 0.9, dict(temperature=0.0), 0, 1.0),
    # temperature 1/2: 64 16 4 1 1.  It comes before the cuts: 0.9 of 86 takes two of them (of 16 it would take four)
    (P, 0.97, dict(temperature=0.5, top_p=0.9), 1, 16 / 80),
    # temperature 2: the roots.  0.7 of 8.24 takes three of them (of 16 it would take two)
    (P, 0.9, dict(temperature=2.0, top_p=0.7), 2, math.sqrt(2) / (math.sqrt(8) + 2 + math.sqrt(2))),
    # 0.3 of the first: one at temperature 1/2, all five at 2 (at temperature 1 it would be two)
    (P, 0.99, dict(temperature=0.5, min_p=0.3), 0, 1.0),
    (P, 0.99, dict(temperature=2.0, min_p=0.3), 4, 1 / (math.sqrt(8) + 2 + math.sqrt(2) + 2)),
    # top-p counts among the top-k: 8 + 4 of 14
    (P, 0.7, dict(top_k=3, top_p=0.85), 1, 4 / 12),
    (P, 0.7, dict(top_k=3), 1, 4 / 14), (P, 0.9, dict(top_k=3), 2, 2 / 14), (P, 0.99, dict(min_p=0.2), 2, 2 / 14),
    ([0.0, 0.0, 0.0, 0.0], 0.3, dict(), 1, 0.25), ([NAN, 0.0, -INF, 0.0], 0.6, dict(), 3, 0.5),
    ([NAN, -INF], 0.6, dict(), -1, 0.0),
]
