"""Routing where 32 bits come close to deciding wrongly: sums of group keys that cancel, biases of the lowest and the largest value,
scores far below one.  Against the statement in 64 bits."""
import numpy as np
import pytest

import expert_ops_oracle as eo
from test_gpu_route_experts import check, logits_of, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("G,h", [(32, 0.5), (32, 1.5), (32, 4.5), (16, 20.0), (24, 300.0)])
def test_group_sums_that_cancel(scoring, G, h):
    """Groups of two experts with biases of +h and -h: a key is rounded to a unit of h, their sum is as small as the scores."""
    keep = G // 2
    bias = h * np.where(np.arange(2 * G) % 2, -1.0, 1.0)
    check(logits_of(int(8 * h) + G, 3000, 2 * G, "f32", 0.01), 2 * keep, bias=bias, scoring=scoring, n_groups=G, topk_groups=keep, group_top=2)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_one_group_of_large_keys_among_small_ones(scoring):
    """Only some groups have keys far larger than their sums; they stay or go beside groups whose keys are exact to their last bits."""
    G, per = 16, 4
    bias = np.zeros((G, per))
    for g in (1, 4, 5, 9, 14):
        bias[g] = [37.0, -37.0, -80.0, -80.0]
    bias[7] = [3e30, -3e30, -3.2e38, -3.2e38]
    check(logits_of(12, 3000, G * per, "f32", 0.02), 8, bias=bias.reshape(-1), scoring=scoring, n_groups=G, topk_groups=8,
          group_top=2, renormalize=False)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("keep", [1, 3, 6])
@pytest.mark.parametrize("top", [1, 2])
def test_biases_of_the_lowest_and_the_largest_value(scoring, keep, top):
    """A bias of the type's lowest value is a mask that still orders: two such keys add up to less than 32 bits hold, and their group
    is still one that can stay.  The same with the largest value."""
    low, high = np.finfo(np.float32).min, np.finfo(np.float32).max
    per, E = 4, 32
    for masked in (range(4, 32), range(0, 28), range(0, 32), [0, 1, 2, 3, 9, 10, 11, 17, 18, 24]):
        bias = np.linspace(-0.1, 0.1, E)
        bias[list(masked)] = low
        check(logits_of(5, 40, E, "f32"), 4, bias=bias, scoring=scoring, n_groups=8, topk_groups=keep, group_top=top)
        bias[[2, 3, 12, 13, 14, 21]] = high
        check(logits_of(6, 40, E, "f32"), 4, bias=bias, scoring=scoring, n_groups=8, topk_groups=keep, group_top=top)


@pytest.mark.parametrize("bias", [None, "masks"])
@pytest.mark.parametrize("scoring,renorm,scale", [("sigmoid", True, 1.0), ("sigmoid", False, 1e30), ("softmax", True, 1e30), ("softmax", False, 1e25)])
def test_weights_of_scores_below_32_bits(scoring, renorm, scale, bias):
    """Selected scores that 32 bits hold with few bits or not at all: their weights, brought back by the sum or the scale, are those
    of 64 bits.  A score is off by less than 2^-45 there, so half a step of the result is all that is left."""
    import torch
    E = 40
    l = torch.full((6, E), -400.0)
    l[0, :4] = torch.tensor([-66.0, -88.5, -95.0, -101.0])
    l[1, :4] = torch.tensor([0.0, -90.25, -103.0, -110.0])
    l[2, 5:9] = torch.tensor([0.0, -60.0, -75.0, -1000.0])
    l[3, 30:] = torch.linspace(-120, -84, 10)
    l[4] = torch.linspace(-3, 3, E)
    l[5, 7] = 4.0
    l[5, 8:12] = -98.0
    b = None if bias is None else np.where(np.arange(E) % 13 == 12, np.finfo(np.float32).min, 0.0)
    sel, w, *_ = run(l.cuda(), 4, bias=b, scoring=scoring, renormalize=renorm, scale=scale)
    want, ww = eo.route(l.double().numpy(), 4, bias=b, scoring=scoring, renormalize=renorm, scale=float(np.float32(scale)))
    assert np.array_equal(sel, want)
    # Rows whose selected scores are all above 1e-30 are held in 32 bits with all their bits (row 3 of a softmax: e^-12 and more of the
    # largest): 110 roundings as in test_gpu_route_experts.check.  The others are done in 64.
    _, scores = eo.route(l.double().numpy(), 4, bias=b, scoring=scoring, renormalize=False)
    small = scores.min(axis=1) < 1e-30
    assert small[[1, 2, 5]].all() and not small[4]
    eo.close(w[small], ww[small], 2.0 ** -45 * ww[small], "f32")
    eo.close(w[~small], ww[~small], 110 * 2.0 ** -24 * ww[~small], "f32")
