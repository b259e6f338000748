"""nn.linear_cross_entropy in float32 on operands of very different sizes.  Formulas and tolerances are
those of test_gpu_class_head.py without its GRAIN: each row's and each class's error is bounded by its own
absolute terms, as for products of floats, whatever the other rows and classes hold.

An operand's three bfloat16 parts hold its 24 bits as far as bfloat16 has an exponent (2^-126); the
dropped products of parts are under 2^-24 of a term, which the 16 u of the bounds hold."""
import pytest
import torch

import test_gpu_class_head as head
from test_gpu_class_head import check, inputs, reference, run
from util import dev

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_grain(monkeypatch):
    monkeypatch.setattr(head, "GRAIN", 0.0)


def compare(x, w, b, t, g, reduction):
    got, want = run(x, w, b, t, g, reduction), reference(x, w, b, t, g, reduction)
    for k in got:
        check(got[k], want[k], "%s, %s" % (k, reduction))
    return got


SIZES = [(512, 64, 4096), (20, 96, 1000), (300, 37, 515), (3000, 130, 4100)]


@pytest.mark.parametrize("V,F,C", SIZES + [(16500, 8, 150)])
def test_every_result_has_float32_precision(V, F, C):
    x, w, b, t, g = inputs(V, F, C, torch.float32)
    compare(x, w, b, t, g, "none")
    compare(x, w, None, t, 1.0, "mean")


@pytest.mark.parametrize("V,F,C", SIZES)
@pytest.mark.parametrize("c", [1e6, 1e8, 1e30])
def test_a_large_row_leaves_the_others_as_they_are(V, F, C, c):
    x, w, b, t, g = inputs(V, F, C, torch.float32, unlabelled=False)
    with torch.no_grad():
        x[V // 2] *= c
    got, want = run(x, w, b, t, g, "none"), reference(x, w, b, t, g, "none")
    for k in got:
        check(got[k], want[k], k)


@pytest.mark.parametrize("V,F,C", SIZES)
def test_a_large_class_and_a_large_feature(V, F, C):
    x, w, b, t, g = inputs(V, F, C, torch.float32)
    with torch.no_grad():
        w[C // 3] *= 1e7
    compare(x, w, b, t, g, "none")
    x, w, b, t, g = inputs(V, F, C, torch.float32)
    with torch.no_grad():
        x[:, 3] *= 1e9
        w[:, 3] *= 1e-9
    compare(x, w, b, t, g, "none")
    compare(x, w, b, t, 1.0, "mean")


@pytest.mark.parametrize("V,F,C", SIZES)
@pytest.mark.parametrize("below", [18.0, 23.0, 28.0, 60.0])
def test_gradients_of_classes_of_small_probability(V, F, C, below):
    """exp(-below) against the others: 1e-8, 1e-10, 1e-12, 1e-26.  Their rows of dw keep their own 24 bits."""
    x, w, b, t, g = inputs(V, F, C, torch.float32)
    with torch.no_grad():
        b[1::3] -= below
    t = torch.where((t >= 0) & (t < C) & (t % 3 == 1), t - 1, t)
    compare(x, w, b, t, g, "none")
    compare(x, w, b, t, 1.0, "mean")


@pytest.mark.parametrize("V,F,C", SIZES)
def test_upstream_gradients_of_different_sizes(V, F, C):
    x, w, b, t, g = inputs(V, F, C, torch.float32)
    g[::2] *= 1e-12
    compare(x, w, b, t, g, "none")


def test_the_largest_floats():
    """An entry over 3.39e38 would round to an infinite bfloat16.  Where a result and its bound reach
    2^128 (1 - 2^-25), from where on float32 rounds to infinity, an infinity of its sign is within the
    bound: dw[74, 2] is d x = -1 times -1 times the largest float, rounded sums of whose parts may pass it."""
    x, w, b, t, g = inputs(40, 16, 90, torch.float32, unlabelled=False)
    with torch.no_grad():
        x[7, 2] = torch.finfo(torch.float32).max
        x[33, 2] = -torch.finfo(torch.float32).max
        w[:, 2] = 1e-36 * torch.arange(90, device=dev())
        w[:, 2].mul_(2.0 ** 20)      # clear of the numbers without 24 bits
    g = g.clamp(-1, 1)
    got, want = run(x, w, b, t, g, "none"), reference(x, w, b, t, g, "none")
    for k in got:
        value, tol = want[k]
        past = value.abs() + tol >= 2.0 ** 128 * (1 - 2.0 ** -25)
        assert k == "dw" and not past[:, torch.arange(16, device=dev()) != 2].any() or not past.any(), k
        infinite = past & torch.isinf(got[k]) & (torch.sign(got[k]) == torch.sign(value))
        result = torch.where(infinite, value, got[k].detach().double())
        assert torch.isfinite(result).all(), k
        check(result, want[k], k)


@pytest.mark.parametrize("V", [1, 8, 32])
@pytest.mark.parametrize("F,C,spread", [(2000, 3000, 3e6), (256, 3000, 1e7), (2000, 700, 3e5), (64, 5000, 1e6)])
def test_few_rows_with_large_logits(V, F, C, spread):
    """Logits so large that their last bit is of the size of one: z - lse may come out over zero where the
    two sums round apart.  A probability is still none over one: with one labelled row and g = 1, db is d."""
    for seed in range(4):
        x, w, b, t, g = inputs(V, F, C, torch.float32, seed=seed, spread=spread, unlabelled=False)
        got = run(x, w, b, t, torch.ones_like(g), "none")
        for k in got:
            assert torch.isfinite(got[k]).all(), k
        row = seed % V
        t = torch.where(torch.arange(V, device=dev()) == row, t, -1)
        got = run(x, w, b, t, torch.ones_like(g), "none")
        for k in got:
            assert torch.isfinite(got[k]).all(), k
        assert got["db"].abs().max() <= 1


@pytest.mark.parametrize("V", [8, 100, 3000])
def test_large_logits_in_bfloat16(V):
    """Both passes sum a bfloat16 logit in the same order, so that z - lse is never over zero."""
    x, w, b, t, g = inputs(V, 512, 3000, torch.bfloat16, spread=1e7, unlabelled=False)
    for row in (0, V - 1, V // 2):
        got = run(x, w, b, torch.where(torch.arange(V, device=dev()) == row, t, -1), torch.ones_like(g), "none")
        for k in got:
            assert torch.isfinite(got[k]).all(), k
        assert got["db"].abs().max() <= 1
