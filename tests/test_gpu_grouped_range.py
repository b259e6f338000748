"""ops.grouped_rows in float32 on the largest floats, in calls of few rows and of many.  Formulas and
tolerances are those of test_gpu_grouped.py, and 2^-126 for each term more: a product of small factors may
be smaller than float32 has numbers (dx[5, 3] sums terms of 2^-160)."""
import pytest
import torch

import test_gpu_grouped as grouped
from test_gpu_grouped import inputs, offsets_of, reference, run

pytestmark = pytest.mark.gpu

MOST = torch.finfo(torch.float32).max


def check(got, want, what):
    ref, size, terms = want
    grouped.check(got, (ref, size + 2.0 ** -126 / grouped.U, terms), what)      # times u and over twice the terms


@pytest.mark.parametrize("sizes", [[9, 0, 7], [60, 70, 50], [9000, 12000, 300]])
@pytest.mark.parametrize("value", [MOST, -MOST, 3.395e38])
def test_the_largest_floats_among_the_rows(sizes, value):
    """An entry over 3.39e38 would round to an infinite bfloat16.  Its factors are small enough (2^-80)
    for every product to be an ordinary float."""
    K, N, off = 37, 45, offsets_of(sizes)
    x, w, b, dout = inputs(sum(sizes), K, N, 3, torch.float32)
    with torch.no_grad():
        x[5, 3] = value
        w[:, 3] *= 2.0 ** -80
        dout[5] *= 2.0 ** -80
    got, want = run(x, w, b, off, dout), reference(x, w, b, off, dout)
    for k in got:
        check(got[k], want[k], k)


@pytest.mark.parametrize("sizes", [[9, 0, 7], [60, 70, 50], [9000, 12000, 300]])
def test_the_largest_floats_among_the_weights(sizes):
    K, N, off = 37, 45, offsets_of(sizes)
    x, w, b, dout = inputs(sum(sizes), K, N, 3, torch.float32)
    with torch.no_grad():
        w[0, 36, 44] = MOST
        w[2, 36, 44] = -3.395e38
        x[:, 36] *= 2.0 ** -40
        dout[:, 44] *= 2.0 ** -40
    got, want = run(x, w, b, off, dout), reference(x, w, b, off, dout)
    for k in got:
        check(got[k], want[k], k)
