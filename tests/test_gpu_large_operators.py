"""Typed product, residual norm and class head on arrays of more than 2^31 elements: the rows and
classes behind the 32-bit mark come out as they do in a small call of their own, or as the formula
says.  bfloat16, so that an array takes 4.3 GB."""
import pytest
import torch

from util import dev

pytestmark = pytest.mark.gpu

WIDE = 1024
ROWS = 2 ** 31 // WIDE + 700      # of WIDE elements: past 2^31 of them
TAIL = 600


def randn(*shape, seed=0, mul=1.0):
    gen = torch.Generator(device=dev()).manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device=dev(), dtype=torch.float32) * mul).to(torch.bfloat16)


def filled(rows, seed):
    """[rows, WIDE] of random rows that repeat every 4096, but for the last TAIL, which are their own."""
    block = randn(4096, WIDE, seed=seed)
    t = torch.empty(rows, WIDE, dtype=torch.bfloat16, device=dev())
    for at in range(0, rows, 4096):
        t[at:at + 4096] = block[:min(4096, rows - at)]
    t[-TAIL:] = randn(TAIL, WIDE, seed=seed + 1)
    return t


def close(got, want, size):
    """want: float64 sums of `size` absolute terms each in float32 arithmetic, rounded to bfloat16 (2^-8)."""
    want, size = want.double(), size.double()
    tol = 4096 * 2.0 ** -24 * size + 2.0 ** -8 * (want.abs() + 4096 * 2.0 ** -24 * size)
    assert bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("narrow", [8, 7])      # streaming tiles, tiles in registers
def test_typed_product(narrow):
    from jittorgeometric_amd.ops import grouped_rows
    x = randn(ROWS, narrow, seed=1).requires_grad_(True)
    w = randn(2, narrow, WIDE, seed=2).requires_grad_(True)
    off = torch.tensor([0, ROWS - TAIL, ROWS], dtype=torch.int32, device=dev())
    out = grouped_rows(x, w, off)
    g = filled(ROWS, 3)
    dx, dw = torch.autograd.grad(out, [x, w], g)
    xs, gs, ws = x.detach()[-TAIL:].double(), g[-TAIL:].double(), w.detach()[1].double()
    close(out.detach()[-TAIL:], torch.mm(xs, ws), torch.mm(xs.abs(), ws.abs()))
    close(dx[-TAIL:], torch.mm(gs, ws.t()), torch.mm(gs.abs(), ws.abs().t()))
    close(dw[1], torch.mm(xs.t(), gs), torch.mm(xs.abs().t(), gs.abs()))


def test_residual_norm():
    from jittorgeometric_amd.nn import residual_norm
    x, y = filled(ROWS, 5), filled(ROWS, 7)
    ds, dh = filled(ROWS, 9), filled(ROWS, 11)
    w = randn(WIDE, seed=13).requires_grad_(True)

    def run(rows):
        a, b = (t[rows].detach().requires_grad_(True) for t in (x, y))
        s, h = residual_norm(a, b, w)
        return [s.detach(), h.detach(), *torch.autograd.grad([s, h], [a, b], [ds[rows], dh[rows]])]

    want = run(slice(ROWS - TAIL, ROWS))
    got = run(slice(0, ROWS))
    for a, b in zip(got, want):      # a row is the same arithmetic wherever it lies
        assert torch.equal(a[-TAIL:], b)


def test_class_head():
    from jittorgeometric_amd.nn import linear_cross_entropy
    V = 5
    x = randn(V, WIDE, seed=15, mul=WIDE ** -0.5).requires_grad_(True)
    w = filled(ROWS, 17).requires_grad_(True)
    t = torch.tensor([0, ROWS - 1, ROWS - TAIL, -1, ROWS // 2], device=dev())
    loss = linear_cross_entropy(x, w, t, reduction="none")
    z = torch.cat([torch.mm(x.detach().double(), w.detach()[a:a + 65536].double().t()) for a in range(0, ROWS, 65536)], 1)
    lse = torch.logsumexp(z, 1)
    ok = t >= 0
    want = torch.where(ok, lse - z.gather(1, t.clamp(min=0)[:, None])[:, 0], 0)
    # a logit: (2 F + 16) 2^-24 of its absolute terms, 1024 / 32 of under 1 on average: 2^-8.  lse: that, and under a
    # thousand additions one after the other (a lane's classes, then lanes and ranges): 2^-13.  Twice, as lse - z:
    off = 2.0 ** -6
    assert bool((torch.mm(x.detach().double().abs(), w.detach()[-TAIL:].double().abs().t()) < 32).all())
    assert bool(((loss.detach().double() - want).abs() <= off).all())
    dx, dw = torch.autograd.grad(loss.sum(), [x, w])
    d = torch.exp(z - lse[:, None])
    d.scatter_add_(1, t.clamp(min=0)[:, None], -torch.ones_like(lse)[:, None])
    d = torch.where(ok[:, None], d, 0)
    tail = d[:, -TAIL:]
    got, ref = dw[-TAIL:].double(), torch.mm(tail.t(), x.detach().double())
    # p is off by its exponent's error, d rounded to bfloat16 (2^-8); g is 1
    assert bool(((got - ref).abs() <= (off + 2.0 ** -8) * torch.mm(tail.abs().t(), x.detach().double().abs()) + 2.0 ** -8 * ref.abs()).all())
    assert not dx[3].any() and bool(torch.isfinite(dx).all())
