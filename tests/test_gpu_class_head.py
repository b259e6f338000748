"""nn.linear_cross_entropy against its formula in float64 (on the GPU's float64 units, elementary
products and exponentials), without the library's kernels.

Tolerances, with u = 2^-24.  A logit is a sum of F + 1 float32 terms added by an adder that may
truncate: |dz| <= (2 F + 16) u S with S its absolute terms; D is a row's largest.  lse adds C
exponentials, each off by its argument's error and a few u: E = 2 D + (2 C + 64) u + 4 u (max |z| +
|lse|) bounds lse and the loss.  d = g (p - onehot) is then off by 3 E g p + r |d|, r = 4 u, or 2^-8
where d is rounded to bfloat16.  Gradients add that through |w|, |x| or 1, and (2 n + 16) u of their
absolute terms for n summands; a result rounded to bfloat16 is off by 2^-8 of itself more.  Numbers
under 2^-126 may be lost: float32 has no exponent for them.  An exponential and its product with g
(|g| < 4 here, but for the scaled means, whose g is under 1) lose under 2^-124 together, a product with
an entry of the other operand under 2^-126.

float32 operands are held as two float16 parts of an array scaled so that its largest entry M lies in
2^14 .. 2^15: two roundings to 11 bits leave 2^-24 of an entry (the 16 u above cover those of both factors
and the product of the second parts), but float16's spacing ends at 2^-24, so that an entry is never held
closer than half of that, 2^-25 2^-14 M < 2^-38 M.  A sum over k is off by 2^-38 (M_x sum |w| + M_w sum |x|)
more, d (M = 1) by 2^-38 |g| more."""
import math

import pytest
import torch

from util import dev

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = 2.0 ** -124
GRAIN = 2.0 ** -38
DTYPES = [torch.float32, torch.bfloat16]


def reference(x, w, b, t, g, reduction):
    half = x.dtype == torch.bfloat16
    x, w = x.detach().double(), w.detach().double()
    V, F = x.shape
    C = w.shape[0]
    b = torch.zeros(C, dtype=torch.float64, device=x.device) if b is None else b.detach().double()
    z = torch.mm(x, w.t()) + b
    live = torch.isfinite(b)
    grain = 0.0 if half else GRAIN
    top = lambda v: float(v.abs().amax()) if v.numel() else 0.0  # noqa: E731
    D = (2 * F + 16) * U * (torch.mm(x.abs(), w.abs().t()) + torch.where(live, b.abs(), 0)).amax(1)
    D = D + grain * (top(x) * w.abs().sum(1).amax() + top(w) * x.abs().sum(1))
    lse = torch.logsumexp(z, 1)
    ok = (t >= 0) & (t < C)
    lab = torch.where(ok, t, 0).long()
    at = z.gather(1, lab[:, None])[:, 0]
    zmax = torch.where(torch.isfinite(z), z.abs(), 0).amax(1)
    E = 2 * D + (2 * C + 64) * U + 4 * U * (zmax + lse.abs())
    row = torch.where(ok, lse - at, 0)
    Erow = torch.where(ok, E, 0)
    n = int(ok.sum())
    if reduction == "none":
        loss, tol = row, Erow + U * row.abs()
        g = g.double()
    else:
        total, err = row.sum(), Erow.sum()
        if reduction == "mean":
            total, err = total / max(n, 1) if n else total * math.nan, err / max(n, 1)
        loss, tol = total, err + 2 * U * total.abs()
        g = torch.full((V,), float(g) / (max(n, 1) if reduction == "mean" else 1), dtype=torch.float64, device=x.device)
    g = torch.where(ok, g, 0)
    p = torch.exp(z - lse[:, None])
    d = p.clone()
    d.scatter_add_(1, lab[:, None], -torch.ones_like(at)[:, None])
    d = torch.where(ok[:, None], d * g[:, None], 0)
    dd = torch.where(ok[:, None], 3 * E[:, None] * p * g.abs()[:, None], 0) + (2.0 ** -8 if half else 4 * U) * d.abs() + TINY
    dd = dd + torch.where(ok, grain * g.abs(), 0)[:, None]
    A = d.abs()
    ones = torch.ones(V, 1, dtype=torch.float64, device=x.device)

    def grad(left, leftd, leftabs, right, terms):
        tol = torch.mm(leftd + (2 * terms + 16) * U * leftabs, right.abs()) + terms * TINY
        return torch.mm(left, right), tol + grain * top(right) * leftabs.sum(1, keepdim=True)

    # with one g a row dw takes g x, rounded to bfloat16 once more: 2^-8 of every term
    again = 2.0 ** -8 * A if half and reduction == "none" else 0
    out = {"loss": (loss, tol), "dx": grad(d, dd, A, w, C), "dw": grad(d.t(), (dd + again).t(), A.t(), x, V)}
    db = grad(d.t(), dd.t(), A.t(), ones, V)
    out["db"] = (db[0][:, 0], db[1][:, 0])
    return out


def check(got, want, what):
    ref, tol = want
    if got.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (ref.abs() + tol)
    got = got.detach().double()
    assert got.shape == ref.shape, what
    same = (got == ref) | (torch.isnan(got) & torch.isnan(ref))
    bad = ~(((got - ref).abs() <= tol) | same)
    assert not bad.any(), "%s: %d of %d off, first at %s" % (what, int(bad.sum()), bad.numel(), bad.nonzero()[0].tolist())


def inputs(V, F, C, dtype, seed=0, spread=2.0, unlabelled=True):
    gen = torch.Generator().manual_seed(seed)

    def rand(*shape, mul=1.0):
        return (torch.randn(*shape, generator=gen) * mul).to(dtype).to(dev()).requires_grad_(True)

    x, w, b = rand(V, F), rand(C, F, mul=spread * F ** -0.5), rand(C, mul=0.5)
    t = torch.randint(0, C, (V,), generator=gen)
    if unlabelled and V > 2:
        t[::5] = torch.tensor([-100, C, -1, 2 ** 31 - 1])[torch.arange(t[::5].numel()) % 4]
    return x, w, b, t.to(dev()), torch.randn(V, generator=gen).to(dev())


def run(x, w, b, t, g, reduction):
    from jittorgeometric_amd.nn import linear_cross_entropy
    loss = linear_cross_entropy(x, w, t, bias=b, reduction=reduction)
    leaves = [v for v in (x, w, b) if v is not None]
    up = g if reduction == "none" else torch.tensor(float(g), device=dev())
    return dict(zip(["loss", "dx", "dw", "db"], [loss, *torch.autograd.grad(loss, leaves, up)]))


def compare(x, w, b, t, g, reduction):
    got, want = run(x, w, b, t, g, reduction), reference(x, w, b, t, g, reduction)
    for k in got:
        check(got[k], want[k], "%s, %s" % (k, reduction))
    return got


SHAPES = [(1, 1, 1), (1, 8, 5), (3, 2, 2), (5, 33, 130), (130, 64, 129), (257, 72, 300), (64, 200, 1000), (7, 256, 5021),
          (300, 100, 2003), (129, 513, 257), (5000, 8, 40), (17, 16, 128), (16, 24, 3001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,F,C", SHAPES)
def test_loss_and_gradients(V, F, C, dtype):
    x, w, b, t, g = inputs(V, F, C, dtype, seed=V + F + C)
    compare(x, w, b, t, g, "none")
    compare(x, w, None, t, 0.7, "mean")
    compare(x, w, b, t.to(torch.int32), 1.0, "mean")
    compare(x, w, b, t, 0.3, "sum")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,F,C", [(3000, 100, 4100), (700, 129, 13000), (2049, 264, 5000), (1025, 7, 6529)])
def test_more_than_small_tiles_take(V, F, C, dtype):
    x, w, b, t, g = inputs(V, F, C, dtype)
    compare(x, w, b, t, g, "none")
    compare(x, w, None, t, 1.0, "sum")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,F,C", [(16500, 8, 150), (20000, 16, 8500), (16390, 40, 8200)])
def test_blocks_of_rows_and_pieces_of_classes(V, F, C, dtype):
    x, w, b, t, g = inputs(V, F, C, dtype)
    got = compare(x, w, b, t, 100.0, "mean")
    again = run(x, w, b, t, 100.0, "mean")
    for k in got:
        assert torch.equal(got[k], again[k]), k


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_without_a_label(dtype):
    x, w, b, t, g = inputs(40, 16, 50, dtype)
    got = run(x, w, b, t, g, "none")
    out = ~((t >= 0) & (t < 50))
    assert out.any() and not got["loss"][out].any() and not got["dx"][out].any()
    nobody = torch.full_like(t, -1)
    got = run(x, w, b, nobody, 1.0, "mean")
    assert torch.isnan(got["loss"])
    for k in ("dx", "dw", "db"):
        assert not got[k].any(), k
    got = run(x, w, b, nobody, 1.0, "sum")
    assert float(got["loss"].detach()) == 0.0
    # what a row without a label holds does not matter
    with torch.no_grad():
        x[out] = float("nan")
    got = run(x, w, b, t, g, "none")
    with torch.no_grad():
        x[out] = 0
    want = reference(x, w, b, t, g, "none")
    assert not got["loss"][out].any() and not got["dx"][out].any()
    check(got["loss"], want["loss"], "loss")
    check(got["dx"], want["dx"], "dx")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,F,C", [(32, 2047, 130), (9, 2060, 70), (31, 130, 1000), (33, 131, 1000), (8, 63, 4099), (4, 1, 65),
                                   (17, 67, 64), (1, 2048, 30001)])
def test_few_rows(V, F, C, dtype):
    x, w, b, t, g = inputs(V, F, C, dtype, seed=V)
    compare(x, w, b, t, g, "none")
    compare(x, w, None, t, 1.0, "mean")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("F", [32, 29])
@pytest.mark.parametrize("left", [math.nan, math.inf, 3e38])
def test_what_a_row_without_a_label_holds(dtype, reduction, F, left):
    V, C = 90, 150
    x, w, b, t, g = inputs(V, F, C, dtype)
    out = ~((t >= 0) & (t < C))
    assert out.any()
    g = g if reduction == "none" else 1.0
    with torch.no_grad():
        x[out] = 0
    want = run(x, w, b, t, g, reduction)
    with torch.no_grad():
        x[out] = left
    got = run(x, w, b, t, g, reduction)
    for k in ("loss", "dx", "dw", "db"):
        assert torch.equal(got[k], want[k]), k


@pytest.mark.parametrize("dtype", DTYPES)
def test_classes_masked_by_the_bias(dtype):
    x, w, b, t, g = inputs(70, 24, 300, dtype)
    with torch.no_grad():
        b[10:200] = float("-inf")
        t[3], t[4] = 15, 250
    compare(x, w, b, t, g, "none")
    assert torch.isinf(run(x, w, b, t, g, "none")["loss"][3])
    with torch.no_grad():
        b[:] = torch.finfo(dtype).min
    got = run(x, w, b, t, g, "none")      # all equal: z is the bias to the last bit
    assert torch.isfinite(got["loss"]).all() and torch.isfinite(got["dx"]).all()
    with torch.no_grad():
        b[:] = float("-inf")
    assert torch.isnan(run(x, w, b, t, g, "none")["loss"][t == 250]).all()


def test_large_logits():
    x, w, b, t, g = inputs(50, 32, 700, torch.float32, spread=3000.0)
    got = compare(x, w, b, t, g, "none")
    assert torch.isfinite(got["loss"]).all()


@pytest.mark.parametrize("by_x,by_w", [(0, -105), (-105, 0), (-70, -70), (100, -110), (-110, 100)])
def test_operands_far_from_one(by_x, by_w):
    x, w, b, t, g = inputs(60, 32, 200, torch.float32)
    with torch.no_grad():
        x *= 2.0 ** by_x
        w *= 2.0 ** by_w
    for reduction, up in (("none", g), ("mean", 1.0)):
        compare(x, w, b, t, up, reduction)


def test_a_bad_row_stays_alone():
    x, w, b, t, g = inputs(140, 36, 260, torch.float32, unlabelled=False)
    want = run(x, w, b, t, g, "none")
    with torch.no_grad():
        x[131, 35] = float("nan")
    got = run(x, w, b, t, g, "none")
    rest = torch.arange(140, device=dev()) != 131
    assert torch.isnan(got["loss"][131]) and torch.isnan(got["dx"][131]).all()
    assert torch.equal(got["loss"][rest], want["loss"][rest]) and torch.equal(got["dx"][rest], want["dx"][rest])


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_unaligned_starts_and_upstream_gradients(dtype):
    from jittorgeometric_amd.nn import linear_cross_entropy
    V, F, C = 37, 40, 210
    x, w, b, t, g = inputs(V, F, C, dtype)
    want = reference(x, w, b, t, torch.full((V,), 2.5, device=dev()), "none")
    xs = torch.empty(F, V, dtype=dtype, device=dev()).t()
    xs.copy_(x.detach())
    store = torch.empty(C * F + 1, dtype=dtype, device=dev())
    ws = store[1:].view(C, F)
    ws.copy_(w.detach())
    ts = torch.stack([t, t], 1)[:, 0]
    xs, ws = xs.requires_grad_(True), ws.requires_grad_(True)
    loss = linear_cross_entropy(xs, ws, ts, bias=b, reduction="none")
    gx, gw, gb = torch.autograd.grad(2.5 * loss.sum(), [xs, ws, b])      # an expanded gradient
    for k, v in (("loss", loss), ("dx", gx), ("dw", gw), ("db", gb)):
        check(v, want[k], k)


def test_only_some_inputs_need_gradients():
    from jittorgeometric_amd.nn import linear_cross_entropy
    x, w, b, t, g = inputs(33, 20, 140, torch.float32)
    want = reference(x, w, b, t, 1.0, "mean")
    for keep in ("x", "w", "b"):
        v = {"x": x.detach(), "w": w.detach(), "b": b.detach()}
        v[keep].requires_grad_(True)
        grad, = torch.autograd.grad(linear_cross_entropy(v["x"], v["w"], t, bias=v["b"]), [v[keep]])
        check(grad, want["d" + keep], keep)
    assert not linear_cross_entropy(x.detach(), w.detach(), t).requires_grad


def test_agrees_with_the_loss_on_logits():
    """Both losses are within the bound of the formula; cross_entropy_loss's own is 1e-5."""
    from jittorgeometric_amd.nn import cross_entropy_loss, linear_cross_entropy
    x, w, b, t, g = inputs(500, 32, 47, torch.float32)
    one = linear_cross_entropy(x, w, t, bias=b)
    two = cross_entropy_loss(x.detach() @ w.detach().t() + b.detach(), t)
    assert abs(float(one.detach()) - float(two)) <= 1e-5 * abs(float(two)) + float(reference(x, w, b, t, 1.0, "mean")["loss"][1])


def test_no_rows():
    x, w, b, t, g = inputs(0, 8, 12, torch.float32)
    got = run(x, w, b, t, 1.0, "mean")
    assert torch.isnan(got["loss"]) and got["dx"].shape == (0, 8) and not got["dw"].any() and not got["db"].any()
    assert run(x, w, b, t, g, "none")["loss"].shape == (0,)
    assert float(run(x, w, b, t, 1.0, "sum")["loss"].detach()) == 0.0


def test_gradients_against_differences():
    """Central differences of the formula in float64 with h = 1e-4: truncation and rounding under 1e-6."""
    x, w, b, t, g = inputs(4, 3, 6, torch.float32)
    got = run(x, w, b, t, g, "none")
    want = reference(x, w, b, t, g, "none")
    v = {"x": x.detach().double(), "w": w.detach().double(), "b": b.detach().double()}

    def loss():
        z = v["x"] @ v["w"].t() + v["b"]
        ok = (t >= 0) & (t < 6)
        row = torch.logsumexp(z, 1) - z.gather(1, torch.where(ok, t, 0)[:, None])[:, 0]
        return float((torch.where(ok, row, 0) * g.double()).sum())

    for k in v:
        for i in range(v[k].numel()):
            flat = v[k].view(-1)
            keep = float(flat[i])
            flat[i] = keep + 1e-4
            up = loss()
            flat[i] = keep - 1e-4
            down = loss()
            flat[i] = keep
            tol = float(want["d" + k][1].reshape(-1)[i]) + 1e-6
            assert abs((up - down) / 2e-4 - float(got["d" + k].view(-1)[i])) <= tol, (k, i)


def test_replays_as_a_graph_and_on_another_stream():
    x, w, b, t, g = inputs(600, 64, 3000, torch.bfloat16)

    def step():
        return list(run_captured())

    from jittorgeometric_amd.nn import linear_cross_entropy

    def run_captured():
        loss = linear_cross_entropy(x, w, t, bias=b)
        return [loss, *torch.autograd.grad(loss, [x, w, b])]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            side = [v.detach().clone() for v in step()]
    torch.cuda.current_stream().wait_stream(s)
    for a, c in zip(side, step()):
        assert torch.equal(a, c)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for trial in range(3):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
            t.copy_(torch.randint_like(t, 0, 3000))
        torch.cuda.synchronize()
        want = [v.detach().clone() for v in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(static, want):
            assert torch.equal(a, c), trial


def test_refusals():
    from jittorgeometric_amd import JgamdError
    from jittorgeometric_amd.nn import linear_cross_entropy
    x, w, b, t, g = inputs(10, 4, 6, torch.float32)
    for args, kw in (((x[0], w, t), {}), ((x, w[0], t), {}), ((x[:, :3], w, t), {}), ((x, w, t[:9]), {}),
                     ((x, w, t[:, None]), {}), ((x, w, t.float()), {}), ((x, w.bfloat16(), t), {}),
                     ((x, w, t), {"bias": b[:5]}), ((x, w, t), {"bias": b.bfloat16()}), ((x, w, t), {"reduction": "max"}),
                     ((x.half(), w.half(), t), {}), ((x, w[:0], t), {}), ((x.cpu(), w, t), {}), ((x, w, t.cpu()), {})):
        with pytest.raises(JgamdError):
            linear_cross_entropy(*args, **kw)
