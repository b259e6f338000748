"""nn.residual_norm and nn.rms_norm against their formulas in float64.

Tolerances, with u = 2^-24.  A sum of n float32 terms is off by at most n u of the sum of the absolute
terms, a chain of a few dozen operations by their number times u; an inverse norm inherits half the
relative error of its mean square.  Every intermediate is bounded by the same expression in absolute
values ("size" below); kappa = mean(|s| (|x| + |v|)) / mean(s^2) says how much larger the parts of s are
than s, which is what the rounding of s costs the norm of s.  |error| <= (2 F + 200) u size, column sums
2 R u of their sizes more; a result rounded to bfloat16 is off by 2^-8 of itself more."""
import itertools

import pytest
import torch

from util import dev

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16]
EPS = 1e-6


def reference(t, ds, dh):
    """{name: (value, size, extra terms)} in float64; t: dict of the inputs, None where left out."""
    D = {k: None if v is None else v.detach().double().cpu() for k, v in t.items()}
    x, y, w, p, gate, k = (D[n] for n in ("x", "y", "w", "post", "gate", "scale"))
    zero = torch.zeros_like(x)
    ds, dh = (zero if v is None else v.detach().double().cpu() for v in (ds, dh))
    one = torch.ones((), dtype=torch.float64)
    g = one if gate is None else torch.sigmoid(gate)
    k = one if k is None else k
    mean = lambda v: v.mean(1, keepdim=True)  # noqa: E731
    if y is None:
        v = zero
    else:
        ry = one if p is None else 1 / torch.sqrt(mean(y * y) + EPS)
        pw = one if p is None else p
        v = k * g * (y * ry * pw)
    s = x + v
    A = x.abs() + v.abs()
    rs = 1 / torch.sqrt(mean(s * s) + EPS)
    kappa = 1 + mean(s.abs() * A) * rs ** 2
    h = s * rs * w
    hw = dh * w
    dx = ds + rs * hw - s * rs ** 3 * mean(hw * s)
    sx = kappa ** 3 * (ds.abs() + rs * hw.abs() + A * rs ** 3 * mean(hw.abs() * A))
    out = {"s": (s, A, 0), "h": (h, kappa * A * rs * w.abs(), 0), "dx": (dx, sx, 0)}
    R = x.shape[0]
    out["dw"] = ((dh * s * rs).sum(0), (dh.abs() * A * rs * kappa).sum(0), R)
    if y is not None:
        dv, sv = dx * k * g, sx * (k * g).abs()
        if p is None:
            out["dy"] = (dv, sv, 0)
        else:
            out["dy"] = (ry * dv * pw - y * ry ** 3 * mean(dv * pw * y),
                         ry * sv * pw.abs() + y.abs() * ry ** 3 * mean(sv * (pw * y).abs()), 0)
            out["dpost"] = ((dv * y * ry).sum(0), (sv * (y * ry).abs()).sum(0), R)
        u = y * ry * pw
        if gate is not None:
            out["dgate"] = (dv * u * (1 - g), sv * u.abs() * (1 + gate.abs()), 0)
        if D["scale"] is not None:
            out["dscale"] = ((dx * g * u).sum(0), (sx * g * u.abs()).sum(0), R)
    return out


def check(got, want, F, what):
    ref, size, terms = want
    tol = (2 * F + 200 + 2 * terms) * U * size
    if got.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (ref.abs() + tol)
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, what
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), "%s: %d of %d off, first at %s" % (what, int(bad.sum()), bad.numel(), bad.nonzero()[0].tolist())


def inputs(R, F, dtype, options="pgk", seed=0, block=True):
    gen = torch.Generator().manual_seed(seed)

    def rand(*shape, mul=1.0, add=0.0):
        return (torch.randn(*shape, generator=gen) * mul + add).to(dtype).to(dev()).requires_grad_(True)

    t = {"x": rand(R, F, mul=2), "y": rand(R, F) if block else None, "w": rand(F, mul=0.2, add=1),
         "post": rand(F, mul=0.2, add=1) if "p" in options else None, "gate": rand(R, F, mul=2) if "g" in options else None,
         "scale": rand(F, mul=0.3, add=0.5) if "k" in options else None}
    return t, rand(R, F).detach(), rand(R, F).detach()


NAMES = {"x": "dx", "y": "dy", "w": "dw", "post": "dpost", "gate": "dgate", "scale": "dscale"}


def forward(t):
    from jittorgeometric_amd.nn import residual_norm, rms_norm
    if t["y"] is None:
        return [rms_norm(t["x"], t["w"], eps=EPS)]
    return list(residual_norm(t["x"], t["y"], t["w"], post_weight=t["post"], gate=t["gate"], scale=t["scale"], eps=EPS))


def run(t, ds, dh):
    outs = forward(t)
    leaves = {k: v for k, v in t.items() if v is not None}
    up = [dh] if t["y"] is None else [ds, dh]
    grads = torch.autograd.grad(outs, list(leaves.values()), up)
    got = {NAMES[k]: g for k, g in zip(leaves, grads)}
    got.update(zip(["h"] if t["y"] is None else ["s", "h"], outs))
    return got


SHAPES = [(1, 1), (3, 7), (5, 64), (2, 65), (130, 100), (300, 256), (7, 512), (9, 513), (40, 1001), (33, 1024), (5, 2048),
          (3, 2056), (4, 4100), (2, 8192), (2, 6001), (40000, 8), (9001, 384)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,F", SHAPES)
def test_results_and_gradients(R, F, dtype):
    for block in (True, False):
        t, ds, dh = inputs(R, F, dtype, "pgk" if block else "", seed=R + F, block=block)
        got = run(t, ds, dh)
        want = reference(t, ds if block else None, dh)
        for k in got:
            check(got[k], want[k], F, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("options", ["".join(c) for n in range(4) for c in itertools.combinations("pgk", n)])
def test_each_part_may_be_left_out(options, dtype):
    t, ds, dh = inputs(70, 136, dtype, options)
    got, again = run(t, ds, dh), run(t, ds, dh)
    want = reference(t, ds, dh)
    assert set(got) == set(want)
    for k in got:
        check(got[k], want[k], 136, k)
        assert torch.equal(got[k], again[k]), k


@pytest.mark.parametrize("which", ["s", "h"])
def test_one_of_the_two_outputs_is_used(which):
    t, ds, dh = inputs(19, 72, torch.float32)
    s, h = forward(t)
    leaves = {k: v for k, v in t.items() if k != "w" or which == "h"}
    grads = torch.autograd.grad(s if which == "s" else h, list(leaves.values()), ds if which == "s" else dh)
    want = reference(t, ds if which == "s" else None, dh if which == "h" else None)
    for k, g in zip(leaves, grads):
        check(g, want[NAMES[k]], 72, k)


def test_only_some_inputs_need_gradients():
    t, ds, dh = inputs(21, 40, torch.float32)
    for keep in (["x"], ["gate"], ["scale", "y"], ["w"]):
        u = {k: v.detach().requires_grad_(k in keep) for k, v in t.items()}
        grads = torch.autograd.grad(forward(u), [u[k] for k in keep], [ds, dh])
        want = reference(t, ds, dh)
        for k, g in zip(keep, grads):
            check(g, want[NAMES[k]], 40, k)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_unaligned_starts(dtype):
    R, F = 23, 88
    t, ds, dh = inputs(R, F, dtype)
    want = reference(t, ds, dh)
    moved = {}
    for k, v in t.items():
        store = torch.empty(v.numel() + 1, dtype=dtype, device=dev())
        moved[k] = store[1:].view(v.shape)
        moved[k].copy_(v.detach())
        moved[k].requires_grad_(True)
    got = run(moved, ds.t().contiguous().t(), dh)
    for k in got:
        check(got[k], want[k], F, k)
    spread = {k: torch.stack([v.detach(), v.detach()], -1)[..., 0].requires_grad_(True) for k, v in t.items()}
    assert not spread["x"].is_contiguous()
    got = run(spread, ds, dh)
    for k in got:
        check(got[k], want[k], F, k)


def test_zero_rows_of_values_bad_values_and_saturated_gates():
    t, ds, dh = inputs(12, 48, torch.float32)
    with torch.no_grad():
        t["x"][0] = 0
        t["y"][0] = 0
        t["gate"][1] = float("-inf")
        t["gate"][2] = float("inf")
        t["gate"][3] = 1000.0
        t["gate"][4] = -1000.0
    got = run(t, ds, dh)
    assert torch.equal(got["s"][1], t["x"][1]) and torch.equal(got["s"][4], t["x"][4])
    assert not got["h"][0].any() and torch.isfinite(got["dx"][0]).all()
    for r in (1, 2, 3, 4):
        assert not got["dgate"][r].any()
    want = reference(t, ds, dh)
    for k in ("s", "h", "dx", "dy"):
        check(got[k][1:], tuple(v[1:] if torch.is_tensor(v) else v for v in want[k]), 48, k)
    with torch.no_grad():
        t["y"][6, 5] = float("nan")
        t["x"][7, 3] = float("inf")
    bad = run(t, ds, dh)
    rest = [i for i in range(12) if i not in (6, 7)]
    for k in ("s", "h", "dx", "dy", "dgate"):
        assert torch.equal(bad[k][rest], got[k][rest]), k
        assert not torch.isfinite(bad[k][6]).all() or k == "dgate"
    assert torch.isnan(bad["h"][6]).all()


def test_no_rows():
    t, ds, dh = inputs(0, 16, torch.float32)
    got = run(t, ds, dh)
    assert got["s"].shape == (0, 16) and got["dx"].shape == (0, 16)
    for k in ("dw", "dpost", "dscale"):
        assert got[k].shape == (16,) and not got[k].any()


def test_gradients_against_differences():
    """Central differences of the formula in float64, which is also what the gradients are compared
    with elsewhere: h = 1e-4 leaves a truncation of h^2 and a rounding of 1e-16 / h, both under 1e-7 of
    the sizes here (all derivatives of the formula up to the third are under 30 on these inputs)."""
    t, ds, dh = inputs(3, 6, torch.float32)
    got = run(t, ds, dh)

    def loss(u):
        v = u["y"] / torch.sqrt((u["y"] ** 2).mean(1, keepdim=True) + EPS) * u["post"] * torch.sigmoid(u["gate"]) * u["scale"]
        s = u["x"] + v
        h = s / torch.sqrt((s ** 2).mean(1, keepdim=True) + EPS) * u["w"]
        return float((s * ds.double().cpu()).sum() + (h * dh.double().cpu()).sum())

    want = reference(t, ds, dh)
    base = {k: v.detach().double().cpu() for k, v in t.items()}
    for k in base:
        ref, size, terms = want[NAMES[k]]
        for i in range(base[k].numel()):
            flat = base[k].view(-1)
            keep = float(flat[i])
            flat[i] = keep + 1e-4
            up = loss(base)
            flat[i] = keep - 1e-4
            down = loss(base)
            flat[i] = keep
            tol = (2 * 6 + 200 + 2 * terms) * U * float(size.reshape(-1)[i]) + 1e-6
            assert abs((up - down) / 2e-4 - float(got[NAMES[k]].view(-1)[i])) <= tol, (k, i)


def test_replays_as_a_graph_and_on_another_stream():
    t, ds, dh = inputs(3000, 200, torch.bfloat16)
    names = list(t)

    def step():
        outs = forward(t)
        return [*outs, *torch.autograd.grad(outs, [t[k] for k in names], [ds, dh])]

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
            t["x"].copy_(torch.randn_like(t["x"]))
            dh.copy_(torch.randn_like(dh))
        torch.cuda.synchronize()
        want = [v.detach().clone() for v in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(static, want):
            assert torch.equal(a, c), trial


def test_refusals():
    from jittorgeometric_amd import JgamdError
    from jittorgeometric_amd.nn import residual_norm, rms_norm
    t, _, _ = inputs(6, 8, torch.float32)
    x, y, w, g = t["x"], t["y"], t["w"], t["gate"]
    for args, kw in (((x[0], y[0], w), {}), ((x, y[:, :4], w), {}), ((x, y, w[:4]), {}), ((x, y.bfloat16(), w), {}),
                     ((x, y, w), {"gate": g[:1]}), ((x, y, w), {"scale": w[:1]}), ((x, y, w), {"post_weight": w.bfloat16()}),
                     ((x.half(), y.half(), w.half()), {}), ((x, None, w), {}), ((x, y, w), {"eps": -1.0}),
                     ((x, y, w), {"eps": float("nan")}), ((x.cpu(), y, w), {}), ((x[:, :0], y[:, :0], w[:0]), {})):
        with pytest.raises(JgamdError):
            residual_norm(*args, **kw)
    wide = torch.zeros(1, 8193, device=dev())
    with pytest.raises(JgamdError):
        rms_norm(wide, wide[0])
