"""nn.residual_norm and nn.rms_norm on rows far from one, with open gates and on more rows than one
dimension of a launch counts.  Formulas and tolerances are those of test_gpu_norm.py: every size there is
an expression in the rows themselves, so that it follows them to any magnitude."""
import pytest
import torch

import test_gpu_norm as norm
from test_gpu_norm import check, inputs, reference, run
from util import dev

pytestmark = pytest.mark.gpu

DTYPES = norm.DTYPES


def scaled(t, rows, by):
    with torch.no_grad():
        for k, c in by.items():
            if t[k] is not None:
                t[k][rows] *= c
    return t


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("options", ["", "pgk"])
@pytest.mark.parametrize("by", [{"x": 1e15, "y": 1e15}, {"x": 1e17, "y": 1e17}, {"x": 1e17}, {"y": 1e17}, {"x": 1e-13, "y": 1e17}])
def test_large_rows(by, options, dtype):
    """Squares of 1e17 and their sums over a row of 256 are far inside float32's range."""
    t, ds, dh = inputs(24, 256, dtype, options)
    t = scaled(t, slice(3, 20), by)
    got, want = run(t, ds, dh), reference(t, ds, dh)
    for k in got:
        check(got[k], want[k], 256, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("options", ["", "pgk"])
@pytest.mark.parametrize("c", [1e-13, 1e-16])
def test_small_rows_without_eps(c, options, dtype, monkeypatch):
    monkeypatch.setattr(norm, "EPS", 0.0)
    t, ds, dh = inputs(24, 256, dtype, options)
    t = scaled(t, slice(None), {"x": c, "y": c, "scale": c} if options else {"x": c, "y": c})
    got, want = run(t, ds, dh), reference(t, ds, dh)
    for k in got:
        check(got[k], want[k], 256, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c,eps", [(1e15, 1e-6), (1e17, 1e-6), (1e-13, 0.0)])
def test_rms_norm_of_large_and_small_rows(c, eps, dtype, monkeypatch):
    monkeypatch.setattr(norm, "EPS", eps)
    t, _, dh = inputs(30, 300, dtype, "", block=False)
    t = scaled(t, slice(None), {"x": c})
    got, want = run(t, None, dh), reference(t, None, dh)
    for k in got:
        check(got[k], want[k], 300, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("F", [72, 1001])
def test_gradient_of_gates_far_open_and_far_shut(F, dtype):
    """dgate = dv u sigmoid(-gate): its error is relative to that product, however small the last factor
    is, times 1 + |gate| for the argument of the exponential."""
    t, ds, dh = inputs(41, F, dtype, "pgk")
    with torch.no_grad():
        t["gate"].copy_(torch.linspace(-60, 60, 41)[:, None].expand(41, F))
    got, want = run(t, ds, dh), reference(t, ds, dh)
    gate, y, p, k = (t[n].detach().double().cpu() for n in ("gate", "y", "post", "scale"))
    shut = torch.sigmoid(-gate)
    u = y / torch.sqrt((y * y).mean(1, keepdim=True) + norm.EPS) * p
    dv = want["dx"][0] * k * torch.sigmoid(gate)
    check(got["dgate"], (dv * u * shut, want["dgate"][1] * shut, 0), F, "dgate")
    for name in ("s", "h", "dx", "dy"):
        check(got[name], want[name], F, name)


def test_more_rows_than_threads_in_one_dimension():
    """2^29 + 3 rows of eight: eight lanes each pass 2^32."""
    from jittorgeometric_amd.nn import rms_norm
    R = 2 ** 29 + 3
    block = torch.randn(4099, 8, generator=torch.Generator(device=dev()).manual_seed(1), device=dev()).to(torch.bfloat16)
    x = torch.empty(R, 8, dtype=torch.bfloat16, device=dev())
    for at in range(0, R, 4099 * 1024):
        part = x[at:at + 4099 * 1024]
        part.copy_(block.repeat(1024, 1)[:part.shape[0]])
    w = torch.linspace(0.5, 2, 8, device=dev()).to(torch.bfloat16)
    h, want = rms_norm(x, w), rms_norm(block, w)      # a row is the same arithmetic wherever it lies
    for at in (0, 2 ** 28 // 4099 * 4099, R // 4099 * 4099 - 4099, R // 4099 * 4099):
        part = h[at:at + 4099]
        assert torch.equal(part, want[:part.shape[0]]), at
