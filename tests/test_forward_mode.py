"""Forward-mode derivatives of the operators that skip their autograd function where no input needs a
gradient: none has a forward-mode formula, so a call with a tangent raises and never returns a result
without one.  On the CPU, the library's calls replaced by nothing."""
import pytest
import torch
from torch.autograd import forward_ad


class _Nothing:
    def __getattr__(self, name):
        return lambda *args: 0


@pytest.fixture
def no_library(monkeypatch):
    from jittorgeometric_amd import _lib
    monkeypatch.setattr(_lib, "load", _Nothing)
    monkeypatch.setattr(_lib, "require_gpu", lambda *tensors: tensors[0].device)
    monkeypatch.setattr(_lib, "stream_ptr", lambda device: None)
    monkeypatch.setattr(_lib, "query", lambda fn, *args: 16)


def calls():
    from jittorgeometric_amd.nn import cross_entropy_loss, linear_cross_entropy, residual_norm, rms_norm
    from jittorgeometric_amd.ops import grouped_rows
    x, f, w = torch.ones(4, 3), torch.ones(3), torch.ones(2, 3, 5)
    off, t = torch.tensor([0, 2, 4], dtype=torch.int32), torch.tensor([0, 1, 2, 1])
    return {
        "grouped_rows, x": (x, lambda v: grouped_rows(v, w, off)),
        "grouped_rows, weight": (w, lambda v: grouped_rows(x, v, off)),
        "grouped_rows, bias": (torch.ones(2, 5), lambda v: grouped_rows(x, w, off, bias=v)),
        "linear_cross_entropy, x": (x, lambda v: linear_cross_entropy(v, w[0].t(), t)),
        "linear_cross_entropy, strided weight": (w[0], lambda v: linear_cross_entropy(x, v.t(), t)),
        "linear_cross_entropy, bias": (torch.ones(5), lambda v: linear_cross_entropy(x, w[0].t(), t, bias=v)),
        "rms_norm, x": (x, lambda v: rms_norm(v, f)),
        "rms_norm, weight": (f, lambda v: rms_norm(x, v)),
        "residual_norm, y": (x, lambda v: residual_norm(x, v, f)),
        "residual_norm, gate": (x, lambda v: residual_norm(x, x, f, gate=v)),
        "residual_norm, scale": (f, lambda v: residual_norm(x, x, f, scale=v)),
        "residual_norm, post_weight": (f, lambda v: residual_norm(x, x, f, post_weight=v)),
        "cross_entropy_loss": (x, lambda v: cross_entropy_loss(v, t)),
    }


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", sorted(calls()))
def test_a_tangent_is_refused(no_library, name, grad):
    v, call = calls()[name]
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            call(forward_ad.make_dual(v, torch.ones_like(v)))


@pytest.mark.parametrize("name", sorted(calls()))
def test_without_a_tangent_the_call_is_direct(no_library, name):
    v, call = calls()[name]
    out = call(v)
    with forward_ad.dual_level():      # an open level alone changes nothing
        again = call(v)
    for o in (out, again):
        o = o[0] if isinstance(o, tuple) else o
        assert not o.requires_grad and forward_ad.unpack_dual(o).tangent is None
