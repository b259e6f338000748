"""Norms around a residual block, fused with its gate and residual scale (csrc/residual_norm.hip):
one pass over the rows forward, one backward.  The residual sums of the reference's deep layers
(nn/conv/gcn2_conv.py:70-73) are plain additions; these keep a deeper stack's rows in range."""
import torch
from torch.autograd.function import once_differentiable

from .. import _lib


def _forward(x, y, w, post, gate, scale, eps, for_backward):
    """(s, h, ry, rs): s None without y, the inverse norms only for a backward pass."""
    lib = _lib.load()
    dev = x.device
    R, F = x.shape
    s = torch.empty_like(x) if y is not None else None
    h = torch.empty_like(x)
    rs = torch.empty(R, dtype=torch.float32, device=dev) if for_backward else None
    ry = torch.empty(R, dtype=torch.float32, device=dev) if for_backward and post is not None else None
    with _lib.on(dev):
        _lib.check(lib.jgamd_residual_norm_fwd(_lib.ptr(x), _lib.ptr(y), _lib.ptr(gate), _lib.ptr(scale), _lib.ptr(post),
                                               _lib.ptr(w), _lib.ptr(s), _lib.ptr(h), _lib.ptr(ry), _lib.ptr(rs), R, F, eps,
                                               _lib.dtype_code(x.dtype), _lib.stream_ptr(dev)))
    return s, h, ry, rs


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, w, post, gate, scale, eps):
        s, h, ry, rs = _forward(x, y, w, post, gate, scale, eps, True)
        ctx.save_for_backward(x, y, w, post, gate, scale, ry, rs)
        ctx.set_materialize_grads(False)
        return h if y is None else (s, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, *upstream):
        x, y, w, post, gate, scale, ry, rs = ctx.saved_tensors
        ds, dh = upstream if y is not None else (None, upstream[0])
        lib = _lib.load()
        dev = x.device
        R, F = x.shape
        ds, dh = (None if t is None else t.contiguous() for t in (ds, dh))
        grads = [torch.empty_like(t) if t is not None and need else None
                 for t, need in zip((x, y, w, post, gate, scale), ctx.needs_input_grad)]
        dx, dy, dw, dpost, dgate, dscale = grads
        nbytes = _lib.query(lib.jgamd_residual_norm_bwd_workspace, R, F)
        ws = _lib.workspace(nbytes, dev)
        with _lib.on(dev):
            _lib.check(lib.jgamd_residual_norm_bwd(_lib.ptr(x), _lib.ptr(y), _lib.ptr(gate), _lib.ptr(scale),
                                                   _lib.ptr(post), _lib.ptr(w), _lib.ptr(ry), _lib.ptr(rs), _lib.ptr(ds),
                                                   _lib.ptr(dh), _lib.ptr(dx), _lib.ptr(dy), _lib.ptr(dgate),
                                                   _lib.ptr(dscale), _lib.ptr(dpost), _lib.ptr(dw), R, F,
                                                   _lib.dtype_code(x.dtype), _lib.ptr(ws), nbytes, _lib.stream_ptr(dev)))
        return (*grads, None)


def _apply(who, x, y, weight, post_weight, gate, scale, eps):
    _lib.require_gpu(x, y, weight, post_weight, gate, scale)
    if x.dim() != 2 or x.shape[1] == 0:
        raise _lib.JgamdError("%s: x must be [rows, features], got %s" % (who, tuple(x.shape)))
    _lib.check_int32(who, x)
    _lib.dtype_code(x.dtype)
    F = x.shape[1]
    for name, t, shape in (("y", y, tuple(x.shape)), ("gate", gate, tuple(x.shape)), ("weight", weight, (F,)),
                           ("post_weight", post_weight, (F,)), ("scale", scale, (F,))):
        if t is None:
            continue
        if tuple(t.shape) != shape:
            raise _lib.JgamdError("%s: %s must be %s, got %s" % (who, name, list(shape), tuple(t.shape)))
        if t.dtype != x.dtype:
            raise _lib.JgamdError("%s: %s is %s, x is %s" % (who, name, t.dtype, x.dtype))
    if not eps >= 0:
        raise _lib.JgamdError("%s: eps must not be negative, got %r" % (who, eps))
    x, y, weight, post_weight, gate, scale = (None if t is None else t.contiguous()
                                              for t in (x, y, weight, post_weight, gate, scale))
    if not _lib.needs_grad(x, y, weight, post_weight, gate, scale):
        s, h, _, _ = _forward(x, y, weight, post_weight, gate, scale, float(eps), False)
        return h if y is None else (s, h)
    return _ResidualNorm.apply(x, y, weight, post_weight, gate, scale, float(eps))


def rms_norm(x, weight, eps=1e-6):
    """x / sqrt(mean(x^2) + eps) * weight over the rows of x [rows, features]; weight [features]."""
    return _apply("rms_norm", x, None, weight, None, None, None, eps)


def residual_norm(x, y, weight, post_weight=None, gate=None, scale=None, eps=1e-6):
    """The end of a residual block with input x and output y, and the norm in front of the next:

        s = x + scale * sigmoid(gate) * rms(y) * post_weight,    h = rms(s) * weight

    with rms(v) = v / sqrt(mean(v^2) + eps) over a row.  Returns (s, h): the residual stream and the
    next block's input.  x, y, gate are [rows, features], weight, post_weight, scale [features], all
    float32 or all bfloat16; without post_weight y is added as it is, without gate or scale their
    factor is 1.  Everything is computed in float32 and rounded once.  At most 8192 features."""
    if y is None:
        raise _lib.JgamdError("residual_norm: y is None; rms_norm is the norm without a block before it")
    return _apply("residual_norm", x, y, weight, post_weight, gate, scale, eps)
