"""Mean cross-entropy over the rows of a logits matrix: the loss of the reference's
training steps (nn.cross_entropy_loss(pred, label) in examples/gcn_example.py:113,
nn.log_softmax + nn.nll_loss in examples/sage_example.py:69,83; both functions live in
the jittor package).  Forward and gradient are one library kernel each
(csrc/loss.hip): with millions of rows and a few dozen classes a generic framework
loss spends most of its time in single-block reductions.  linear_cross_entropy is the same
loss behind a linear map onto many classes, without the logits (csrc/class_head.hip)."""
import torch
from torch.autograd.function import once_differentiable

from .. import _lib


class _CrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, output, target, log_probs):
        lib = _lib.load()
        dev = _lib.require_gpu(output, target)
        if output.dim() != 2:
            raise _lib.JgamdError("cross_entropy_loss: output must be [rows, classes], got %s" % (tuple(output.shape),))
        if target.dim() != 1 or target.shape[0] != output.shape[0]:
            raise _lib.JgamdError("cross_entropy_loss: %d labels for %d rows" % (target.numel(), output.shape[0]))
        if target.dtype not in (torch.int32, torch.int64):
            target = target.to(torch.int64)
        x = output if output.dtype == torch.float32 else output.to(torch.float32)
        x = x.contiguous()
        target = target.contiguous()
        V, C = x.shape
        loss = torch.empty((), dtype=torch.float32, device=dev)
        count = torch.empty((), dtype=torch.int32, device=dev)
        lse = torch.empty(V, dtype=torch.float32, device=dev)
        nbytes = _lib.query(lib.jgamd_cross_entropy_workspace, V, C)
        ws = _lib.workspace(nbytes, dev)
        i64 = 1 if target.dtype == torch.int64 else 0
        _lib.check(lib.jgamd_cross_entropy_fwd(_lib.ptr(x), _lib.ptr(target), i64, int(bool(log_probs)), V, C,
                                               _lib.ptr(loss), _lib.ptr(count),
                                               _lib.ptr(lse), _lib.ptr(ws), nbytes, _lib.stream_ptr(dev)))
        ctx.save_for_backward(x, target, lse, count)
        ctx.i64 = i64
        ctx.in_dtype = output.dtype
        return loss

    @staticmethod
    def backward(ctx, g):
        if not ctx.needs_input_grad[0]:
            return None, None, None
        x, target, lse, count = ctx.saved_tensors
        lib = _lib.load()
        dev = x.device
        g = g.to(torch.float32).contiguous()
        grad = torch.empty_like(x)
        V, C = x.shape
        _lib.check(lib.jgamd_cross_entropy_bwd(_lib.ptr(x), _lib.ptr(target), ctx.i64, _lib.ptr(lse), _lib.ptr(count),
                                               _lib.ptr(g), V, C, _lib.ptr(grad), _lib.stream_ptr(dev)))
        return (grad if ctx.in_dtype == torch.float32 else grad.to(ctx.in_dtype)), None, None


def cross_entropy_loss(output, target):
    """mean_i (logsumexp(output[i,:]) - output[i, target[i]]) over the rows whose label lies in
    [0, classes); the other rows are left out and get a zero gradient."""
    return _CrossEntropy.apply(output, target, False)


def nll_loss(log_probs, target):
    """mean_i -log_probs[i, target[i]] for rows of log-probabilities (the second half of
    log_softmax + nll_loss, examples/sage_example.py:69,83); the gradient is -1 / rows at the
    labels and zero elsewhere.  Same kernels, with the softmax term switched off."""
    return _CrossEntropy.apply(log_probs, target, True)


_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}      # JGAMD_LOSS_NONE, JGAMD_LOSS_MEAN, JGAMD_LOSS_SUM


def _linear_forward(x, weight, bias, target, reduction, for_backward):
    """(loss, lse, count); without a backward pass the last two are not kept (one allocation less each)."""
    lib = _lib.load()
    dev = x.device
    V, F = x.shape
    C = weight.shape[0]
    code = _lib.dtype_code(x.dtype)
    loss = torch.empty((V,) if reduction == 0 else (), dtype=torch.float32, device=dev)
    nbytes = _lib.query(lib.jgamd_linear_cross_entropy_workspace, V, F, C, code, 0)
    if for_backward:
        count = torch.empty((), dtype=torch.int32, device=dev)
        lse = torch.empty(V, dtype=torch.float32, device=dev)
        ws = _lib.workspace(nbytes, dev)
        lse_at, count_at = _lib.ptr(lse), _lib.ptr(count)
    else:
        ws = _lib.workspace(nbytes + 4 * V + 4, dev)
        lse, count, lse_at, count_at = None, None, ws.data_ptr() + nbytes, ws.data_ptr() + nbytes + 4 * V
    with _lib.on(dev):
        _lib.check(lib.jgamd_linear_cross_entropy_fwd(_lib.ptr(x), _lib.ptr(weight), _lib.ptr(bias), _lib.ptr(target),
                                                      1 if target.dtype == torch.int64 else 0, V, F, C, code, reduction,
                                                      _lib.ptr(loss), count_at, lse_at, _lib.ptr(ws), nbytes,
                                                      _lib.stream_ptr(dev)))
    return loss, lse, count


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, target, reduction):
        loss, lse, count = _linear_forward(x, weight, bias, target, reduction, True)
        ctx.save_for_backward(x, weight, bias, target, lse, count)
        ctx.reduction = reduction
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        x, weight, bias, target, lse, count = ctx.saved_tensors
        lib = _lib.load()
        dev = x.device
        V, F = x.shape
        C = weight.shape[0]
        code = _lib.dtype_code(x.dtype)
        g = g.to(torch.float32).contiguous()
        dx = torch.empty_like(x) if ctx.needs_input_grad[0] else None
        dw = torch.empty_like(weight) if ctx.needs_input_grad[1] or ctx.needs_input_grad[2] else None
        db = torch.empty_like(bias) if ctx.needs_input_grad[2] else None
        nbytes = _lib.query(lib.jgamd_linear_cross_entropy_workspace, V, F, C, code, 1)
        ws = _lib.workspace(nbytes, dev)
        with _lib.on(dev):
            _lib.check(lib.jgamd_linear_cross_entropy_bwd(_lib.ptr(x), _lib.ptr(weight), _lib.ptr(bias), _lib.ptr(target),
                                                          1 if target.dtype == torch.int64 else 0, _lib.ptr(lse),
                                                          _lib.ptr(count), _lib.ptr(g), V, F, C, code, ctx.reduction,
                                                          _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db), _lib.ptr(ws), nbytes,
                                                          _lib.stream_ptr(dev)))
        return dx, dw, db, None, None


def linear_cross_entropy(x, weight, target, bias=None, reduction="mean"):
    """cross_entropy_loss(x @ weight.t() + bias, target) without the [rows, classes] logits, in memory
    or in the workspace: for classes by the ten thousand (items, entities, words).

    x [rows, features], weight [classes, features] (a row per class, as an embedding table), bias
    [classes] or None, all float32 or all bfloat16; target [rows], int32 or int64.  Rows whose label
    lies outside [0, classes) are left out of the mean, have loss 0 and get a zero gradient.
    reduction: "mean" over the rows with a label (NaN when there is none), "sum" or "none" ([rows]);
    the loss is float32.  A class may be masked with a bias of -inf.  What a row without a label holds
    does not matter.

    Products are summed in float32.  float32 entries, and float32 gradients of the logits, keep their 24
    bits (from 2^-103 on; below, an absolute 2^-126); an infinity or a NaN makes the logits it enters NaN or
    infinite.  In bfloat16 the gradient of the logits is rounded to bfloat16 on its way into the other
    gradients, and with reduction="none" so are the rows of x times their own gradient.  The scratch
    memory of a backward pass is up to a gigabyte of gradients of logits, float32 sums of the size of
    weight, and, in float32 one and a half times their size each, copies of x and weight."""
    _lib.require_gpu(x, weight, target, bias)
    if x.dim() != 2 or weight.dim() != 2 or weight.shape[1] != x.shape[1]:
        raise _lib.JgamdError("linear_cross_entropy: x must be [rows, features] and weight [classes, features], got %s "
                              "and %s" % (tuple(x.shape), tuple(weight.shape)))
    if 0 in weight.shape:
        raise _lib.JgamdError("linear_cross_entropy: weight has no elements: %s" % (tuple(weight.shape),))
    if target.dim() != 1 or target.shape[0] != x.shape[0]:
        raise _lib.JgamdError("linear_cross_entropy: %d labels for %d rows" % (target.numel(), x.shape[0]))
    if target.dtype not in (torch.int32, torch.int64):
        raise _lib.JgamdError("linear_cross_entropy: labels must be int32 or int64, got %s" % target.dtype)
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise _lib.JgamdError("linear_cross_entropy: bias must be [%d], got %s" % (weight.shape[0], tuple(bias.shape)))
    if reduction not in _REDUCTIONS:
        raise _lib.JgamdError("linear_cross_entropy: reduction must be 'mean', 'sum' or 'none', got %r" % (reduction,))
    _lib.check_int32("linear_cross_entropy", x, weight)
    _lib.dtype_code(x.dtype)
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.dtype != x.dtype:
            raise _lib.JgamdError("linear_cross_entropy: %s is %s, x is %s" % (name, t.dtype, x.dtype))
    x, weight = (t if t.data_ptr() % 16 == 0 else t.clone() for t in (x.contiguous(), weight.contiguous()))
    if bias is not None:
        bias = bias.contiguous()
    target = target.contiguous()
    if not _lib.needs_grad(x, weight, bias):
        return _linear_forward(x, weight, bias, target, _REDUCTIONS[reduction], False)[0]
    return _LinearCrossEntropy.apply(x, weight, bias, target, _REDUCTIONS[reduction])
