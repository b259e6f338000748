"""Product of rows with the weight of their type (csrc/grouped_rows.hip): rows sorted by type with
offsets, as the conversions sort edges by destination (`row_offset` of a CSR).  The layers' x @ W
(nn/conv/gcn_conv.py:95 in the reference) is the case of one type."""
import torch
from torch.autograd.function import once_differentiable

from .. import _lib

_WEIGHT_TRANSPOSED = 1


def _product(x, weight, bias, offsets, transposed):
    lib = _lib.load()
    M, K = x.shape
    G = weight.shape[0]
    N = weight.shape[1 if transposed else 2]
    out = torch.empty((M, N), dtype=x.dtype, device=x.device)
    with _lib.on(x.device):
        _lib.check(lib.jgamd_grouped_rows(_lib.ptr(x), _lib.ptr(weight), _lib.ptr(bias), _lib.ptr(offsets), _lib.ptr(out),
                                          M, K, N, G, _lib.dtype_code(x.dtype), _WEIGHT_TRANSPOSED if transposed else 0,
                                          _lib.stream_ptr(x.device)))
    return out


class _GroupedRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, offsets):
        ctx.save_for_backward(x, weight, offsets)
        return _product(x, weight, bias, offsets, False)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        x, weight, offsets = ctx.saved_tensors
        gx = gw = gb = None
        g = g.contiguous()
        if ctx.needs_input_grad[0]:
            gx = _product(g, weight, None, offsets, True)
        if ctx.needs_input_grad[1] or ctx.needs_input_grad[2]:
            lib = _lib.load()
            dev = x.device
            M, K = x.shape
            G, _, N = weight.shape
            gw = torch.empty((G, K, N), dtype=x.dtype, device=dev)
            gb = torch.empty((G, N), dtype=x.dtype, device=dev) if ctx.needs_input_grad[2] else None
            nbytes = _lib.query(lib.jgamd_grouped_rows_weight_grad_workspace, M, K, N, G)
            ws = _lib.workspace(nbytes, dev)
            with _lib.on(dev):
                _lib.check(lib.jgamd_grouped_rows_weight_grad(_lib.ptr(x), _lib.ptr(g), _lib.ptr(offsets), _lib.ptr(gw),
                                                              _lib.ptr(gb), M, K, N, G, _lib.dtype_code(x.dtype),
                                                              _lib.ptr(ws), nbytes, _lib.stream_ptr(dev)))
        return gx, gw, gb, None


def grouped_rows(x, weight, offsets, bias=None):
    """out[r] = x[r] @ weight[g] (+ bias[g]) for offsets[g] <= r < offsets[g+1].

    x [rows, Fin], weight [types, Fin, Fout], bias [types, Fout] or None, all float32 or all bfloat16;
    offsets [types + 1], integers on the GPU, where they stay: nothing waits for the device.  Rows of
    no type (before offsets[0], from offsets[types] on) give zero rows and get zero gradients; a type
    may have no rows.  Offsets that fall or leave [0, rows] are read as their running maximum clamped
    to that range.  Sums are held in float32; a float32 product keeps float32's 24 bits (of entries from
    2^-103 on; below, an absolute 2^-126).  An infinity or a NaN makes the results it enters infinite or NaN:
    in float32 NaN, except where few rows read the weights on the vector unit."""
    _lib.require_gpu(x, weight, offsets, bias)
    if x.dim() != 2 or weight.dim() != 3 or weight.shape[1] != x.shape[1]:
        raise _lib.JgamdError("grouped_rows: x must be [rows, Fin] and weight [types, Fin, Fout], got %s and %s"
                              % (tuple(x.shape), tuple(weight.shape)))
    if 0 in weight.shape:
        raise _lib.JgamdError("grouped_rows: weight has no elements: %s" % (tuple(weight.shape),))
    if offsets.dim() != 1 or offsets.shape[0] != weight.shape[0] + 1:
        raise _lib.JgamdError("grouped_rows: offsets must be [types + 1] = [%d], got %s"
                              % (weight.shape[0] + 1, tuple(offsets.shape)))
    if offsets.dtype not in (torch.int32, torch.int64):
        raise _lib.JgamdError("grouped_rows: offsets must be int32 or int64, got %s" % offsets.dtype)
    if bias is not None and tuple(bias.shape) != (weight.shape[0], weight.shape[2]):
        raise _lib.JgamdError("grouped_rows: bias must be [types, Fout] = [%d, %d], got %s"
                              % (weight.shape[0], weight.shape[2], tuple(bias.shape)))
    _lib.check_int32("grouped_rows", x, weight)
    _lib.dtype_code(x.dtype)
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.dtype != x.dtype:
            raise _lib.JgamdError("grouped_rows: %s is %s, x is %s" % (name, t.dtype, x.dtype))
    if offsets.dtype == torch.int64:      # beyond int32 is past the last row anyway
        offsets = offsets.clamp(0, 2**31 - 1).to(torch.int32)
    x, weight, offsets = x.contiguous(), weight.contiguous(), offsets.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    if not _lib.needs_grad(x, weight, bias):
        return _product(x, weight, bias, offsets, False)
    return _GroupedRows.apply(x, weight, bias, offsets)
