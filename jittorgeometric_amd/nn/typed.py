"""The layers' dense transform with a weight per type of row."""
import torch
from torch import nn

from ..ops.grouped import grouped_rows
from .inits import glorot, zeros


class TypedLinear(nn.Module):
    """out[r] = x[r] @ weight[type of r] + bias[type of r] for rows sorted by type: type g has the rows
    offsets[g] .. offsets[g+1] - 1.  Parameters as in the conv layers ([in, out] weights, glorot;
    zero bias), one per type."""

    def __init__(self, in_channels, out_channels, types, bias=True):
        super().__init__()
        self.in_channels, self.out_channels, self.types = in_channels, out_channels, types
        self.weight = nn.Parameter(torch.empty(types, in_channels, out_channels))
        self.bias = nn.Parameter(torch.empty(types, out_channels)) if bias else None
        self.reset_parameters()

    def reset_parameters(self):
        glorot(self.weight)
        zeros(self.bias)

    def forward(self, x, offsets):
        return grouped_rows(x, self.weight, offsets, bias=self.bias)

    execute = forward

    def __repr__(self):
        return "{}({}, {}, types={})".format(self.__class__.__name__, self.in_channels, self.out_channels, self.types)
