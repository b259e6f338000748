"""ops.grouped_rows on more rows than one dimension of a launch counts threads for."""
import pytest
import torch

from util import dev

pytestmark = pytest.mark.gpu


def test_more_rows_than_threads_in_one_dimension():
    """2^31 - 1 rows of one float: 2^24 tiles of 128 rows, 256 threads each."""
    from jittorgeometric_amd.ops import grouped_rows
    M, cut = 2 ** 31 - 1, 2 ** 30 + 77
    x = torch.empty(M, 1, device=dev())
    block = torch.randn(1 << 20, 1, generator=torch.Generator(device=dev()).manual_seed(1), device=dev())
    for at in range(0, M, 1 << 20):
        part = x[at:at + (1 << 20)]
        part.copy_(block[:part.shape[0]])
    w = torch.tensor([[[2.0]], [[-0.5]]], device=dev())
    out = grouped_rows(x, w, torch.tensor([0, cut, M], dtype=torch.int32, device=dev()))
    for a, b, by in ((0, cut, 2.0), (cut, M, -0.5)):      # a product with a power of two is exact
        for at in range(a, b, 1 << 26):
            to = min(b, at + (1 << 26))
            assert torch.equal(out[at:to], by * x[at:to]), at
