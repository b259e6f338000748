"""nn.rms_norm on more rows than one dimension of a launch counts threads for."""
import pytest
import torch

from util import dev

pytestmark = pytest.mark.gpu


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
