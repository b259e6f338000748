"""nn.linear_cross_entropy on more pieces of its operands than one dimension of a launch counts threads for."""
import pytest
import torch

from util import dev

pytestmark = pytest.mark.gpu


def test_more_pieces_than_threads_in_one_dimension():
    """Rows of 17 bfloat16 are laid out anew in three pieces of 8, a thread each: 2^32 / 3 rows pass 2^32.
    Every row's loss is that of the formula within float32's rounding of its 17 + 3 terms (under 64 u of
    their absolute sum, which is under 2^8)."""
    from jittorgeometric_amd.nn import linear_cross_entropy
    V, F, C, n = 2 ** 32 // 3 + 100_000, 17, 3, 1 << 20
    gen = torch.Generator(device=dev()).manual_seed(1)
    block = torch.randn(n, F, generator=gen, device=dev()).to(torch.bfloat16)
    w = torch.randn(C, F, generator=gen, device=dev()).to(torch.bfloat16)
    x = torch.empty(V, F, dtype=torch.bfloat16, device=dev())
    t = torch.empty(V, dtype=torch.int32, device=dev())
    for at in range(0, V, n):
        x[at:at + n] = block[:min(n, V - at)]
        t[at:at + n] = torch.arange(min(n, V - at), device=dev()) % 4 - 1
    loss = linear_cross_entropy(x, w, t, reduction="none")
    del x
    z = torch.mm(block.double(), w.double().t())
    label = torch.arange(n, device=dev()) % 4 - 1
    want = torch.logsumexp(z, 1) - z.gather(1, label.clamp(min=0)[:, None])[:, 0]
    want = torch.where(label >= 0, want, 0)
    assert (torch.mm(block.double().abs(), w.double().abs().t()) < 2 ** 8).all()
    for at in range(0, V, n):
        part = loss[at:at + n]
        assert ((part.double() - want[:part.shape[0]]).abs() <= 64 * 2.0 ** -24 * 2 ** 8).all(), at
