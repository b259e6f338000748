"""nn.linear_cross_entropy in float32 on operands of very different sizes."""
import pytest
import torch

from test_gpu_class_head import inputs, run
from util import dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [1, 8, 32])
@pytest.mark.parametrize("F,C,spread", [(2000, 3000, 3e6), (256, 3000, 1e7), (2000, 700, 3e5), (64, 5000, 1e6)])
def test_few_rows_with_large_logits(V, F, C, spread):
    """Logits so large that their last bit is of the size of one: z - lse may come out over zero where the
    two sums round apart.  A probability is still none over one: with one labelled row and g = 1, db is d."""
    for seed in range(4):
        x, w, b, t, g = inputs(V, F, C, torch.float32, seed=seed, spread=spread, unlabelled=False)
        got = run(x, w, b, t, torch.ones_like(g), "none")
        for k in got:
            assert torch.isfinite(got[k]).all(), k
        row = seed % V
        t = torch.where(torch.arange(V, device=dev()) == row, t, -1)
        got = run(x, w, b, t, torch.ones_like(g), "none")
        for k in got:
            assert torch.isfinite(got[k]).all(), k
        assert got["db"].abs().max() <= 1


@pytest.mark.parametrize("V", [8, 100, 3000])
def test_large_logits_in_bfloat16(V):
    """Both passes sum a bfloat16 logit in the same order, so that z - lse is never over zero."""
    x, w, b, t, g = inputs(V, 512, 3000, torch.bfloat16, spread=1e7, unlabelled=False)
    for row in (0, V - 1, V // 2):
        got = run(x, w, b, torch.where(torch.arange(V, device=dev()) == row, t, -1), torch.ones_like(g), "none")
        for k in got:
            assert torch.isfinite(got[k]).all(), k
        assert got["db"].abs().max() <= 1
