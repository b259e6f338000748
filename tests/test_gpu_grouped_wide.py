"""The typed product in bfloat16 in its widest tiles (256 x 256), over several steps of k, ragged ones,
several tiles of columns and of rows a workgroup and several pieces of a weight gradient; and at widths
next to those where narrower tiles take over.  Formulas and tolerances are those of test_gpu_grouped.py."""
import pytest
import torch

from test_gpu_grouped import check, inputs, offsets_of, reference, run
from util import dev

pytestmark = pytest.mark.gpu

SIZES = [23011, 0, 255, 256, 257, 9001, 1, 7300]


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("K,N", [(256, 256), (264, 512), (512, 248), (248, 264), (256, 200), (200, 1000), (520, 776)])
def test_widest_tiles(K, N, bias):
    x, w, b, dout = inputs(sum(SIZES) + 11, K, N, len(SIZES), torch.bfloat16, seed=K + N, bias=bias)
    off = offsets_of(SIZES, start=5)
    got, again, want = run(x, w, b, off, dout), run(x, w, b, off, dout), reference(x, w, b, off, dout)
    for k in got:
        check(got[k], want[k], k)
        assert torch.equal(got[k], again[k]), k
    for k in ("out", "dx"):
        assert not got[k][:5].any() and not got[k][-6:].any()


@pytest.mark.parametrize("K,N", [(64, 64), (64, 72), (72, 64), (56, 192), (192, 128), (136, 320), (320, 136), (64, 256), (1024, 64)])
def test_widths_at_the_borders_of_the_tiles(K, N):
    x, w, b, dout = inputs(sum(SIZES), K, N, len(SIZES), torch.bfloat16, seed=K + N)
    off = offsets_of(SIZES)
    got, want = run(x, w, b, off, dout), reference(x, w, b, off, dout)
    for k in got:
        check(got[k], want[k], k)


def test_more_tiles_than_a_workgroup_keeps():
    """90 types of two tiles of rows and 200 tiles of columns: over 64 tiles for each of 256 workgroups."""
    from jittorgeometric_amd.ops import grouped_rows
    G, K, N, each = 90, 8, 200 * 256 - 8, 257
    gen = torch.Generator(device=dev()).manual_seed(1)
    x = torch.randn(G * each, K, generator=gen, device=dev()).to(torch.bfloat16)
    w = torch.randn(G, K, N, generator=gen, device=dev()).to(torch.bfloat16)
    out = grouped_rows(x, w, torch.arange(0, G * each + 1, each, dtype=torch.int32, device=dev()))
    for g in (0, 1, 44, 88, 89):
        rows = slice(g * each, (g + 1) * each)
        a, c = x[rows].double(), w[g].double()
        check(out[rows], (torch.mm(a, c).cpu(), torch.mm(a.abs(), c.abs()).cpu(), K), "type %d" % g)
