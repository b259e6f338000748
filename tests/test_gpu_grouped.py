"""The typed product (ops.grouped_rows, nn.TypedLinear) against the same sums in float64.

Tolerances, with u = 2^-24 and S the sum of the absolute terms of a result: n terms are added one
by one in float32 by an adder that may truncate (2 u of a partial sum, which S bounds), float32
factors enter as parts that hold their 24 bits (dropped products of parts: under 4 u of a term in
all), so |error| <= (2 n + 16) u S; a result rounded to bfloat16 is off by 2^-8 of itself more."""
import numpy as np
import pytest
import torch

from util import dev

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16]


def clean(offsets, M):
    return np.maximum.accumulate(np.clip(np.asarray(offsets, dtype=np.int64), 0, M))


def reference(x, w, b, offsets, dout):
    """(results, sums of absolute terms, terms) of out, dx, dw, db in float64."""
    x, w, dout = (t.detach().double().cpu() for t in (x, w, dout))
    b = None if b is None else b.detach().double().cpu()
    M, K = x.shape
    G, _, N = w.shape
    off = clean(offsets, M)
    out, sout = torch.zeros(M, N).double(), torch.zeros(M, N).double()
    dx, sdx = torch.zeros(M, K).double(), torch.zeros(M, K).double()
    dw, sdw = torch.zeros(G, K, N).double(), torch.zeros(G, K, N).double()
    db, sdb = torch.zeros(G, N).double(), torch.zeros(G, N).double()
    most = 0
    for g in range(G):
        r = slice(int(off[g]), int(off[g + 1]))
        most = max(most, r.stop - r.start)
        out[r], sout[r] = x[r] @ w[g], x[r].abs() @ w[g].abs()
        if b is not None:
            out[r] += b[g]
            sout[r] += b[g].abs()
        dx[r], sdx[r] = dout[r] @ w[g].t(), dout[r].abs() @ w[g].abs().t()
        dw[g], sdw[g] = x[r].t() @ dout[r], x[r].abs().t() @ dout[r].abs()
        db[g], sdb[g] = dout[r].sum(0), dout[r].abs().sum(0)
    return {"out": (out, sout, K + 1), "dx": (dx, sdx, N), "dw": (dw, sdw, most), "db": (db, sdb, most)}


def check(got, want, what):
    ref, size, terms = want
    tol = (2 * terms + 16) * U * size
    if got.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (ref.abs() + tol)
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, what
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), "%s: %d of %d off, first at %s" % (what, int(bad.sum()), bad.numel(), bad.nonzero()[0].tolist())


def inputs(M, K, N, G, dtype, seed=0, bias=True):
    g = torch.Generator().manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=g).to(dtype).to(dev()).requires_grad_(True)

    return rand(M, K), rand(G, K, N), rand(G, N) if bias else None, rand(M, N).detach()


def run(x, w, b, offsets, dout):
    from jittorgeometric_amd.ops import grouped_rows
    off = torch.tensor(np.asarray(offsets), dtype=torch.int32, device=dev())
    out = grouped_rows(x, w, off, bias=b)
    grads = torch.autograd.grad(out, [t for t in (x, w, b) if t is not None], dout)
    return dict(zip(["out", "dx", "dw", "db"], [out, *grads]))


def offsets_of(sizes, start=0):
    return [start + int(v) for v in np.concatenate([[0], np.cumsum(sizes)])]


SHAPES = [
    (1, 1, [1]), (3, 2, [2, 0, 3]), (8, 8, [1]), (16, 300, [5, 0, 0, 128]), (129, 200, [0, 100, 1, 199]),
    (31, 33, [127, 1, 129]), (72, 64, [64] * 5), (256, 256, [1] * 16), (100, 47, [257, 0, 515, 3]),
    (64, 7, list(range(70))), (512, 136, [40, 3]), (7, 513, [0, 33]),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,N,sizes", SHAPES)
def test_results_and_gradients(K, N, sizes, dtype):
    M = sum(sizes)
    off = offsets_of(sizes)
    x, w, b, dout = inputs(M, K, N, len(sizes), dtype, seed=K + N)
    got = run(x, w, b, off, dout)
    want = reference(x, w, b, off, dout)
    for k in got:
        check(got[k], want[k], k)
    got = run(x, w, None, off, dout)
    want = reference(x, w, None, off, dout)
    for k in got:
        check(got[k], want[k], k + " without bias")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", [[20011, 0, 255, 256, 257], [1, 30000], [9000]])
def test_weight_gradient_of_many_rows_is_summed_in_pieces(sizes, dtype):
    M = sum(sizes)
    off = offsets_of(sizes)
    x, w, b, dout = inputs(M, 24, 40, len(sizes), dtype)
    got, again = run(x, w, b, off, dout), run(x, w, b, off, dout)
    want = reference(x, w, b, off, dout)
    for k in got:
        check(got[k], want[k], k)
        assert torch.equal(got[k], again[k]), k


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("K,N", [(24, 40), (33, 47), (72, 264), (40, 128), (129, 100), (264, 72), (100, 129)])
def test_more_rows_than_small_tiles_take(K, N, bias, dtype):
    sizes = [20001, 0, 30011, 1, 127, 255]
    x, w, b, dout = inputs(sum(sizes) + 7, K, N, len(sizes), dtype, bias=bias)
    off = offsets_of(sizes, start=3)
    got, want = run(x, w, b, off, dout), reference(x, w, b, off, dout)
    names = ["out", "dx", "dw", "db"] if bias else ["out", "dx", "dw"]
    for k in names:
        check(got[k], want[k], k)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_no_type_are_zero_and_not_read(dtype):
    M, K, N = 300, 40, 24
    off = [7, 7, 150, 280]
    x, w, b, dout = inputs(M, K, N, 3, dtype)
    with torch.no_grad():
        for t in (x, dout):
            t[:7] = float("nan")
            t[280:] = float("inf")
    got = run(x, w, b, off, dout)
    for k in ("out", "dx"):
        assert not got[k][:7].any() and not got[k][280:].any()
    with torch.no_grad():
        for t in (x, dout):
            t[:7] = 0
            t[280:] = 0
    want = reference(x, w, b, off, dout)
    for k in got:
        check(got[k], want[k], k)


@pytest.mark.parametrize("offsets", [[0, 50, 20, 100], [-5, 30, 60, 400], [90, 10, 10, 10], [200, 300, 400, 500],
                                     [-3, -2, -1, 0]])
def test_offsets_that_fall_or_leave_the_rows_are_clamped(offsets):
    M, K, N = 100, 12, 20
    x, w, b, dout = inputs(M, K, N, 3, torch.float32)
    got = run(x, w, b, offsets, dout)
    want = reference(x, w, b, offsets, dout)
    for k in got:
        check(got[k], want[k], k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_bad_entry_stays_in_its_row_and_its_type(dtype, bad):
    sizes, K, N = [60, 70, 50], 37, 45
    off = offsets_of(sizes)
    x, w, b, dout = inputs(180, K, N, 3, dtype)
    want = reference(x, w, b, off, dout)
    with torch.no_grad():
        x[65, 36] = bad
    got = run(x, w, b, off, dout)
    assert not torch.isfinite(got["out"][65]).any()
    assert not torch.isfinite(got["dw"][1, 36]).any()
    keep = torch.ones(180, dtype=torch.bool)
    keep[65] = False
    check(got["out"][keep.to(dev())], tuple(t[keep] if torch.is_tensor(t) else t for t in want["out"]), "out")
    check(got["dx"], want["dx"], "dx")
    ref, size, n = want["dw"]
    check(got["dw"][:, :36], (ref[:, :36], size[:, :36], n), "dw")
    check(got["dw"][[0, 2]], (ref[[0, 2]], size[[0, 2]], n), "dw")


def test_strides_offsets_types_and_unaligned_starts():
    from jittorgeometric_amd.ops import grouped_rows
    sizes, K, N = [30, 0, 41], 20, 36
    M, off = sum(sizes), offsets_of(sizes)
    for dtype in DTYPES:
        x, w, b, dout = inputs(M, K, N, 3, dtype)
        want = reference(x, w, b, off, dout)
        xs = torch.empty(K, M + 3, dtype=dtype, device=dev()).t()[:M]
        xs.copy_(x.detach())
        ws = w.detach().transpose(1, 2).contiguous().transpose(1, 2)
        store = torch.empty(M * K + 1, dtype=dtype, device=dev())
        x1 = store[1:].view(M, K)
        x1.copy_(x.detach())
        wstore = torch.empty(w.numel() + 3, dtype=dtype, device=dev())
        w1 = wstore[3:].view(w.shape)
        w1.copy_(w.detach())
        for xx, ww in ((xs, ws), (x1, w1)):
            xx, ww = xx.requires_grad_(True), ww.requires_grad_(True)
            for ot in (torch.int32, torch.int64):
                out = grouped_rows(xx, ww, torch.tensor(off, dtype=ot, device=dev()), bias=b)
                gx, gw = torch.autograd.grad(out, [xx, ww], dout.t().contiguous().t())
                check(out, want["out"], "out")
                check(gx, want["dx"], "dx")
                check(gw, want["dw"], "dw")
        # a gradient without memory of its own
        out = grouped_rows(x, w, torch.tensor(off, dtype=torch.int32, device=dev()))
        gx, gw = torch.autograd.grad(out.sum(), [x, w])
        one = torch.ones_like(dout)
        ref = reference(x, w, None, off, one)
        check(gx, ref["dx"], "dx of a sum")
        check(gw, ref["dw"], "dw of a sum")


def test_no_rows():
    from jittorgeometric_amd.ops import grouped_rows
    x, w, b, dout = inputs(0, 8, 12, 2, torch.float32)
    got = run(x, w, b, [0, 0, 0], dout)
    assert got["out"].shape == (0, 12) and got["dx"].shape == (0, 8)
    assert not got["dw"].any() and not got["db"].any()
    assert grouped_rows(x.detach(), w.detach(), torch.zeros(3, dtype=torch.int32, device=dev())).shape == (0, 12)


def test_gradients_against_differences():
    """The loss is linear in each input, so a central difference has no truncation error: what is
    left is the rounding of the two sums, each within (2 n + 16) u of its absolute terms, over 2 h."""
    sizes, K, N = [5, 0, 6], 6, 10
    off = offsets_of(sizes)
    x, w, b, dout = inputs(11, K, N, 3, torch.float32)
    got = run(x, w, b, off, dout)

    def loss():
        from jittorgeometric_amd.ops import grouped_rows
        out = grouped_rows(x.detach(), w.detach(), torch.tensor(off, dtype=torch.int32, device=dev()), bias=b.detach())
        return float((out.double() * dout.double()).sum())

    h = 0.5
    want = reference(x, w, b, off, dout)
    size = float((want["out"][1] * dout.abs().double().cpu()).sum()) + h * 40
    tol = (2 * (K + 1) + 16) * U * size / h
    for t, k in ((x, "dx"), (w, "dw"), (b, "db")):
        for i in range(0, t.numel(), 7):
            flat = t.detach().view(-1)
            keep = float(flat[i])
            flat[i] = keep + h
            up, at_up = loss(), float(flat[i])
            flat[i] = keep - h
            down, at_down = loss(), float(flat[i])
            flat[i] = keep
            assert abs((up - down) / (at_up - at_down) - float(got[k].view(-1)[i])) <= tol, (k, i)


def test_only_what_is_asked_for_and_the_layer():
    from jittorgeometric_amd.nn import TypedLinear
    torch.manual_seed(0)
    layer = TypedLinear(20, 28, 3).to(dev())
    off = torch.tensor([0, 10, 10, 35], dtype=torch.int32, device=dev())
    x = torch.randn(35, 20, device=dev())
    out = layer(x, off)
    dout = torch.randn_like(out)
    out.backward(dout)
    want = reference(x, layer.weight, layer.bias, off.cpu().numpy(), dout)
    check(out, want["out"], "out")
    check(layer.weight.grad, want["dw"], "dw")
    check(layer.bias.grad, want["db"], "db")
    assert not layer.weight.grad[1].any()
    half = layer.to(torch.bfloat16)(x.bfloat16(), off)
    assert half.dtype == torch.bfloat16
    xg = x.clone().requires_grad_(True)
    from jittorgeometric_amd.ops import grouped_rows
    w = torch.randn(3, 20, 28, device=dev())
    gx, = torch.autograd.grad(grouped_rows(xg, w, off), [xg], dout)
    check(gx, reference(x, w, None, off.cpu().numpy(), dout)["dx"], "dx")


def test_forward_and_backward_replay_as_a_graph_and_on_another_stream():
    from jittorgeometric_amd.ops import grouped_rows
    sizes = [700, 0, 9, 4000]
    M, K, N, off = sum(sizes), 48, 56, offsets_of(sizes)
    o = torch.tensor(off, dtype=torch.int32, device=dev())
    x, w, b, dout = inputs(M, K, N, 4, torch.float32)

    def step():
        out = grouped_rows(x, w, o, bias=b)
        return [out, *torch.autograd.grad(out, [x, w, b], dout)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            side = [t.detach().clone() for t in step()]
    torch.cuda.current_stream().wait_stream(s)
    for a, c in zip(side, step()):
        assert torch.equal(a, c)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for trial in range(3):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
            dout.copy_(torch.randn_like(dout))
        torch.cuda.synchronize()
        want = [t.detach().clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(static, want):
            assert torch.equal(a, c), trial


def test_refusals():
    from jittorgeometric_amd import JgamdError
    from jittorgeometric_amd.ops import grouped_rows
    x, w, b, _ = inputs(10, 4, 6, 2, torch.float32)
    o = torch.tensor([0, 5, 10], dtype=torch.int32, device=dev())
    for args, kw in (((x[0], w, o), {}), ((x, w[0], o), {}), ((x[:, :3], w, o), {}), ((x, w, o[:2]), {}),
                     ((x, w, o.float()), {}), ((x, w.bfloat16(), o), {}), ((x, w, o), {"bias": b[:1]}),
                     ((x, w, o), {"bias": b.bfloat16()}), ((x.half(), w.half(), o), {}), ((x.double(), w.double(), o), {}),
                     ((x, w[:, :, :0], o), {}), ((x.cpu(), w, o), {}), ((x, w, o.cpu()), {})):
        with pytest.raises(JgamdError):
            grouped_rows(*args, **kw)
