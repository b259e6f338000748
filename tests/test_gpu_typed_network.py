"""The typed product, the residual norm and the class head together, behind one of the library's graph
layers: what a network with node types and many labels runs in a step.  The reference is the same
network in float64 under torch's autograd on the CPU."""
import numpy as np
import pytest
import torch

import oracle
from util import dev, rand_graph, to_gpu

pytestmark = pytest.mark.gpu

V, F, H, C, TYPES = 300, 24, 48, 500, 4
U = 2.0 ** -24


def build(dtype=torch.float32, seed=3):
    from jittorgeometric_amd.nn import GCNConv, TypedLinear
    from jittorgeometric_amd.ops import cootocsc, cootocsr
    rng = np.random.default_rng(seed)
    ei, _ = rand_graph(rng, V, 2000, 1)
    ei = ei[:, ei[0] != ei[1]]
    ei, w = oracle.gcn_norm(ei, None, V)
    ei = ei.astype(np.int32)
    net = {"csc": cootocsc(to_gpu(ei), to_gpu(w), V), "csr": cootocsr(to_gpu(ei), to_gpu(w), V)}
    A = torch.zeros(V, V, dtype=torch.float64)
    A.index_put_((torch.from_numpy(ei[1]).long(), torch.from_numpy(ei[0]).long()), torch.from_numpy(w).double(), accumulate=True)
    torch.manual_seed(seed)
    net["conv"] = GCNConv(F, H, spmm=False).to(dev())
    net["typed"] = [TypedLinear(H, H, TYPES).to(dev()).to(dtype) for _ in range(2)]

    def param(*shape, mul=0.2, add=0.0):
        return (torch.randn(*shape, device=dev()) * mul + add).to(dtype).requires_grad_(True)

    net["norm"] = [param(H, add=1.0) for _ in range(3)]
    net["post"] = [param(H, add=1.0) for _ in range(2)]
    net["scale"] = [param(H, add=0.5) for _ in range(2)]
    net["gate_w"] = param(H, H)
    net["head_w"], net["head_b"] = param(C, H), param(C)
    net["dtype"] = dtype
    net["off"] = torch.tensor([0, 70, 70, 210, V], dtype=torch.int32, device=dev())
    net["x"] = torch.randn(V, F, device=dev())
    t = torch.randint(0, C, (V,))
    t[::11] = -1
    net["t"] = t.to(dev())
    return net, A


def parameters(net):
    own = list(net["conv"].parameters()) + [p for m in net["typed"] for p in m.parameters()]
    return own + net["norm"] + net["post"] + net["scale"] + [net["gate_w"], net["head_w"], net["head_b"]]


def forward(net):
    from jittorgeometric_amd.nn import linear_cross_entropy, residual_norm, rms_norm
    s = net["conv"](net["x"], net["csc"], net["csr"]).to(net["dtype"])
    h = rms_norm(s, net["norm"][0])
    for i in range(2):
        y = net["typed"][i](h, net["off"])
        s, h = residual_norm(s, y, net["norm"][i + 1], post_weight=net["post"][i], gate=h @ net["gate_w"],
                             scale=net["scale"][i])
    return linear_cross_entropy(h, net["head_w"], net["t"], bias=net["head_b"])


def reference(net, A):
    P = [p.detach().double().cpu().requires_grad_(True) for p in parameters(net)]
    it = iter(P)
    cw, cb = next(it), next(it)
    typed = [(next(it), next(it)) for _ in range(2)]
    norm, post, scale = [next(it) for _ in range(3)], [next(it) for _ in range(2)], [next(it) for _ in range(2)]
    gw, hw, hb = next(it), next(it), next(it)
    off = net["off"].tolist()

    def rms(v):
        return v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-6)

    s = A @ (net["x"].double().cpu() @ cw) + cb
    h = rms(s) * norm[0]
    for i in range(2):
        w, b = typed[i]
        y = torch.cat([h[off[g]:off[g + 1]] @ w[g] + b[g] for g in range(TYPES)])
        s = s + scale[i] * torch.sigmoid(h @ gw) * (rms(y) * post[i])
        h = rms(s) * norm[i + 1]
    loss = torch.nn.functional.cross_entropy(h @ hw.t() + hb, net["t"].cpu(), ignore_index=-1)
    return loss, torch.autograd.grad(loss, P)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_loss_and_gradients_of_the_network(dtype):
    """Ten operators follow one another, forward and back: the error of a gradient, relative in norm, is at
    most the sum of twenty operators' own, each under (2 n + 200) u with n = 500 classes the longest sum
    (fp32) or 2 x 2^-8 (two roundings to bfloat16, of inputs or results), times 2 for each of the three
    norms it passes (an inverse norm of a vector of comparable entries at most doubles a relative error)."""
    net, A = build(dtype)
    P = parameters(net)
    loss = forward(net)
    grads = torch.autograd.grad(loss, P)
    want, wgrads = reference(net, A)
    each = (2 * C + 200) * U if dtype == torch.float32 else 2 * 2.0 ** -8
    assert abs(float(loss.detach()) - float(want.detach())) <= 10 * each * max(1.0, abs(float(want.detach())))
    for i, (g, r) in enumerate(zip(grads, wgrads)):
        assert g.dtype == P[i].dtype and g.shape == P[i].shape
        off = float((g.double().cpu() - r).norm() / r.norm())
        assert off <= 20 * 8 * each, (i, tuple(g.shape), off)


def test_training_steps_run_and_repeat():
    """Two runs of five optimiser steps from the same start agree: no operator's result depends on the order
    in which its workgroups end (the weight gradient of the graph layer, which goes through the BLAS
    library, is not held to the last bit)."""
    runs = []
    for _ in range(2):
        net, _ = build()
        opt = torch.optim.AdamW(parameters(net), lr=1e-2)
        losses = []
        for _ in range(5):
            opt.zero_grad()
            loss = forward(net)
            loss.backward()
            opt.step()
            losses.append(loss.detach().clone())
        runs.append((torch.stack(losses), [p.detach().clone() for p in parameters(net)]))
    assert torch.isfinite(runs[0][0]).all()
    for a, b in zip(runs[0][1], runs[1][1]):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)


def test_inference_replays_as_a_graph():
    net, _ = build(torch.bfloat16)

    def step():
        with torch.no_grad():
            return forward(net)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for trial in range(3):
        net["x"].copy_(torch.randn_like(net["x"]))
        want = step().clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(static, want), trial


def test_two_calls_at_once_on_two_streams():
    """Each operator on two streams at a time, on inputs of its own, against the same call alone."""
    from jittorgeometric_amd.nn import linear_cross_entropy, residual_norm
    from jittorgeometric_amd.ops import grouped_rows
    g = torch.Generator().manual_seed(1)

    def rand(*shape):
        return torch.randn(*shape, generator=g).to(dev())

    sets = []
    for n in (30000, 20000):
        x = rand(n, 64).requires_grad_(True)
        w = rand(3, 64, 128).requires_grad_(True)
        e = rand(3000, 128).requires_grad_(True)
        sets.append((x, w, e, torch.tensor([0, n // 3, n // 2, n], dtype=torch.int32, device=dev()),
                     torch.randint(0, 3000, (n,), generator=g).to(dev()), rand(n, 128), rand(128)))

    def call(x, w, e, off, t, r, nw):
        y = grouped_rows(x, w, off)
        s, h = residual_norm(r, y, nw)
        loss = linear_cross_entropy(h, e, t)
        return [loss.detach(), *torch.autograd.grad(loss, [x, w, e])]

    alone = [call(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        got = []
        for s, st in zip(sets, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(call(*s))
        for st in streams:
            torch.cuda.current_stream().wait_stream(st)
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            for u, v in zip(a, b):
                assert torch.equal(u, v)
