"""The residual add with dropout on the GPU against the 64-bit formula.

Tolerance: the kernel forms fma(x, alpha scale, residual) in fp32 from an fp32 product
alpha scale (2^-24 relative), rounds the sum once (2^-24) and once more to bf16 (2^-8):
|err| <= u |out| + 2^-23 (|residual| + |alpha scale x|), u = 2^-8 for bf16, 2^-24 for fp32."""
import numpy as np
import pytest
import torch

import attention_reference as ref
from genet5_amd import residual

pytestmark = pytest.mark.gpu


def make(n, d, dtype, seed, dev):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(n, d, generator=g).to(dtype).to(dev) for _ in range(3)]


def expect(x, r, do, p, alpha, seed):
    keep, up = ref.keep_mask(np.arange(x.shape[0]), x.shape[1], seed, p)
    m = torch.from_numpy(keep).double() * (up * alpha)
    x, r, do = (t.double().cpu() for t in (x, r, do))
    return r + m * x, m * do, (m * x).abs() + r.abs(), (m * do).abs()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,d", [(1, 1), (1, 768), (777, 768), (33, 127), (5, 770), (64, 8),
                                 (3, 12), (300, 4)])
@pytest.mark.parametrize("p,alpha", [(0.1, 1.0), (0.5, 0.70710678), (0.0, -2.0), (1.0, 1.0)])
def test_values_and_gradients(cuda_device, dtype, n, d, p, alpha):
    print(f"dropout_add n={n} d={d} p={p} {dtype}", flush=True)
    x, r, do = make(n, d, dtype, n + d, cuda_device)
    seed = (9 << 35) + 17
    a, b = x.clone().requires_grad_(True), r.clone().requires_grad_(True)
    out = residual.dropout_add(a, b, p, alpha=alpha, seed=seed)
    dx, dr = torch.autograd.grad(out, (a, b), do)
    torch.cuda.synchronize()
    want, wdx, size, gsize = expect(x, r, do, p, alpha, seed)
    u = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    for got, w, s in ((out.detach(), want, size), (dx, wdx, gsize)):
        assert got.dtype == dtype and got.shape == (n, d)
        assert ((got.double().cpu() - w).abs() <= u * w.abs() + 2.0 ** -23 * s + 1e-38).all()
    assert torch.equal(dr, do)
    # dropped elements are the residual itself
    keep, _ = ref.keep_mask(np.arange(n), d, seed, p)
    k = torch.from_numpy(keep).to(cuda_device)
    assert torch.equal(out.detach()[~k], r[~k]) and (dx[~k] == 0).all()


def test_dropped_infinities_stay_out(cuda_device):
    x, r, _ = make(16, 768, torch.bfloat16, 3, cuda_device)
    keep = torch.from_numpy(ref.keep_mask(np.arange(16), 768, 5, 0.5)[0]).to(cuda_device)
    y = torch.where(keep, x, torch.full_like(x, float("nan")))
    assert torch.equal(residual.dropout_add(y, r, 0.5, seed=5),
                       residual.dropout_add(x, r, 0.5, seed=5))


def test_views_of_rows(cuda_device):
    """Leading dimensions, transposed and unaligned views give the same bits."""
    x, r, do = make(60, 768, torch.bfloat16, 5, cuda_device)
    want = residual.dropout_add(x, r, 0.3, seed=8)
    assert torch.equal(residual.dropout_add(x.view(3, 20, 768), r.view(3, 20, 768), 0.3,
                                            seed=8).view(60, 768), want)
    xt = x.t().contiguous().t()
    assert torch.equal(residual.dropout_add(xt, r, 0.3, seed=8), want)
    flat = torch.empty(60 * 768 + 1, dtype=torch.bfloat16, device=cuda_device)
    odd = flat[1:].view(60, 768)
    odd.copy_(x)
    assert torch.equal(residual.dropout_add(odd, r, 0.3, seed=8), want)


def test_seeds_training_flag_and_refusals(cuda_device):
    x, r, _ = make(40, 768, torch.bfloat16, 7, cuda_device)
    torch.manual_seed(3)
    a, b = residual.dropout_add(x, r, 0.2), residual.dropout_add(x, r, 0.2)
    torch.manual_seed(3)
    assert torch.equal(residual.dropout_add(x, r, 0.2), a) and not torch.equal(a, b)
    assert torch.equal(residual.dropout_add(x, r, 0.2, training=False),
                       (x.float() + r.float()).to(torch.bfloat16))
    e = residual.dropout_add(x[:0], r[:0], 0.2)
    assert e.shape == (0, 768)
    for args, error, match in (((x, r[:3], 0.1), ValueError, "shape"),
                               ((x, r.float(), 0.1), TypeError, "dtype"),
                               ((x, r, 1.5), ValueError, "probability"),
                               ((x, r.cpu(), 0.1), ValueError, "cpu"),
                               ((x.half(), r.half(), 0.1), TypeError, "bfloat16")):
        with pytest.raises(error, match=match):
            residual.dropout_add(*args)
    with pytest.raises(ValueError, match="seed"):
        residual.dropout_add(x, r, 0.1, seed=-1)


def test_compiled_equals_eager(cuda_device):
    x, r, do = make(50, 768, torch.bfloat16, 9, cuda_device)
    f = torch.compile(lambda a, b: residual.dropout_add(a, b, 0.25, alpha=0.5, seed=6),
                      fullgraph=True, backend="aot_eager")
    res = []
    for fn in (f, lambda a, b: residual.dropout_add(a, b, 0.25, alpha=0.5, seed=6)):
        a, b = x.clone().requires_grad_(True), r.clone().requires_grad_(True)
        out = fn(a, b)
        res.append((out.detach(), *torch.autograd.grad(out, (a, b), do)))
    for a, b in zip(*res):
        assert torch.equal(a, b)


def test_graph_replays(cuda_device):
    sets = [make(200, 768, torch.bfloat16, 11 + i, cuda_device) for i in range(3)]
    static = [t.clone() for t in sets[0]]

    def step(x, r, do):
        a, b = x.detach().requires_grad_(True), r.detach().requires_grad_(True)
        out = residual.dropout_add(a, b, 0.1, seed=4)
        return (out.detach(),) + torch.autograd.grad(out, (a, b), do)

    want = [[t.clone() for t in step(*s)] for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step(*static)
    for rep in range(6):
        for a, b in zip(static, sets[rep % 3]):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for g, w in zip(res, want[rep % 3]):
            assert torch.equal(g, w)
        step(*sets[(rep + 1) % 3])


def test_second_derivatives_are_refused(cuda_device):
    x = torch.randn(5, 64, device=cuda_device, requires_grad=True)
    do = torch.randn(5, 64, device=cuda_device, requires_grad=True)
    out = residual.dropout_add(x, torch.zeros_like(x), 0.5, seed=3)
    dx = torch.autograd.grad(out, x, do, create_graph=True)[0]
    with pytest.raises(RuntimeError):  # (torch names do as unused)
        torch.autograd.grad(dx.sum(), do)
