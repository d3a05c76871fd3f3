"""The typed graph layer of examples/typed_graph_training.py: its first output
and gradients against a dense 64-bit computation, and its loss falls."""

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example(spmm_npu):
    path = os.path.join(REPO, "examples", "typed_graph_training.py")
    spec = importlib.util.spec_from_file_location("typed_graph_training", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


# The sparse operators' own tolerances (2e-2 for fp16, 1e-4 for fp32), against
# the largest value; gradients pass through four fp16 roundings of that size.
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.float16, 2e-2)])
def test_layer_against_dense(example, dtype, tol):
    nodes, types, width = 500, 4, 64
    layer = example.TypedLayer(nodes, types, width, dtype=dtype, seed=3)
    x = torch.randn(nodes, width).to(dtype).cuda()
    grad = torch.randn(nodes, width).to(dtype).cuda()
    y = layer(x)
    grads = torch.autograd.grad(y, layer.parameters(), grad)

    rowptr, col, value = layer.csr
    a = torch.zeros(nodes, nodes, dtype=torch.float64)
    a[torch.repeat_interleave(torch.arange(nodes), rowptr.diff()), col] = value.double()
    w, scale, shift = (p.detach().double().cpu().requires_grad_(True) for p in layer.parameters())
    xd = x.double().cpu()
    h = (xd - xd.mean(1, keepdim=True)) / (xd.var(1, unbiased=False, keepdim=True) + 1e-5).sqrt() * scale + shift
    want = a @ torch.stack([h[i] @ w[t] for i, t in enumerate(layer.node_type.tolist())])
    dense = torch.autograd.grad(want, (w, scale, shift), grad.double().cpu())
    for got, ref in zip((y, *grads), (want, *dense)):
        off = (got.detach().double().cpu() - ref.detach()).abs().max() / ref.detach().abs().max()
        assert off <= tol


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_loss_falls(example, dtype):
    losses = example.train(nodes=1500, types=5, width=64, steps=25, dtype=dtype, report=None)
    assert losses[-1] < 0.5 * losses[0] and all(l == l for l in losses)
