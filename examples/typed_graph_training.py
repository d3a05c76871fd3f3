#!/usr/bin/env python3
"""Trains one layer of a graph whose nodes have types, on the GPU.

    python examples/typed_graph_training.py [--nodes 4000] [--types 5] [--width 128] [--steps 30] [--dtype fp32]

A layer norm of the node features, a matrix of its own for each node type, and
the product with the graph's adjacency matrix:

    y = A * typed(norm(x)),   typed(h)[i] = h[i] W[type of i]

with ``spmm_npu``'s operators throughout: ``layer_norm``; ``pack_node_tensor``
into the order of types, ``grouped_matmul`` over the types' row ranges and
``restore_node_tensor``; ``PackedGraph`` for A and, in the backward pass, its
transpose.  The weights of all types are updated together by ``orthogonalize``
of their momentum, the norm's parameters by plain gradient steps.  The layer
learns the outputs of another one with random weights, on a random graph.
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ascend-spmm_amd"))

import spmm_npu  # noqa: E402

DTYPES = {"fp16": torch.float16, "fp32": torch.float32}


def random_graph(nodes, degree, dtype, generator):
    """CSR of a random graph with about ``degree`` in-neighbours a node, each
    row's values summing to one."""
    edges = torch.randint(0, nodes * nodes, (nodes * degree,), generator=generator).unique()
    row, col = edges // nodes, edges % nodes
    counts = torch.bincount(row, minlength=nodes)
    rowptr = torch.zeros(nodes + 1, dtype=torch.int64)
    rowptr[1:] = counts.cumsum(0)
    return rowptr, col, (1.0 / counts.clamp_min(1).double())[row].to(dtype)


class TypedLayer:
    """The layer's graph, the order of its nodes by type, and its parameters."""

    def __init__(self, nodes, types, width, degree=8, dtype=torch.float32, seed=0):
        g = torch.Generator().manual_seed(seed)
        rowptr, col, value = random_graph(nodes, degree, dtype, g)
        self.csr = (rowptr, col, value)
        self.graph = spmm_npu.PackedGraph(
            spmm_npu.preprocess(rowptr.cuda(), col.cuda(), value.cuda(), nodes, nodes, graph_layout=True))
        self.node_type = torch.randint(0, types, (nodes,), generator=g)
        by_type = self.node_type.argsort(stable=True)
        place = torch.empty_like(by_type)
        place[by_type] = torch.arange(nodes)
        self.place = place.cuda()  # of each node in the order of types
        edges = torch.bincount(self.node_type, minlength=types).cumsum(0)
        self.offsets = torch.cat([edges.new_zeros(1), edges]).to(torch.int32).cuda()
        normal = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.weight = (normal(types, width, width) / width ** 0.5).to(dtype).cuda().requires_grad_(True)
        self.scale = torch.ones(width, device="cuda", dtype=dtype, requires_grad=True)
        self.shift = torch.zeros(width, device="cuda", dtype=dtype, requires_grad=True)
        self.momentum = torch.zeros_like(self.weight, requires_grad=False)

    def parameters(self):
        return self.weight, self.scale, self.shift

    def __call__(self, x):
        h = spmm_npu.layer_norm(x, self.scale, self.shift)
        h = spmm_npu.pack_node_tensor(h, self.place)
        h = spmm_npu.grouped_matmul(h, self.weight, self.offsets)
        h = spmm_npu.restore_node_tensor(h, self.place)
        return self.graph.restore(self.graph(self.graph.pack(h)))

    @torch.no_grad()
    def update(self, grads, rate):
        """One optimiser step: the weights along their orthogonalised momentum,
        with the length of a random matrix's row kept; the rest along its
        gradient."""
        dweight, dscale, dshift = grads
        self.momentum.mul_(0.9).add_(dweight, alpha=0.1)
        self.weight.sub_(spmm_npu.orthogonalize(self.momentum), alpha=rate)
        self.scale.sub_(dscale, alpha=rate)
        self.shift.sub_(dshift, alpha=rate)


def train(nodes=4000, types=5, width=128, steps=30, dtype=torch.float32, rate=0.02, report=print):
    """The losses of ``steps`` steps."""
    layer = TypedLayer(nodes, types, width, dtype=dtype, seed=1)
    g = torch.Generator().manual_seed(2)
    x = torch.randn(nodes, width, generator=g).to(dtype).cuda()
    with torch.no_grad():
        own = layer.weight.clone()
        layer.weight.copy_(torch.randn(own.shape, generator=g).to(dtype) / width ** 0.5)
        target = layer(x).float()
        layer.weight.copy_(own)
    losses = []
    for step in range(steps):
        y = layer(x)
        # mean over elements of 1000 (y - target)^2: small gradients would leave fp16's range
        loss = 1000.0 * (y.float() - target).square().mean()
        layer.update(torch.autograd.grad(loss, layer.parameters()), rate)
        losses.append(loss.detach())
    losses = torch.stack(losses).tolist()
    if report:
        for step, loss in enumerate(losses):
            report(f"step {step:3d}  loss {loss:.4f}")
    return losses


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--nodes", type=int, default=4000)
    p.add_argument("--types", type=int, default=5)
    p.add_argument("--width", type=int, default=128)
    p.add_argument("--steps", type=int, default=30)
    p.add_argument("--dtype", choices=sorted(DTYPES), default="fp32")
    a = p.parse_args(argv)
    train(a.nodes, a.types, a.width, a.steps, DTYPES[a.dtype])


if __name__ == "__main__":
    main()
