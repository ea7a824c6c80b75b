"""EGNN(node_norm=True): the float64 oracle's layers with layer norms between
them, values and gradients.  fp32 mode is held to max(1e-5, 3x the float32
oracle's own error), as the layers are."""
import pytest
import torch

from conftest import check_tensors, tolerances
from oracle import egnn_oracle as O
from pymolecular_b200 import CSR, EGNN, graph_sum_mse
from pymolecular_b200.datasets import molecules
from pymolecular_b200.parallel import build_halo_plan, partitioned_forward

pytestmark = pytest.mark.gpu


def _oracle(model, b, dtype):
    p = {k: v.detach().cpu().to(dtype).requires_grad_() for k, v in model.state_dict().items()}
    h, x = b.h.to(dtype), b.x.to(dtype)
    h = h @ p["embedding_in.weight"].T + p["embedding_in.bias"]
    for i in range(model.n_layers):
        h, x = O.e_gcl(p, "gcl_%d." % i, h, b.row, b.col, x)
        centred = h - h.mean(1, keepdim=True)
        h = centred / (centred.square().mean(1, keepdim=True) + 1e-5).sqrt()
        h = h * p["norm_%d.weight" % i] + p["norm_%d.bias" % i]
    h = h @ p["embedding_out.weight"].T + p["embedding_out.bias"]
    loss = O.graph_sum_mse(h, b.graph_index(), b.target)
    loss.backward()
    return {"h": h.detach(), "x": x.detach(), "loss": loss.detach(),
            **{k: v.grad if v.grad is not None else torch.zeros_like(v) for k, v in p.items()}}


def _model(dev, hidden=64):
    torch.manual_seed(4)
    model = EGNN(5, hidden, 1, n_layers=3, device=dev, node_norm=True)
    with torch.no_grad():
        for i in range(3):
            model._modules["norm_%d" % i].weight.add_(0.3 * torch.randn(hidden, device=dev))
            model._modules["norm_%d" % i].bias.add_(0.3 * torch.randn(hidden, device=dev))
    return model


def test_model_with_norms_against_the_oracle(cuda_device):
    b = molecules(10, seed=1)
    model = _model(cuda_device)
    csr = CSR.from_edges(b.row, b.col, n_nodes=b.n_nodes, device=cuda_device)
    ho, xo = model(b.h.to(cuda_device), b.x.to(cuda_device), csr)
    loss = graph_sum_mse(ho[:, 0], b.graph_ptr.to(cuda_device), b.target.to(cuda_device))
    loss.backward()
    got = {"h": ho, "x": xo, "loss": loss,
           **{k: v.grad if v.grad is not None else torch.zeros_like(v) for k, v in model.named_parameters()}}
    ref = _oracle(model, b, torch.float64)
    check_tensors(got, ref, tolerances(ref, _oracle(model, b, torch.float32), 1e-5, 3.0))


def test_without_norms_nothing_changes(cuda_device):
    torch.manual_seed(4)
    plain = EGNN(5, 64, 1, n_layers=3, device=cuda_device)
    sd = _model(cuda_device).state_dict()
    assert all(torch.equal(v, sd[k]) for k, v in plain.state_dict().items())   # the same seeded weights
    assert not any(k.startswith("norm") for k in plain.state_dict())


def test_partitioned_forward_normalises_too(cuda_device):
    b = molecules(6, seed=2)
    model = _model(cuda_device)
    plan = build_halo_plan(b.row, b.col, b.n_nodes, 0, 1)
    csr = CSR.from_edges(plan.row, plan.col, n_nodes=plan.n_local, device=cuda_device)
    h, x = b.h.to(cuda_device), b.x.to(cuda_device)
    with torch.no_grad():
        want = model(h, x, csr)
        got = partitioned_forward(model, h, x, csr, plan)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
