"""Calls that the documentation of the layer norm, the orthogonalisation and
the momentum step allows beside the ordinary ones."""
import pytest
import torch
from torch import nn
from torch.autograd import forward_ad

from pymolecular_b200 import _native as nat, layer_norm, muon_step, orthogonalize

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("where", ["x", "weight", "bias"])
def test_dual_tensors_are_refused(where, cuda_device):
    """The result is written by pointer: without a refusal it would lack its tangent."""
    x = torch.randn(6, 32, device=cuda_device)
    layer = nn.LayerNorm(32, device=cuda_device).requires_grad_(False)
    with torch.no_grad():
        want = layer_norm(x, layer)
    for grad in (False, True):
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            assert torch.equal(layer_norm(x, layer), want)   # plain tensors beside dual ones
            t = {"x": x, "weight": layer.weight.detach(), "bias": layer.bias.detach()}
            t[where] = forward_ad.make_dual(t[where], torch.ones_like(t[where]))
            dual = nn.LayerNorm(32, device=cuda_device)
            for name in ("weight", "bias"):
                delattr(dual, name)
                setattr(dual, name, t[name])
            with pytest.raises(NotImplementedError, match="jvp"):
                layer_norm(t["x"], dual)
    with torch.no_grad():
        assert torch.equal(layer_norm(x, layer), want)


@pytest.mark.parametrize("shape", [(6, 32), (2, 3, 32)])
def test_traced_call_computes(shape, cuda_device):
    x, other = (torch.randn(*shape, device=cuda_device) for _ in range(2))
    layer = nn.LayerNorm(32, device=cuda_device).requires_grad_(False)
    for grad in (False, True):
        with torch.set_grad_enabled(grad):
            traced = torch.jit.trace(lambda t: 2 * layer_norm(t, layer), (x,))
            assert torch.equal(traced(other), 2 * layer_norm(other, layer))


@pytest.mark.parametrize("shape", [(0, 5), (5, 0), (0, 0), (3, 0, 4), (0, 3, 4), (2, 3, 4, 0), (2, 0, 3, 4)])
def test_matrices_with_an_empty_side(shape, cuda_device):
    """Alone and in batches, as in lists."""
    for dtype in (torch.float32, torch.bfloat16):
        out = orthogonalize(torch.zeros(shape, dtype=dtype, device=cuda_device))
        assert out.shape == shape and out.dtype == dtype and out.device == cuda_device


@pytest.mark.parametrize("shapes", [[(64, 129), (128, 257)], [(200, 333), (256, 513)], [(64, 2000), (40, 50)],
                                    [(256, 513)] * 30])
def test_a_step_whose_waits_run_out_leaves_the_weights(shapes, cuda_device, monkeypatch):
    """EGNN_DEBUG_WAIT_POLLS=0: the readers of either kernel give up at once
    (the products complete and are drained).  There is no update then, and
    none is made of what lies in the workspace."""
    g = torch.Generator(device="cuda").manual_seed(3)
    w0, grads, m0 = ([torch.randn(*s, device=cuda_device, generator=g) for s in shapes] for _ in range(3))
    lib = nat.lib()

    def step():
        w, m = [t.clone() for t in w0], [t.clone() for t in m0]
        muon_step(w, grads, m, lr=0.1, weight_decay=0.1)
        return w, m

    monkeypatch.delenv("EGNN_DEBUG_WAIT_POLLS", raising=False)
    want = step()
    assert lib.egnn_device_status(nat.stream_ptr()) == nat.EGNN_OK, nat.last_error()
    monkeypatch.setenv("EGNN_DEBUG_WAIT_POLLS", "0")
    w, m = step()
    assert lib.egnn_device_status(nat.stream_ptr()) == nat.EGNN_ERR_CUDA and "timed out" in nat.last_error()
    assert all(torch.equal(a, b) for a, b in zip(w, w0))
    assert all(torch.equal(a, b) for a, b in zip(m, want[1]))
    monkeypatch.delenv("EGNN_DEBUG_WAIT_POLLS")
    assert all(torch.equal(a, b) for a, b in zip(sum(step(), []), sum(want, [])))
