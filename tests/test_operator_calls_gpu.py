"""Calls that the documentation of the layer norm, the orthogonalisation and
the momentum step allows beside the ordinary ones."""
import pytest
import torch
from torch import nn
from torch.autograd import forward_ad

from pymolecular_b200 import layer_norm, orthogonalize

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
