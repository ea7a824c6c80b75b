"""Calls of the layer norm, the orthogonalisation and the momentum step that
have to be refused, or answered without a launch, shown without a GPU."""
import ctypes as C

import pytest
import torch
from torch import nn

from pymolecular_b200 import Muon, _native as nat, layer_norm, muon_step, orthogonalize


class OnDevice(torch.Tensor):
    """A CPU tensor that says it is on device 0."""

    def get_device(self):
        return 0


@pytest.mark.parametrize("name", ["weight", "bias"])
@pytest.mark.parametrize("shape", [(7,), (9,), (1,), (0,), (8, 1), (1, 8), ()])
def test_parameters_of_another_shape_are_refused(name, shape):
    """A kernel reads C elements of the weight and bias and writes C of their
    gradients, however many there are."""
    layer = nn.LayerNorm(8)
    for n in ("weight", "bias"):
        setattr(layer, n, nn.Parameter(torch.ones(shape if n == name else 8).as_subclass(OnDevice)))
    with pytest.raises(ValueError, match="normalized_shape"):
        layer_norm(torch.zeros(4, 8).as_subclass(OnDevice), layer)
    with pytest.raises(RuntimeError):   # as nn.LayerNorm does
        layer(torch.zeros(4, 8))


@pytest.mark.parametrize("shape", [(0, 5), (5, 0), (0, 0), (3, 0, 4), (2, 3, 4, 0)])
def test_matrices_with_an_empty_side_come_as_far_as_others(shape):
    with pytest.raises(ValueError, match="CUDA"):
        orthogonalize(torch.zeros(shape))


def test_tracing_of_results_written_by_pointer_is_refused():
    def step(w):
        muon_step([w], [w.clone().as_subclass(OnDevice)], [w.clone().as_subclass(OnDevice)], lr=0.1)
        return w

    for call in (orthogonalize, lambda w: orthogonalize([w, w])[0], step):
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(lambda t: call(t.as_subclass(OnDevice)), (torch.ones(4, 4),))


@pytest.mark.parametrize("steps,coefficients,taken", [
    (2, (0.0, 3.0, -1.0), False),     # s^3: 2 for s = 1, 6e-4 for s = 0.06
    (1, (0.0, 3.0, -1.0), True),      # nothing is held between steps
    (2, (0.125, 1.0, 1.0), False),    # 2.125 against 1/8 s: 17 times
    (2, (0.125, 1.0, 0.5), True),     # 13 times
    (6, (0.5, 0.5, 0.0), False),      # 1 against 2^-5 before the last step
    (5, (0.5, 0.5, 0.0), True),       # 16 times
    (64, (1.875, -1.25, 0.375), True)])
def test_coefficients_that_leave_small_singular_values_behind(steps, coefficients, taken):
    """The operands' scales follow the largest singular value that the
    coefficients allow; beside it small ones have to keep their bits."""
    o = nat.NsOptions(steps, 0, *coefficients, 1e-7)
    m = nat.Matrix(16, 16, 8, 8, 4, 8, nat.DTYPE_F32, 0)
    status = nat.lib().egnn_orthogonalize(1, (nat.Matrix * 1)(m), C.byref(o), None, 0, None)   # no workspace: no launch
    assert status == (nat.EGNN_ERR_WORKSPACE if taken else nat.EGNN_ERR_INVALID_ARG)
    assert taken or "fall too far behind" in nat.last_error()


@pytest.mark.parametrize("make,match", [
    (lambda: torch.zeros(1025, 1025), "at most"), (lambda: torch.zeros(2, 16385), "at most"),
    (lambda: torch.zeros(16385, 1), "at most"), (lambda: torch.zeros(6, 4).t(), "dense rows"),
    (lambda: torch.zeros(6, 8)[:, ::2], "dense rows"), (lambda: torch.zeros(1, 4).expand(6, 4), "dense rows")])
def test_muon_refuses_matrices_that_no_step_can_take(make, match):
    """When it is made, and not at the first step."""
    good = nn.Parameter(torch.zeros(4, 6))
    with pytest.raises(ValueError, match=match):
        Muon([good, nn.Parameter(make())])
    opt = Muon([good])
    with pytest.raises(ValueError, match=match):
        opt.add_param_group({"params": [nn.Parameter(make())]})
    assert len(opt.param_groups) == 1


def test_muon_takes_what_a_step_takes():
    Muon([nn.Parameter(t) for t in (torch.zeros(1024, 2000), torch.zeros(16384, 1024), torch.zeros(3, 20)[:, 2:9],
                                    torch.zeros(0, 5), torch.zeros(1, 5).t(), torch.zeros(6, 5)[:, :1])])
