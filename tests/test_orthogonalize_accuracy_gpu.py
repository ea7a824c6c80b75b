"""Accuracy of the Newton-Schulz products against float32's own.

Every product takes its operands with 22 bits where float32 has 24, so what
rounding adds to them is at most four times float32's; to first order the
error of the result is linear in it.  What else enters (sums) is at float32's
level.  So the 2-norm of the error may be 4 times that of the same iteration
in float32 in torch, on the same inputs, without a floor.
"""
import pytest
import torch

from pymolecular_b200 import muon_step, orthogonalize
from pymolecular_b200._native import EgnnError
from pymolecular_b200.optim import COEFFICIENTS

pytestmark = pytest.mark.gpu

FACTOR = 4.0


def _iterate(G, dtype, steps, coefficients, eps=1e-7):
    a, b, c = coefficients
    X = G.to(dtype)
    X = X.mT if G.shape[0] > G.shape[1] else X
    X = X / (X.double().norm() + eps).to(dtype)
    for _ in range(steps):
        A = X @ X.mT
        X = a * X + (b * A + c * (A @ A)) @ X
    return X.mT if G.shape[0] > G.shape[1] else X


def _errors(G, **kw):
    """(ours, float32's), of float64's 2-norm."""
    want = _iterate(G.double(), torch.float64, **kw)
    size = want.norm()
    return (((t.double() - want).norm() / size).item() for t in (orthogonalize(G, **kw), _iterate(G, torch.float32, **kw)))


def _gradient(rows, cols, g):
    k = max(1, min(rows, cols) // 2)
    u = torch.randn(rows, k, device="cuda", generator=g)
    v = torch.randn(k, cols, device="cuda", generator=g)
    return (u @ v) / k ** 0.5 + 0.5 * torch.randn(rows, cols, device="cuda", generator=g)


# one block with one and with three accumulators, and the whole device: one
# band, two, eight, a long sum in pieces, tall
SIZES = [(64, 129), (128, 257), (60, 1000), (256, 513), (64, 2000), (513, 97), (1024, 2048)]


@pytest.mark.parametrize("steps,coefficients", [(5, COEFFICIENTS), (2, (6.0, -3.0, 0.3)), (1, (6.0, -3.0, 0.3)),
                                                (2, (30.0, 0.0, 0.0)), (3, (8.0, -4.0, 0.5)), (4, (0.25, 0.1, 0.01)),
                                                (2, (0.0, 3.0, -1.0)), (10, (2.0, -1.2, 0.25)), (1, (1.0, -900.0, 100.0))])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_coefficients(rows, cols, steps, coefficients, cuda_device):
    """Bounds of the singular values up to 900 and shrinking steps: no step's
    operands run out of fp16's range, or the coefficients are refused."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    G = _gradient(rows, cols, g)
    # the bound passes 1024 in the third step; small values shrink to their third power behind it
    refused = {(8.0, -4.0, 0.5): "grow past", (0.0, 3.0, -1.0): "fall too far behind"}.get(coefficients)
    if refused:
        with pytest.raises(EgnnError, match=refused):
            orthogonalize(G, steps=steps, coefficients=coefficients)
        return
    own, plain = _errors(G, steps=steps, coefficients=coefficients)
    assert own <= FACTOR * plain, (own, plain)


@pytest.mark.parametrize("norm", [1e-8, 1e-12, 1e-16, 1e-20, 1e-23, 1e-28, 1e-33])
@pytest.mark.parametrize("rows,cols", [(64, 129), (256, 513)])
def test_gradients_far_below_eps(rows, cols, norm, cuda_device):
    """The result shrinks with the gradient, and keeps its bits: |G| / (|G| + eps) down to 2^-86."""
    g = torch.Generator(device="cuda").manual_seed(1)
    G = _gradient(rows, cols, g)
    G = G * (norm / G.norm())
    own, plain = _errors(G, steps=5, coefficients=COEFFICIENTS)
    assert own <= FACTOR * plain, (own, plain)
    if norm == 1e-20:   # the same numbers in a step: W - O, rounded once more
        w, m = torch.zeros_like(G), torch.zeros_like(G)
        muon_step([w], [G], [m], lr=1.0, momentum=0.0)
        assert ((w + orthogonalize(G) * max(1, rows / cols) ** 0.5).norm() / w.norm()).item() <= 4 * 2.0 ** -24


@pytest.mark.parametrize("rows,cols", [(64, 129), (256, 513)])
def test_a_cubic_step_far_below_eps(rows, cols, cuda_device):
    """Without a linear term nothing else covers what such a gradient's cube comes to."""
    g = torch.Generator(device="cuda").manual_seed(2)
    G = _gradient(rows, cols, g)
    own, plain = _errors(G * (1e-18 / G.norm()), steps=1, coefficients=(0.0, 3.0, -1.0))
    assert own <= FACTOR * plain, (own, plain)


def test_small_singular_values(cuda_device):
    """s0 down to 0.0005 of the norm: a sum of rank-one parts whose values
    follow s <- a s + b s^3 + c s^5.  The values of the result are compared
    with the polynomial's; an error of the parts of size d moves them by d at
    most, and float32's own d is the measure."""
    g = torch.Generator(device="cuda").manual_seed(7)
    q = torch.linalg.qr(torch.randn(128, 128, device="cuda", generator=g, dtype=torch.float64))[0]
    r = torch.linalg.qr(torch.randn(257, 128, device="cuda", generator=g, dtype=torch.float64))[0]
    s = torch.logspace(-3.3, 0, 128, device="cuda", dtype=torch.float64)
    G = ((q * s) @ r.mT).float()
    a, b, c = COEFFICIENTS
    t = torch.linalg.svdvals(G.double())
    t = t / (t.norm() + 1e-7)
    for _ in range(5):
        t = a * t + b * t ** 3 + c * t ** 5
    want = t.sort(descending=True).values
    own, plain = ((torch.linalg.svdvals(x.double()) - want).abs().max().item()
                  for x in (orthogonalize(G), _iterate(G, torch.float32, 5, COEFFICIENTS)))
    total = (_iterate(G, torch.float32, 5, COEFFICIENTS).double() - _iterate(G.double(), torch.float64, 5, COEFFICIENTS)).norm().item()
    assert own <= FACTOR * max(plain, total), (own, plain, total)
    assert want.min() < 0.3   # some stay far from 1
