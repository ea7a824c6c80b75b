"""layer_norm against float64, element by element.

Tolerances (u = 2^-24, one rounding of float32; a sum of a row passes at most
8192 / 256 = 32 additions in a thread and 10 in the tree, so 43 u with the
division, relative to the mean magnitude of its terms):
  the mean is off by at most 43 u max|x|, 1 / sqrt(var + eps) by half of
  43 u + 2 u and two roundings, relatively 25 u, so the normalised value by
    du <= u (43 s max|x| + 27 |unit|);
  y by |w| du + 2 u (|unit w| + |b|), and half a step of its type;
  dx = s (g - mean g - unit mean(g unit)) with D = max|g|, U = max|unit|:
    s D (u (50 + 46 U^2) + 2 U max du) + 30 u |dx|, and half a step;
  dw, db: rows of one thread in sequence (rows / 148 at most, with at least
  one block per SM) and less than 80 partials:
    (rows / 148 + 80) u sum|dy unit| + sum|dy| du, and half a step.
float16 adds half of its smallest step, 2^-25.
"""
import pytest
import torch
from torch import nn

from pymolecular_b200 import layer_norm
from pymolecular_b200.graphs import GraphedStep

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def _layer(cols, g, dtype=torch.float32, affine=True, bias=True, eps=1e-5):
    layer = nn.LayerNorm(cols, eps=eps, elementwise_affine=affine, bias=bias, device="cuda", dtype=dtype)
    with torch.no_grad():
        if layer.weight is not None:
            layer.weight.copy_(1 + 0.3 * torch.randn(cols, device="cuda", generator=g))
        if layer.bias is not None:
            layer.bias.copy_(torch.randn(cols, device="cuda", generator=g))
    return layer


def _oracle(x, layer, dy):
    """Values and error bounds: {name: (float64 value, bound without the final rounding)}."""
    x, dy = x.detach().double(), dy.double()
    rows, cols = x.shape
    w = torch.ones(cols, dtype=torch.float64, device=x.device) if layer.weight is None else layer.weight.detach().double()
    b = torch.zeros_like(w) if layer.bias is None else layer.bias.detach().double()
    mu = x.mean(1, keepdim=True)
    s = ((x - mu).square().mean(1, keepdim=True) + layer.eps).rsqrt()
    unit = (x - mu) * s
    du = U * (43 * s * x.abs().amax(1, keepdim=True) + 27 * unit.abs())
    y = unit * w + b
    g = dy * w
    dx = s * (g - g.mean(1, keepdim=True) - unit * (g * unit).mean(1, keepdim=True))
    D, Um = g.abs().amax(1, keepdim=True), unit.abs().amax(1, keepdim=True)
    n = rows / 148 + 80
    return {"y": (y, w.abs() * du + 2 * U * ((unit * w).abs() + b.abs())),
            "dx": (dx, s * D * (U * (50 + 46 * Um ** 2) + 2 * Um * du.amax(1, keepdim=True)) + 30 * U * dx.abs()),
            "dw": ((dy * unit).sum(0), n * U * (dy * unit).abs().sum(0) + (dy.abs() * du).sum(0)),
            "db": (dy.sum(0), n * U * dy.abs().sum(0))}


def _check(name, got, want):
    value, bound = want
    bound = bound + HALF[got.dtype] * (value.abs() + bound) + TINY[got.dtype]
    over = ((got.double() - value).abs() - bound).max().item()
    assert not over > 0 and torch.isfinite(got).all(), (name, over)


def _run(x, layer, dy):
    leaves = [x] + [p for p in (layer.weight, layer.bias) if p is not None]
    y = layer_norm(x, layer)
    grads = torch.autograd.grad(y, leaves, dy)
    names = ["dx"] + [n for n, p in (("dw", layer.weight), ("db", layer.bias)) if p is not None]
    return {"y": y.detach(), **dict(zip(names, grads))}


def _features(rows, cols, g, dtype=torch.float32, pad=0, offset=0.5):
    x = torch.randn(rows, cols + pad, device="cuda", generator=g)
    x = x * torch.exp(0.5 * torch.randn(rows, 1, device="cuda", generator=g)) + offset
    return x.to(dtype)[:, :cols].detach().requires_grad_()


# every sharing of a row: 8, 16, 32 lanes, several vectors, blocks; both
# sides of each border, scalar and 16-byte accesses
COLS = [1, 2, 7, 8, 31, 32, 33, 64, 100, 128, 129, 256, 257, 320, 512, 516, 1000, 1024, 1032, 2048, 2052, 2055, 4096,
        8191, 8192]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cols", COLS)
def test_against_float64(cols, dtype, cuda_device):
    g = torch.Generator(device="cuda").manual_seed(cols)
    rows = 37 if cols > 600 else 301
    x, layer = _features(rows, cols, g, dtype), _layer(cols, g)
    dy = torch.randn(rows, cols, device="cuda", generator=g).to(dtype)
    got, want = _run(x, layer, dy), _oracle(x, layer, dy)
    for k in got:
        assert got[k].dtype == (dtype if k in ("y", "dx") else torch.float32) and got[k].is_contiguous()
        _check(k, got[k], want[k])
    with torch.no_grad():   # the inference call keeps no statistics
        assert torch.equal(layer_norm(x, layer), got["y"])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cols", [321, 383, 385, 511])
def test_widths_of_scalar_rows(cols, dtype, cuda_device):
    """12 and 16 scalars to a lane."""
    g = torch.Generator(device="cuda").manual_seed(cols)
    x, layer = _features(777, cols, g, dtype, pad=3), _layer(cols, g)
    dy = torch.randn(777, cols, device="cuda", generator=g).to(dtype)
    got, want = _run(x, layer, dy), _oracle(x, layer, dy)
    for k in got:
        _check(k, got[k], want[k])


@pytest.mark.parametrize("rows,cols", [(1, 64), (2, 128), (1850, 64), (9939, 128), (4001, 256), (70000, 40)])
def test_row_counts(rows, cols, cuda_device):
    g = torch.Generator(device="cuda").manual_seed(rows)
    x, layer = _features(rows, cols, g), _layer(cols, g)
    dy = torch.randn(rows, cols, device="cuda", generator=g)
    got, want = _run(x, layer, dy), _oracle(x, layer, dy)
    for k in got:
        _check(k, got[k], want[k])
    again = _run(x, layer, dy)
    assert all(torch.equal(got[k], again[k]) for k in got)   # fixed order


@pytest.mark.parametrize("dtype,pad", [(torch.float32, 1), (torch.float32, 4), (torch.bfloat16, 8), (torch.float16, 3)])
def test_slices_of_wider_rows(dtype, pad, cuda_device):
    g = torch.Generator(device="cuda").manual_seed(pad)
    rows, cols = 211, 128
    x, layer = _features(rows, cols, g, dtype, pad), _layer(cols, g)
    wide = torch.randn(rows, 3 * cols + 5, device="cuda", generator=g).to(dtype)
    for dy in (wide[:, 5:5 + cols], wide[:, :cols], wide[:1, :cols].expand(rows, cols), wide[:, ::3][:, :cols]):
        got, want = _run(x, layer, dy), _oracle(x, layer, dy)
        for k in got:
            _check(k, got[k], want[k])
    # rows that start off a 16-byte boundary
    x = wide[:, 1:1 + cols].detach().requires_grad_()
    got, want = _run(x, layer, wide[:, :cols]), _oracle(x, layer, wide[:, :cols])
    for k in got:
        _check(k, got[k], want[k])


@pytest.mark.parametrize("affine,bias,pdt", [(False, False, None), (True, False, torch.float32),
                                             (True, True, torch.bfloat16)])
def test_parameters_absent_or_of_the_rows_type(affine, bias, pdt, cuda_device):
    g = torch.Generator(device="cuda").manual_seed(7)
    rows, cols = 333, 96
    dtype = torch.bfloat16
    layer = _layer(cols, g, pdt or torch.float32, affine, bias, eps=1e-3)
    x = _features(rows, cols, g, dtype)
    dy = torch.randn(rows, cols, device="cuda", generator=g).to(dtype)
    got, want = _run(x, layer, dy), _oracle(x, layer, dy)
    assert len(got) == 2 + (layer.weight is not None) + (layer.bias is not None)
    for k in got:
        _check(k, got[k], want[k])


def test_gradients_asked_for_one_at_a_time(cuda_device):
    g = torch.Generator(device="cuda").manual_seed(8)
    x, layer = _features(500, 64, g), _layer(64, g)
    dy = torch.randn(500, 64, device="cuda", generator=g)
    full = _run(x, layer, dy)
    for k, leaf in (("dx", x), ("dw", layer.weight), ("db", layer.bias)):
        for p in (x, layer.weight, layer.bias):
            p.requires_grad_(p is leaf)
        (got,) = torch.autograd.grad(layer_norm(x, layer), [leaf], dy)
        assert torch.equal(got, full[k])


def test_leading_axes_no_rows_and_large_offsets(cuda_device):
    g = torch.Generator(device="cuda").manual_seed(9)
    layer = _layer(48, g)
    x = torch.randn(3, 5, 7, 48, device="cuda", generator=g)
    y = layer_norm(x, layer)
    assert y.shape == x.shape and torch.equal(y.view(-1, 48), layer_norm(x.view(-1, 48), layer))
    assert layer_norm(x[0, 0, 0], layer).shape == (48,)
    t = x.transpose(0, 2)
    assert torch.equal(layer_norm(t, layer), y.transpose(0, 2))
    none = torch.zeros(0, 48, device="cuda", requires_grad=True)
    dx, dw, db = torch.autograd.grad(layer_norm(none, layer), [none, layer.weight, layer.bias], torch.zeros_like(none))
    assert dx.shape == (0, 48) and not dw.any() and not db.any()
    x = _features(100, 48, g, offset=1000.0)
    dy = torch.randn(100, 48, device="cuda", generator=g)
    got, want = _run(x, layer, dy), _oracle(x, layer, dy)
    for k in got:
        _check(k, got[k], want[k])


def test_constant_rows_and_nan_rows(cuda_device):
    """A constant row gives the bias and finite gradients; a row with a NaN or
    an infinity spoils itself alone (and the weight's gradient, a sum over
    all rows)."""
    g = torch.Generator(device="cuda").manual_seed(10)
    layer = _layer(128, g)
    x = torch.randn(64, 128, device="cuda", generator=g)
    x[3] = 0.0
    x[4] = 2.5
    clean = layer_norm(x, layer)
    assert torch.equal(clean[3], layer.bias) and torch.allclose(clean[4], layer.bias, rtol=0, atol=1e-4)
    bad = x.clone()
    bad[7, 5], bad[9, 0] = float("nan"), float("inf")
    bad.requires_grad_()
    y = layer_norm(bad, layer)
    (dx,) = torch.autograd.grad(y, [bad], torch.ones_like(y))
    keep = torch.ones(64, dtype=torch.bool, device="cuda")
    keep[[7, 9]] = False
    assert torch.equal(y[keep], clean[keep]) and torch.isfinite(dx[keep]).all()
    assert torch.isnan(y[7]).all() and torch.isnan(dx[7]).all() and torch.isnan(y[9]).any()


def test_against_differences(cuda_device):
    """The gradients against central differences of the kernel's own forward.
    With step h = 2^-4 the difference quotient of a loss of size ~8 (its
    float32 terms off by ~2^-20 in sum) is off by 2^-19 / 2^-4, and by h^2
    times a third derivative of order 1: 2e-2 of the gradient's size holds."""
    g = torch.Generator(device="cuda").manual_seed(11)
    x, layer = _features(4, 24, g), _layer(24, g)
    dy = torch.randn(4, 24, device="cuda", generator=g)
    got = _run(x, layer, dy)
    h = 2.0 ** -4
    for leaf, k in ((x, "dx"), (layer.weight, "dw"), (layer.bias, "db")):
        flat, num = leaf.data.view(-1), torch.zeros(leaf.numel(), dtype=torch.float64)
        for i in range(leaf.numel()):
            keep = flat[i].item()
            side = []
            for d in (h, -h):
                flat[i] = keep + d
                with torch.no_grad():
                    side.append((layer_norm(x, layer).double() * dy.double()).sum().item())
            flat[i] = keep
            num[i] = (side[0] - side[1]) / (2 * h)
        want = num.view(leaf.shape)
        assert (got[k].double().cpu() - want).abs().max() <= 2e-2 * want.abs().max(), k


def test_captured_replayed_and_on_another_stream(cuda_device):
    g = torch.Generator(device="cuda").manual_seed(12)
    x, layer = _features(700, 128, g), _layer(128, g)
    dy = torch.randn(700, 128, device="cuda", generator=g)

    def step():
        y = layer_norm(x, layer)
        return torch.cat([t.reshape(-1) for t in (y.detach(), *torch.autograd.grad(y, [x, layer.weight, layer.bias], dy))])

    graphed = GraphedStep(step, warmup=1)
    with torch.no_grad():
        x.add_(torch.randn(700, 128, device="cuda", generator=g))
    replayed = graphed.replay().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(eager, replayed)
    graphed.release()


def test_second_derivative_is_refused(cuda_device):
    g = torch.Generator(device="cuda").manual_seed(13)
    x, layer = _features(5, 16, g), _layer(16, g)
    (dx,) = torch.autograd.grad(layer_norm(x, layer).square().sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
