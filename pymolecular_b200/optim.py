"""The update of a model's weight matrices: momentum, orthogonalised by
Newton-Schulz products (the Muon optimiser), on the library's kernels.

* ``orthogonalize(g)``: X0 = G / (|G|_F + eps), then ``steps`` times
  X <- a X + (b A + c A A) X with A = X X^T, which moves the singular values
  by s <- a s + b s^3 + c s^5 and keeps the singular vectors.  One matrix, a
  batch, or a list of matrices of any sizes in one call
  (``egnn_orthogonalize``).
* ``muon_step(params, grads, buffers, lr)``: for every matrix
  M <- mu M + (1 - mu) G, U = mu M + (1 - mu) G (Nesterov) or M,
  W <- (1 - lr weight_decay) W - lr sqrt(max(1, rows / cols)) orthogonalize(U)
  (``egnn_muon_step``), in place.
* ``Muon``: the same as a ``torch.optim.Optimizer`` for an ``EGNN``'s weight
  matrices (``Muon.split`` separates them from its vectors).

All matrices of a call share its launches; nothing synchronises with the
host, so a step with them can be captured (``graphs.GraphedStep``).
"""
from __future__ import annotations

import ctypes as C
import functools
import struct
from typing import Iterable, List, Sequence, Tuple, Union

import torch

from . import _native as nat
from .norm import DTYPES

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7
MAX_SIDE, MAX_SMALL_SIDE = 16384, 1024
TOO_LARGE = f"matrices have at most {MAX_SIDE} rows and columns, and the smaller side at most {MAX_SMALL_SIDE}"
NOT_DENSE = "parameters and momenta must have dense rows (they are updated in place)"


@functools.lru_cache(maxsize=64)
def _options(steps, a, b, c, eps):
    return nat.NsOptions(steps, 0, a, b, c, eps)


def _workspace(sizes: Sequence[int], device) -> Tuple[torch.Tensor, int]:
    """sizes: rows, cols of each matrix in turn."""
    nbytes = 0
    if max(sizes) < 1 << 31:
        nbytes = nat.lib().egnn_orthogonalize_workspace_size(len(sizes) // 2, struct.pack("%di" % len(sizes), *sizes))
    if not nbytes:
        raise ValueError(TOO_LARGE)
    return torch.empty(nbytes, dtype=torch.uint8, device=device), nbytes


def _dense_rows(t: torch.Tensor) -> bool:
    rows, cols = t.shape
    return not rows * cols or (t.stride(1) == 1 or cols <= 1) and (t.stride(0) >= cols or rows <= 1)


def _refuse_tracing(t: torch.Tensor) -> None:
    if t.dim() and type(t.shape[0]) is not int:   # torch.jit.trace makes tensors of sizes
        raise RuntimeError("torch.jit.trace does not see what these kernels write: their results are written by pointer")


def orthogonalize(g: Union[torch.Tensor, Sequence[torch.Tensor]], steps: int = STEPS,
                  coefficients: Tuple[float, float, float] = COEFFICIENTS, eps: float = EPS):
    """The matrix, batch of matrices (..., m, n) or list of matrices `g` with
    its singular values driven towards 1 by `steps` Newton-Schulz products.

    float32, bfloat16 or float16 CUDA tensors of one device; the result has
    each one's type and shape (dense; the results of one size and type lie in
    one allocation).  The products' operands have 22 bits, their sums float32's
    24 (``egnn_orthogonalize`` states the error).  Not differentiable: it
    treats `g` as data.
    """
    if isinstance(g, torch.Tensor):
        if g.dim() < 2:
            raise ValueError("orthogonalize takes matrices")
        batch = g.detach()
        mats = batch.flatten(0, -3).unbind(0) if g.dim() > 2 else (batch,)   # reshape(-1, ...) refuses empty sides
        if not mats:
            return torch.empty_like(g, memory_format=torch.contiguous_format)
    else:
        mats = list(g)
        if not mats:
            return []
    device = mats[0].get_device()
    if device < 0:
        raise ValueError("orthogonalize takes CUDA tensors (pymolecular_b200 has no CPU path)")
    _refuse_tracing(mats[0])
    groups, sizes, ptrs, strides, copies = {}, [], [], [], []
    for k, t in enumerate(mats):
        size, code = t.shape, DTYPES.get(t.dtype)
        if len(size) != 2:
            raise ValueError("orthogonalize takes matrices")
        if t.get_device() != device:
            raise ValueError("the matrices of a call must be on one device")
        if code is None:
            raise TypeError(f"matrices must be float32, bfloat16 or float16, got {t.dtype}")
        stride = size[1]
        if not t.is_contiguous():
            if t.stride(1) == 1 and t.stride(0) >= stride:
                stride = t.stride(0)
            else:
                t = t.contiguous()
                copies.append(t)   # lives until the launch
        sizes += size
        ptrs.append(t.data_ptr())
        strides.append(stride)
        key = (size, code)
        if key in groups:
            groups[key].append(k)
        else:
            groups[key] = [k]
    fields, out = [0] * (6 * len(mats)), [None] * len(mats)
    for (size, code), members in groups.items():
        rows, cols = size
        n = len(members)
        made = mats[members[0]].new_empty((n * rows, cols))
        at, step, both = made.data_ptr(), rows * cols * made.element_size(), rows | cols << 32
        # unsafe: `made` itself is not used beside its parts (which then are no views for autograd, and quicker)
        for k, o in zip(members, made.unsafe_split_with_sizes([rows] * n) if n > 1 else (made,)):
            out[k] = o
            fields[6 * k:6 * k + 6] = ptrs[k], at, strides[k], cols, both, code
            at += step
    with nat.device_of(mats[0]):
        ws, nbytes = _workspace(sizes, device)
        items = struct.pack("%dQ" % len(fields), *fields)
        nat.check(nat.lib().egnn_orthogonalize(len(mats), items, C.byref(_options(steps, *coefficients, eps)),
                                               ws.data_ptr(), nbytes, nat.stream_ptr()), "egnn_orthogonalize")
    if not isinstance(g, torch.Tensor):
        return out
    return made.view(g.shape)


def muon_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], buffers: Sequence[torch.Tensor],
              lr: Union[float, torch.Tensor], momentum: float = 0.95, nesterov: bool = True,
              weight_decay: float = 0.0, steps: int = STEPS,
              coefficients: Tuple[float, float, float] = COEFFICIENTS, eps: float = EPS) -> None:
    """One momentum step with orthogonalised updates, in place on `params` and
    their momenta `buffers` (float32 CUDA matrices with dense rows, no two of
    them overlapping each other or a gradient).  `lr` is a number or a one-element float32 CUDA tensor,
    which a captured step reads at each replay."""
    params, grads, buffers = list(params), list(grads), list(buffers)
    if not len(params) == len(grads) == len(buffers):
        raise ValueError("muon_step takes one gradient and one momentum buffer for each parameter")
    if not params:
        return
    if len(set(map(id, params + buffers))) < 2 * len(params):
        raise ValueError("a parameter or momentum buffer is given twice")
    device = params[0].get_device()
    if device < 0:
        raise ValueError("muon_step takes CUDA tensors (pymolecular_b200 has no CPU path)")
    _refuse_tracing(params[0])
    on_device = isinstance(lr, torch.Tensor)
    if on_device and (lr.numel() != 1 or lr.dtype != torch.float32 or lr.get_device() != device):
        raise ValueError("lr must be a number or one float32 on the parameters' device")
    f32 = torch.float32
    sizes, fields, written, read, copies = [], [], [], [], []
    for k, (p, g, m) in enumerate(zip(params, grads, buffers)):
        size = p.shape
        if len(size) != 2 or g.shape != size or m.shape != size:
            raise ValueError(f"parameter {k}: a matrix and its gradient and momentum of the same shape are needed, got "
                             f"{tuple(size)}, {tuple(g.shape)}, {tuple(m.shape)}")
        if p.get_device() != device or g.get_device() != device or m.get_device() != device:
            raise ValueError("the tensors of a step must be on one device")
        if p.dtype is not f32 or g.dtype is not f32 or m.dtype is not f32:
            raise TypeError("muon_step takes float32 parameters, gradients and momenta")
        rows, cols = size
        ldp = ldg = ldm = cols
        if not (p.is_contiguous() and m.is_contiguous()):
            ldp, ldm = p.stride(0), m.stride(0)
            if not (_dense_rows(p) and _dense_rows(m)):
                raise ValueError(NOT_DENSE)
        if not g.is_contiguous():
            if g.stride(1) == 1 and g.stride(0) >= cols:
                ldg = g.stride(0)
            else:
                g = g.contiguous()
                copies.append(g)   # lives until the launch
        sizes += size
        pp, pg, pm = p.data_ptr(), g.data_ptr(), m.data_ptr()
        if rows * cols:
            written += (pp, pm)
            read.append(pg)
        fields += (pp, pg, pm, ldp, ldg, ldm, rows, cols,
                   (rows / cols) ** 0.5 if rows > cols > 0 else 1.0, 0)
    places = set(written)
    if len(places) < len(written):   # other tensors on the same memory
        raise ValueError("a parameter or momentum buffer is given twice")
    if not places.isdisjoint(read):
        raise ValueError("a gradient lies where a parameter or momentum buffer is written")
    options = nat.MuonOptions(_options(steps, *coefficients, eps), momentum, weight_decay,
                              0.0 if on_device else lr, nat.ptr(lr) if on_device else None, int(nesterov), 0)
    with nat.device_of(params[0]):
        ws, nbytes = _workspace(sizes, device)
        items = struct.pack("QQQqqqiifi" * len(params), *fields)
        nat.check(nat.lib().egnn_muon_step(len(params), items, C.byref(options), ws.data_ptr(), nbytes,
                                           nat.stream_ptr()), "egnn_muon_step")
    torch.autograd.graph.increment_version((*params, *buffers))


class Muon(torch.optim.Optimizer):
    """Momentum with orthogonalised updates for weight matrices.

    Takes float32 matrices with dense rows and of the sizes that
    ``muon_step`` takes: an ``EGNN``'s weights go here, its biases and
    normalisation vectors to another optimiser (``Muon.split``).  `lr` may be
    a one-element CUDA tensor (captured steps).  State: ``momentum_buffer``.
    """

    def __init__(self, params, lr: Union[float, torch.Tensor] = 0.02, momentum: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.0, steps: int = STEPS,
                 coefficients: Tuple[float, float, float] = COEFFICIENTS, eps: float = EPS):
        if not isinstance(lr, torch.Tensor) and not lr >= 0.0:
            raise ValueError(f"lr must not be negative, got {lr}")
        if not 0.0 <= momentum < 1.0:
            raise ValueError(f"momentum must be in [0, 1), got {momentum}")
        if not weight_decay >= 0.0:
            raise ValueError(f"weight_decay must not be negative, got {weight_decay}")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay,
                                      steps=steps, coefficients=tuple(coefficients), eps=eps))

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            wrong = None   # with what a step would refuse, before a backward has been paid for
            if p.dim() != 2 or p.dtype != torch.float32:
                wrong = (f"Muon takes float32 matrices, got {tuple(p.shape)} {p.dtype} (Muon.split gives them and "
                         "the rest apart)")
            elif max(p.shape) > MAX_SIDE or min(p.shape) > MAX_SMALL_SIDE:
                wrong = f"{TOO_LARGE}, got {tuple(p.shape)}"
            elif not _dense_rows(p):
                wrong = f"{NOT_DENSE}, got {tuple(p.shape)} with strides {p.stride()}"
            if wrong:
                del self.param_groups[-1]
                raise ValueError(wrong)

    @staticmethod
    def split(params: Iterable[torch.Tensor]) -> Tuple[List[torch.Tensor], List[torch.Tensor]]:
        """(matrices with more than one row and column, the rest)."""
        params = list(params)
        mats = [p for p in params if p.dim() == 2 and min(p.shape) > 1]
        chosen = {id(p) for p in mats}
        return mats, [p for p in params if id(p) not in chosen]

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            buffers = []
            for p in params:
                state = self.state[p]
                if "momentum_buffer" not in state:
                    state["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                buffers.append(state["momentum_buffer"])
            muon_step(params, [p.grad for p in params], buffers, group["lr"], group["momentum"], group["nesterov"],
                      group["weight_decay"], group["steps"], group["coefficients"], group["eps"])
        return loss


__all__ = ["COEFFICIENTS", "Muon", "muon_step", "orthogonalize"]
