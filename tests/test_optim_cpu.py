"""Refusals of the layer-norm, orthogonalisation and momentum-step entry
points, which need no GPU: nothing is launched.  Pointers here are never
read."""
import ctypes as C

import pytest
import torch
from torch import nn

from conftest import ROOT
from pymolecular_b200 import EGNN, Muon, layer_norm, muon_step, orthogonalize
from pymolecular_b200 import _native as nat, optim
from pymolecular_b200.optim import COEFFICIENTS

BAD, UNSUPPORTED, WORKSPACE = nat.EGNN_ERR_INVALID_ARG, nat.EGNN_ERR_UNSUPPORTED, nat.EGNN_ERR_WORKSPACE
F32, BF16, F16 = nat.DTYPE_F32, nat.DTYPE_BF16, nat.DTYPE_F16


def test_structures_match_the_header():
    text = (ROOT / "include" / "egnn_b200.h").read_text()
    assert "EGNN_DTYPE_F32 = 0, EGNN_DTYPE_BF16 = 1, EGNN_DTYPE_F16 = 2" in text and (F32, BF16, F16) == (0, 1, 2)
    assert C.sizeof(nat.NsOptions) == 40 and C.sizeof(nat.Matrix) == 48
    assert C.sizeof(nat.MuonMatrix) == 64 and C.sizeof(nat.MuonOptions) == 80


def test_layer_norm_entry_points_refuse_before_any_launch():
    lib = nat.lib()

    def fwd(rows=4, cols=8, x=16, ldx=8, dtype=F32, w=16, b=16, pdt=F32, eps=1e-5, y=16):
        return lib.egnn_layer_norm_fwd(rows, cols, x, ldx, dtype, w, b, pdt, eps, y, None, None)

    def bwd(rows=4, cols=8, x=16, ldx=8, dy=16, lddy=8, dtype=F32, pdt=F32, stats=16, dx=16, dw=16, db=16, ws=16, nws=1 << 20):
        return lib.egnn_layer_norm_bwd(rows, cols, x, ldx, dy, lddy, dtype, 16, pdt, stats, dx, dw, db, ws, nws, None)

    for call in (fwd, bwd):
        for kw in (dict(rows=-1), dict(cols=0), dict(cols=-3), dict(ldx=7), dict(dtype=3), dict(dtype=-1), dict(pdt=BF16),
                   dict(dtype=BF16, pdt=F16), dict(x=None)):
            assert call(**kw) == BAD, kw
        assert call(cols=8193, ldx=9000) == UNSUPPORTED
    assert fwd(eps=-1.0) == BAD and fwd(eps=float("nan")) == BAD and fwd(y=None) == BAD
    assert fwd(rows=0, x=None, y=None) == nat.EGNN_OK
    assert bwd(lddy=7) == BAD and bwd(dy=None) == BAD and bwd(stats=None) == BAD
    assert bwd(dx=None, dw=None, db=None) == nat.EGNN_OK
    assert bwd(ws=None) == WORKSPACE and bwd(nws=16) == WORKSPACE and bwd(dw=None, nws=0) == WORKSPACE
    assert lib.egnn_layer_norm_workspace_size(4, 0) == lib.egnn_layer_norm_workspace_size(4, 8193) == 0
    assert lib.egnn_layer_norm_workspace_size(1 << 40, 8) <= 148 * 64 * 8 * 4   # a partial per block, not per row


def _ns(steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    return nat.NsOptions(steps, 0, *coefficients, eps)


def test_orthogonalize_entry_point_refuses_before_any_launch():
    lib = nat.lib()

    def call(o=None, count=1, ws=256, nws=1 << 24, **kw):
        f = dict(in_=16, out=16, ld_in=8, ld_out=8, rows=4, cols=8, dtype=F32, reserved=0)
        m = (nat.Matrix * 1)(nat.Matrix(**{**f, **kw}))
        return lib.egnn_orthogonalize(count, m, C.byref(o or _ns()), ws, nws, None)

    for kw in (dict(rows=-1), dict(cols=-1), dict(dtype=3), dict(in_=None), dict(out=None), dict(ld_in=7), dict(ld_out=7),
               dict(count=-1)):
        assert call(**kw) == BAD, kw
    assert call(rows=1025, cols=1025, ld_in=2000, ld_out=2000) == UNSUPPORTED
    assert call(cols=16385, ld_in=20000, ld_out=20000) == UNSUPPORTED
    assert call(nws=0) == WORKSPACE and call(ws=None) == WORKSPACE
    assert call(rows=0, in_=None, out=None) == nat.EGNN_OK
    assert lib.egnn_orthogonalize(1, None, C.byref(_ns()), 256, 1 << 20, None) == BAD
    assert lib.egnn_orthogonalize(0, None, None, 256, 1 << 20, None) == BAD
    assert lib.egnn_orthogonalize(0, None, C.byref(_ns()), None, 0, None) == nat.EGNN_OK
    nan, inf = float("nan"), float("inf")
    for o in (_ns(-1), _ns(65), _ns(eps=-1.0), _ns(eps=nan), _ns(eps=inf), _ns(coefficients=(nan, 0, 0)),
              _ns(coefficients=(1, inf, 0)),
              _ns(coefficients=(5.0, 0.0, 0.0)),        # 5^5 > 1024
              _ns(coefficients=(4.0, -3.0, 1.0)),       # 2, 16, then past every bound
              _ns(coefficients=(-3.0, -3.0, 0.0))):
        assert call(o=o) == BAD, (o.steps, o.a, o.b, o.c, o.eps)
    # within bounds: only the workspace is refused
    for o in (_ns(0), _ns(64, (1.5, -0.5, 0.0)), _ns(4, (5.0, 0.0, 0.0)), _ns(64, (1.875, -1.25, 0.375))):
        assert call(o=o, nws=0) == WORKSPACE


def test_orthogonalize_workspace_size():
    lib = nat.lib()

    def size(*sizes):
        flat = [v for s in sizes for v in s]
        return lib.egnn_orthogonalize_workspace_size(len(sizes), (C.c_int32 * len(flat))(*flat))

    assert 0 < size() <= size((64, 64)) <= size((64, 64), (200, 333)) < size((64, 64), (400, 1333))
    assert size((1025, 1025)) == size((-1, 4)) == size((4, 16385)) == 0
    assert size((0, 5), (16384, 1024)) > 0
    assert lib.egnn_orthogonalize_workspace_size(-1, None) == lib.egnn_orthogonalize_workspace_size(2, None) == 0


def test_muon_entry_point_refuses_before_any_launch():
    lib = nat.lib()

    def call(o=None, count=1, ws=256, nws=1 << 24, **kw):
        f = dict(weight=16, grad=16, momentum=16, ld_weight=8, ld_grad=8, ld_momentum=8, rows=4, cols=8, gain=1.0, reserved=0)
        m = (nat.MuonMatrix * 1)(nat.MuonMatrix(**{**f, **kw}))
        return lib.egnn_muon_step(count, m, C.byref(o or nat.MuonOptions(_ns(), 0.95, 0.0, 0.1, None, 1, 0)), ws, nws, None)

    for kw in (dict(rows=-1), dict(weight=None), dict(grad=None), dict(momentum=None), dict(ld_weight=7), dict(ld_grad=7),
               dict(ld_momentum=7), dict(count=-1)):
        assert call(**kw) == BAD, kw
    for mu in (-0.1, 1.0, float("nan")):
        assert call(o=nat.MuonOptions(_ns(), mu, 0.0, 0.1, None, 1, 0)) == BAD
    assert call(o=nat.MuonOptions(_ns(65), 0.9, 0.0, 0.1, None, 1, 0)) == BAD
    assert call(nws=0) == WORKSPACE
    assert call(rows=1030, cols=1030, ld_weight=2000, ld_grad=2000, ld_momentum=2000) == UNSUPPORTED


def test_python_refusals():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        layer_norm(x, nn.LayerNorm(8))
    with pytest.raises(ValueError, match="CUDA"):
        orthogonalize(x)
    with pytest.raises(ValueError, match="CUDA"):
        muon_step([x], [x], [x.clone()], lr=0.1)
    with pytest.raises(ValueError, match="matrices"):
        orthogonalize(torch.zeros(4))
    with pytest.raises(ValueError, match="one gradient"):
        muon_step([x], [], [x], lr=0.1)
    with pytest.raises(ValueError, match="twice"):
        muon_step([x, x], [x, x], [x.clone(), x.clone()], lr=0.1)
    with pytest.raises(ValueError, match="twice"):
        muon_step([x], [x], [x], lr=0.1)


def test_muon_arguments_and_split():
    model = EGNN(5, 32, 1, n_layers=2, node_norm=True)
    mats, rest = Muon.split(model.parameters())
    assert len(mats) == 2 * 5 + 1 and len(mats) + len(rest) == len(list(model.parameters()))
    assert all(p.dim() == 2 and min(p.shape) > 1 for p in mats)
    Muon(mats)
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(momentum=-0.1), dict(weight_decay=-1.0)):
        with pytest.raises(ValueError):
            Muon(mats, **kw)
    with pytest.raises(ValueError, match="matrices"):
        Muon(rest)
    with pytest.raises(ValueError, match="matrices"):
        Muon([nn.Parameter(torch.zeros(4, 4, dtype=torch.float64))])
    opt = Muon(mats[:2])
    with pytest.raises(ValueError, match="matrices"):
        opt.add_param_group({"params": rest[:1]})
    assert len(opt.param_groups) == 1
    opt.add_param_group({"params": mats[2:], "lr": 0.1})
    assert len(opt.param_groups) == 2


def test_node_norm_keeps_the_other_parameters():
    torch.manual_seed(1)
    plain = EGNN(5, 32, 1, n_layers=2).state_dict()
    torch.manual_seed(1)
    normed = EGNN(5, 32, 1, n_layers=2, node_norm=True).state_dict()
    assert set(normed) - set(plain) == {f"norm_{i}.{n}" for i in range(2) for n in ("weight", "bias")}
    assert all(torch.equal(v, normed[k]) for k, v in plain.items())


def test_models_from_before_there_were_norms():
    model = EGNN(2, 32, 1, n_layers=1)
    del model.__dict__["node_norm"]   # as unpickled
    h = torch.zeros(3, 32)
    assert model.normalized(0, h) is h


def test_sides_past_32_bits_are_refused():
    with pytest.raises(ValueError, match="16384"):
        optim._workspace([1 << 31, 1], "cpu")


def test_workspace_is_that_of_the_largest_batch():
    def size(*sizes):
        flat = [v for s in sizes for v in s]
        return nat.lib().egnn_orthogonalize_workspace_size(len(sizes), (C.c_int32 * len(flat))(*flat))

    full = size(*[(200, 333)] * 64)
    assert size(*[(200, 333)] * 63) < full == size(*[(200, 333)] * 65) == size(*[(200, 333)] * 1000)
    assert size(*[(200, 333)] * 64, *[(64, 64)] * 99, *[(400, 1333)] * 64, (1, 1)) == size(*[(400, 1333)] * 64)
