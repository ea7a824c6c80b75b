"""orthogonalize, muon_step and Muon against float64.

Tolerance of orthogonalize (relative 2-norm of the difference from the
float64 iteration): max(1e-5, 2x the error of the float32 iteration in torch
on the same inputs), as the layers' fp32 mode is held to its algorithm's own
float32 error; a 16-bit result adds half a step of its type (every element is
off by at most that, relatively, so the 2-norm is) and, in float16, 2^-25 per
element for values below its normal range.
muon_step: M and W are sums of two or three products, each off by at most
4 x 2^-24 of its terms' size, and W by lr gain times the error above.
"""
import math

import pytest
import torch

from pymolecular_b200 import CSR, EGNN, Muon, graph_sum_mse, layer_norm, muon_step, orthogonalize
from pymolecular_b200 import _native as nat
from pymolecular_b200.datasets import molecules
from pymolecular_b200.graphs import GraphedStep
from pymolecular_b200.optim import COEFFICIENTS

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def _plain(G, dtype, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    X = G.to(dtype)
    X = X.mT if G.shape[0] > G.shape[1] else X
    X = X / (X.double().norm().to(dtype) + eps)
    for _ in range(steps):
        A = X @ X.mT
        X = a * X + (b * A + c * (A @ A)) @ X
    return X.mT if G.shape[0] > G.shape[1] else X


def _tolerance(G, **kw):
    """(float64 result, absolute bound of the difference's 2-norm)."""
    want = _plain(G.double(), torch.float64, **kw)
    own = (_plain(G.float(), torch.float32, **kw).double() - want).norm().item()
    size = want.norm().item()
    return want, max(1e-5 * size, 2 * own) + HALF[G.dtype] * size + TINY[G.dtype] * math.sqrt(G.numel())


def _check(G, got, **kw):
    want, tol = _tolerance(G, **kw)
    assert got.dtype == G.dtype and got.shape == G.shape and got.is_contiguous()
    off = (got.double() - want).norm().item()
    assert off <= tol, (tuple(G.shape), off, tol)


def _gradient(rows, cols, g, scale=1.0):
    k = max(1, min(rows, cols) // 2)
    u = torch.randn(rows, k, device="cuda", generator=g)
    v = torch.randn(k, cols, device="cuda", generator=g)
    return scale * ((u @ v) / k ** 0.5 + 0.5 * torch.randn(rows, cols, device="cuda", generator=g))


# one row or column, sizes around the multiples of 16, 64 and 128, the
# framework's (H, 2H + 1), (H, H), (H, 2H), both orientations, long sides
SIZES = [(1, 1), (1, 128), (128, 1), (2, 3), (3, 3), (5, 128), (15, 17), (16, 16), (31, 77), (32, 65), (33, 32), (63, 64),
         (64, 64), (64, 129), (65, 64), (64, 128), (127, 126), (128, 128), (128, 257), (257, 128), (128, 256), (128, 320),
         (128, 321), (129, 130), (100, 1025), (1100, 64), (200, 333), (256, 256), (256, 513), (513, 256), (256, 512),
         (300, 301), (512, 700)]


@pytest.mark.parametrize("rows,cols", SIZES)
def test_sizes_against_float64(rows, cols, cuda_device):
    g = torch.Generator(device="cuda").manual_seed(rows * 2000 + cols)
    G = _gradient(rows, cols, g)
    _check(G, orthogonalize(G))


def test_largest_sides(cuda_device):
    g = torch.Generator(device="cuda").manual_seed(1)
    for rows, cols in [(1024, 1024), (16, 16384), (16384, 3)]:
        G = _gradient(rows, cols, g)
        _check(G, orthogonalize(G))


@pytest.mark.parametrize("rows,cols", [(1, 767), (1, 769), (17, 5000), (100, 769), (2000, 65), (130, 770), (1555, 129), (257, 2100), (600, 4000)])
def test_long_sums_in_pieces(rows, cols, cuda_device):
    """Matrices whose A = X X^T is computed in pieces of its long sum, and the
    same result in a list, where other groups of blocks share them out."""
    g = torch.Generator(device="cuda").manual_seed(16)
    G = _gradient(rows, cols, g)
    one = orthogonalize(G)
    _check(G, one)
    others = [_gradient(200, 300, g) for _ in range(40)]
    assert torch.equal(orthogonalize([*others[:7], G])[7], one)
    assert torch.equal(orthogonalize([G, *others])[0], one)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_lists_batches_and_strides(dtype, cuda_device):
    """One call over matrices of many sizes gives each what a call of its own
    gives, bit for bit; slices, transposes and columns apart as well."""
    g = torch.Generator(device="cuda").manual_seed(2)
    mats = [_gradient(r, c, g).to(dtype) for r, c in [(64, 129), (128, 5), (33, 200), (1, 7), (0, 4), (200, 140), (7, 0)]]
    wide = _gradient(70, 300, g).to(dtype)
    mats += [wide[:, 3:130], wide[5:60:2, 7:90], wide.t(), wide[:, ::2]]
    got = orthogonalize(mats)
    assert [t.shape for t in got] == [t.shape for t in mats]
    for t, o in zip(mats, got):
        if t.numel():
            _check(t, o)
            assert torch.equal(o, orthogonalize(t))
    many = [mats[k % 4] for k in range(100)]   # more than one launch holds
    for k, o in enumerate(orthogonalize(many)):
        assert torch.equal(o, got[k % 4])
    batch = torch.stack([_gradient(40, 72, g).to(dtype) for _ in range(6)]).view(2, 3, 40, 72)
    out = orthogonalize(batch)
    assert out.shape == batch.shape
    for i in range(2):
        for j in range(3):
            assert torch.equal(out[i, j], orthogonalize(batch[i, j]))
    assert orthogonalize([]) == []


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e-4, 1e4, 1e25])
def test_scale_of_the_gradient(scale, cuda_device):
    """Squares of the entries overflow or vanish in float32, the norm must
    not.  Below eps the result shrinks with the gradient, as defined."""
    g = torch.Generator(device="cuda").manual_seed(3)
    for rows, cols in [(48, 96), (200, 140)]:
        G = _gradient(rows, cols, g, scale)
        _check(G, orthogonalize(G, eps=0.0 if scale < 1e-20 else 1e-7), eps=0.0 if scale < 1e-20 else 1e-7)


@pytest.mark.parametrize("kw", [dict(steps=0), dict(steps=1), dict(steps=12, coefficients=(1.5, -0.5, 0.0)),
                                dict(steps=8, coefficients=(1.875, -1.25, 0.375)), dict(eps=0.5),
                                dict(steps=3, coefficients=(3.0, -3.2, 1.2))])
def test_options(kw, cuda_device):
    g = torch.Generator(device="cuda").manual_seed(4)
    for rows, cols in [(60, 33), (128, 257), (150, 400)]:
        G = _gradient(rows, cols, g)
        _check(G, orthogonalize(G, **kw), **kw)


def test_zero_rank_one_and_orthogonal_inputs(cuda_device):
    g = torch.Generator(device="cuda").manual_seed(5)
    for rows, cols in [(64, 100), (140, 130)]:
        assert not orthogonalize(torch.zeros(rows, cols, device="cuda")).any()
        one = torch.randn(rows, 1, device="cuda", generator=g) @ torch.randn(1, cols, device="cuda", generator=g)
        _check(one, orthogonalize(one))
        q = torch.linalg.qr(torch.randn(cols, rows, device="cuda", generator=g).double())[0].float()
        _check(q, orthogonalize(q))


def test_a_matrix_with_nan_or_infinity_spoils_itself_alone(cuda_device):
    g = torch.Generator(device="cuda").manual_seed(6)
    for rows, cols in [(64, 100), (200, 140)]:
        mats = [_gradient(rows, cols, g) for _ in range(4)]
        clean = orthogonalize(mats)
        mats[1][3, 4], mats[2][0, 0] = float("nan"), float("inf")
        got = orthogonalize(mats)
        assert torch.equal(got[0], clean[0]) and torch.equal(got[3], clean[3])
        assert torch.isnan(got[1]).all() and torch.isnan(got[2]).all()


def test_singular_values_follow_the_polynomial(cuda_device):
    """s <- a s + b s^3 + c s^5 on the singular values: for s0 in
    [0.003, 1] / |.|_F the values end in [0.65, 1.25] after five steps."""
    g = torch.Generator(device="cuda").manual_seed(7)
    q = torch.linalg.qr(torch.randn(128, 128, device="cuda", generator=g, dtype=torch.float64))[0]
    r = torch.linalg.qr(torch.randn(257, 128, device="cuda", generator=g, dtype=torch.float64))[0]
    s = torch.logspace(-0.5, 0, 128, device="cuda", dtype=torch.float64)
    G = ((q * s) @ r.mT).float()
    a, b, c = COEFFICIENTS
    t = s / s.norm()
    for _ in range(5):
        t = a * t + b * t ** 3 + c * t ** 5
    got = torch.linalg.svdvals(orthogonalize(G).double())
    assert (got - t.sort(descending=True).values).abs().max() < 1e-4
    assert got.min() > 0.65 and got.max() < 1.25


def _step_case(shapes, g):
    w = [torch.randn(r, c, device="cuda", generator=g) * 0.1 for r, c in shapes]
    gr = [_gradient(r, c, g, 0.01) for r, c in shapes]
    m = [_gradient(r, c, g, 0.01) for r, c in shapes]
    return w, gr, m


def _check_step(w0, g0, m0, w, m, lr, mu, nesterov, decay):
    for W, G, M, gotw, gotm in zip(w0, g0, m0, w, m):
        M2 = mu * M.double() + (1 - mu) * G.double()
        assert ((gotm.double() - M2).abs() <= 4 * U * (mu * M.double().abs() + (1 - mu) * G.double().abs())).all()
        Un = mu * M2 + (1 - mu) * G.double() if nesterov else M2
        want, tol = _tolerance(Un.float())
        # U itself is rounded to float32 a few times: elements off by 4 U, a relative 2-norm of 4 U before the
        # iteration, which amplifies it by at most a^5 = 485 relative to singular values of 0.7
        gain = lr * math.sqrt(max(1.0, W.shape[0] / W.shape[1]))
        W2 = (1 - lr * decay) * W.double() - gain * want
        off = (gotw.double() - W2).norm().item()
        assert off <= 4 * U * W.double().norm().item() + gain * (tol + 4 * U * 485), (tuple(W.shape), off)


@pytest.mark.parametrize("nesterov,decay,mu", [(True, 0.0, 0.95), (False, 0.1, 0.9), (True, 0.01, 0.0)])
def test_step_against_float64(nesterov, decay, mu, cuda_device):
    g = torch.Generator(device="cuda").manual_seed(8)
    shapes = [(64, 129), (64, 64), (128, 257), (128, 5), (300, 64), (200, 333), (256, 513), (0, 5), (1, 1)]
    w0, g0, m0 = _step_case(shapes, g)
    w, m = [t.clone() for t in w0], [t.clone() for t in m0]
    gr = [t.clone() for t in g0]
    muon_step(w, gr, m, lr=0.03, momentum=mu, nesterov=nesterov, weight_decay=decay)
    _check_step(w0, g0, m0, w, m, 0.03, mu, nesterov, decay)
    assert all(torch.equal(a, b) for a, b in zip(gr, g0))   # gradients are only read
    # the rate from the device is the same call with that float32's value, bit for bit
    rate, runs = torch.tensor([0.03], device="cuda"), []
    for lr in (rate, rate.item()):
        w2, m2 = [t.clone() for t in w0], [t.clone() for t in m0]
        muon_step(w2, gr, m2, lr=lr, momentum=mu, nesterov=nesterov, weight_decay=decay)
        runs.append(w2 + m2)
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_step_on_slices_leaves_their_surroundings(cuda_device):
    g = torch.Generator(device="cuda").manual_seed(9)
    for rows, cols in [(40, 70), (150, 137)]:
        wide = torch.randn(3, rows + 2, cols + 9, device="cuda", generator=g)
        before = wide.clone()
        w, gr, m = (wide[k, 1:1 + rows, 4:4 + cols] for k in range(3))
        muon_step([w], [gr], [m], lr=0.1)
        _check_step(*([before[k, 1:1 + rows, 4:4 + cols]] for k in range(3)), [w], [m], 0.1, 0.95, True, 0.0)
        inside = torch.zeros_like(wide, dtype=torch.bool)
        inside[[0, 2], 1:1 + rows, 4:4 + cols] = True
        assert torch.equal(wide[~inside], before[~inside])


def test_optimizer_state_closure_and_groups(cuda_device):
    g = torch.Generator(device="cuda").manual_seed(10)
    w0, g0, _ = _step_case([(64, 64), (96, 32), (20, 20)], g)
    ps = [torch.nn.Parameter(t.clone()) for t in w0]
    opt = Muon([{"params": ps[:1]}, {"params": ps[1:], "lr": 0.5, "nesterov": False}], lr=0.1, weight_decay=0.1)
    ref = [t.clone() for t in w0]
    mom = [torch.zeros_like(t) for t in w0]
    for k in range(3):
        for p, t in zip(ps[:2], g0):   # the last one has no gradient: left alone
            p.grad = t * (k + 1)
        version = ps[0]._version
        assert opt.step(lambda: torch.tensor(3.0)) == 3.0
        assert ps[0]._version > version
        muon_step(ref[:1], [g0[0] * (k + 1)], mom[:1], lr=0.1, weight_decay=0.1)
        muon_step(ref[1:2], [g0[1] * (k + 1)], mom[1:2], lr=0.5, nesterov=False, weight_decay=0.1)
        if k == 1:   # state moves through a checkpoint
            other = Muon([{"params": ps[:1]}, {"params": ps[1:], "lr": 0.5, "nesterov": False}], lr=0.1, weight_decay=0.1)
            other.load_state_dict(opt.state_dict())
            opt = other
    assert all(torch.equal(p.detach(), r) for p, r in zip(ps, ref))
    assert torch.equal(opt.state[ps[0]]["momentum_buffer"], mom[0]) and ps[2] not in opt.state


def _model_step(opt_of, dev):
    b = molecules(24, seed=3)
    torch.manual_seed(0)
    model = EGNN(5, 64, 1, n_layers=3, device=dev, node_norm=True)
    opts = opt_of(model)
    csr = CSR.from_edges(b.row, b.col, n_nodes=b.n_nodes, device=dev)
    h, x, gp, tgt = b.h.to(dev), b.x.to(dev), b.graph_ptr.to(dev), b.target.to(dev)

    def step():
        for o in opts:
            o.zero_grad(set_to_none=True)
        ho, _ = model(h, x, csr)
        loss = graph_sum_mse(ho[:, 0], gp, tgt)
        loss.backward()
        for o in opts:
            o.step()
        return loss.detach()

    return model, step


def test_normalised_model_trained_with_muon_captured_equals_eager(cuda_device):
    """The operators together, as a training step uses them: EGNN with norms,
    the loss, the backward, Muon on the matrices and SGD on the vectors,
    eager and captured; the learning rate is a device tensor that changes
    between replays."""
    def build():
        lr = torch.tensor(0.02, device=cuda_device)

        def opt_of(model):
            mats, rest = Muon.split(model.parameters())
            assert len(mats) == 3 * 5 + 1 and all(p.dim() == 1 or min(p.shape) == 1 for p in rest)
            return [Muon(mats, lr=lr, weight_decay=0.01), torch.optim.SGD(rest, lr=1e-4)]

        return (lr, *_model_step(opt_of, cuda_device))

    lr, model, step = build()
    for _ in range(2):
        step()
    eager = []
    for k in range(4):
        lr.fill_(0.02 / (k + 1))
        eager.append(step().clone())
    lr2, model2, step2 = build()
    graphed = GraphedStep(step2, warmup=2)
    replayed = []
    for k in range(4):
        lr2.fill_(0.02 / (k + 1))
        replayed.append(graphed.replay().clone())
    torch.cuda.synchronize()
    graphed.release()
    eager, replayed = torch.stack(eager), torch.stack(replayed)
    assert torch.isfinite(eager).all() and not torch.equal(eager[0], eager[-1])
    assert torch.equal(eager, replayed)
    for (name, a), b in zip(model.named_parameters(), model2.parameters()):
        assert torch.equal(a, b), name


def test_two_streams_at_once(cuda_device):
    g = torch.Generator(device="cuda").manual_seed(11)
    sets = [[_gradient(r, c, g) for r, c in [(128, 257), (64, 64), (200, 140)]] for _ in range(2)]
    want = [orthogonalize(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(8):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(orthogonalize(sets[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for outs in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want[k]))


def test_waits_that_run_out_are_reported_and_the_context_stays_usable(cuda_device, monkeypatch):
    """EGNN_DEBUG_WAIT_POLLS=0 makes the accumulator readers of both kernels
    give up on their first wait (nothing hangs: the products complete and are
    drained); the status says so once, and later calls give the same results."""
    lib = nat.lib()
    g = torch.Generator(device="cuda").manual_seed(12)
    mats = [_gradient(r, c, g) for r, c in [(64, 129), (128, 257), (200, 333), (256, 513)]]
    monkeypatch.delenv("EGNN_DEBUG_WAIT_POLLS", raising=False)
    want = orthogonalize(mats)
    assert lib.egnn_device_status(nat.stream_ptr()) == nat.EGNN_OK, nat.last_error()
    for only in (mats[:2], mats[2:]):   # one kernel, then the other
        monkeypatch.setenv("EGNN_DEBUG_WAIT_POLLS", "0")
        orthogonalize(only)
        assert lib.egnn_device_status(nat.stream_ptr()) == nat.EGNN_ERR_CUDA and "timed out" in nat.last_error()
        assert lib.egnn_device_status(nat.stream_ptr()) == nat.EGNN_OK
        monkeypatch.delenv("EGNN_DEBUG_WAIT_POLLS")
        assert all(torch.equal(a, b) for a, b in zip(orthogonalize(mats), want))


def test_many_matrices_and_two_graphs_that_share_a_pool(cuda_device):
    """More matrices than one launch takes, of both kernels, and two captured
    calls whose workspaces come from one pool, replayed in turn."""
    g = torch.Generator(device="cuda").manual_seed(13)
    mats = [_gradient(*s, g) for s in [(40, 60), (130, 150)] * 70]
    want = orthogonalize(mats)
    assert all(torch.equal(o, orthogonalize(t)) for t, o in list(zip(mats, want))[::23])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        orthogonalize(mats[:4])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for k in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[k], pool=graphs[0].pool() if k else None):
            outs.append(orthogonalize(mats[2 * k:2 * k + 2]))
    for _ in range(3):
        for k in (0, 1):
            graphs[k].replay()
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(a, b) for a, b in zip(outs[k], want[2 * k:2 * k + 2]))


@pytest.mark.parametrize("shapes", [[(64, 2000)], [(257, 2100), (40, 50)], [(256, 513)] * 30])
def test_waits_that_run_out_in_pieces_and_wide_tiles(shapes, cuda_device, monkeypatch):
    """As above, for long sums in pieces, a side stream, and tiles of 128 columns."""
    lib = nat.lib()
    g = torch.Generator(device="cuda").manual_seed(19)
    mats = [_gradient(*s, g) for s in shapes]
    monkeypatch.delenv("EGNN_DEBUG_WAIT_POLLS", raising=False)
    want = orthogonalize(mats)
    assert lib.egnn_device_status(nat.stream_ptr()) == nat.EGNN_OK, nat.last_error()
    monkeypatch.setenv("EGNN_DEBUG_WAIT_POLLS", "0")
    orthogonalize(mats)
    assert lib.egnn_device_status(nat.stream_ptr()) == nat.EGNN_ERR_CUDA and "timed out" in nat.last_error()
    monkeypatch.delenv("EGNN_DEBUG_WAIT_POLLS")
    assert all(torch.equal(a, b) for a, b in zip(orthogonalize(mats), want))


@pytest.mark.parametrize("count", [13, 30, 64, 75])
def test_large_matrices_that_share_the_device(count, cuda_device):
    """Lists of equal and of different sizes, more than one launch takes among
    them: each result is that of a call of its own, bit for bit."""
    g = torch.Generator(device="cuda").manual_seed(18)
    sizes = [(256, 513), (256, 256), (513, 256), (129, 130), (1, 1200), (300, 700), (256, 512), (140, 1000), (520, 560)]
    mats = [_gradient(*sizes[(k * k) % len(sizes)], g) for k in range(count)]
    once = [orthogonalize(t) for t in mats]
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(orthogonalize(mats), once))
    equal = [_gradient(256, 513, g) for _ in range(count)]
    got = orthogonalize(equal)
    assert all(torch.equal(got[k], orthogonalize(equal[k])) for k in range(0, count, 5))


def test_batches_share_the_workspace(cuda_device):
    """More large matrices than a batch holds, small ones between them."""
    g = torch.Generator(device="cuda").manual_seed(20)
    sizes = [(130, 140), (64, 64), (300, 200), (20, 2000)]
    mats = [_gradient(*sizes[k % 4], g) for k in range(300)]
    got = orthogonalize(mats)
    for k in (0, 1, 84, 85, 86, 87, 170, 171, 172, 256, 258, 298, 299):
        assert torch.equal(got[k], orthogonalize(mats[k]))


@pytest.mark.parametrize("shapes", [[(100, 2192)], [(100, 2192), (64, 1100)], [(1, 16384), (257, 2100)],
                                    [(256, 513)] * 30, [(300, 700)] * 20])
def test_many_calls_give_the_same(shapes, cuda_device):
    """Blocks with no tile of a product, one, and several: what warps hand over
    must be complete however far they are apart."""
    g = torch.Generator(device="cuda").manual_seed(21)
    mats = [_gradient(*s, g) for s in shapes]
    want = [orthogonalize(t) for t in mats]
    for _ in range(60):
        outs = [orthogonalize(mats) for _ in range(10)]
        assert all(torch.equal(a, b) for out in outs for a, b in zip(out, want))


def test_more_small_matrices_than_a_batch_holds(cuda_device):
    g = torch.Generator(device="cuda").manual_seed(17)
    mats = [_gradient(9 + k % 5, 20, g) for k in range(333)] + [_gradient(140, 150, g)]
    got = orthogonalize(mats)
    for k in (0, 159, 160, 161, 319, 320, 332, 333):
        assert torch.equal(got[k], orthogonalize(mats[k]))
    _check(mats[200], got[200])


def test_rows_far_apart_and_an_offset_past_32_bits(cuda_device):
    """Row strides that put a matrix over more than 4 GB."""
    g = torch.Generator(device="cuda").manual_seed(14)
    store = torch.empty(34 * (1 << 27), dtype=torch.bfloat16, device="cuda")   # 9.1 GB
    far = store.as_strided((33, 50), (1 << 27, 1))
    far.copy_(_gradient(33, 50, g))
    near = far.clone()
    assert torch.equal(orthogonalize(far), orthogonalize(near))
    x = store.as_strided((33, 64), (1 << 27, 1))
    x.normal_(generator=g)
    layer = torch.nn.LayerNorm(64, device="cuda")
    with torch.no_grad():
        assert torch.equal(layer_norm(x, layer), layer_norm(x.clone(), layer))


def test_tensors_that_a_step_would_spoil_are_refused(cuda_device):
    def t(*shape, dtype=torch.float32):
        return torch.zeros(*shape, dtype=dtype, device="cuda")

    store = t(40, 40)
    w, g, m = t(40, 40), t(40, 40), t(40, 40)
    for args in (([w, w], [g, g], [m, t(40, 40)]), ([w], [g], [w]), ([store], [g], [store.view(40, 40)]),
                 ([w], [m.view(40, 40)], [m]), ([w], [w], [m]), ([t(40, 41)[:, 1:].t()], [g], [m]), ([w], [g], [m.t()[:, ::2]]),
                 ([w], [g], [m.cpu()]), ([w], [g], [m], torch.tensor(0.1)), ([w], [g], [m], t(2)),
                 ([t(40)], [t(40)], [t(40)]), ([t(1100, 1100)], [t(1100, 1100)], [t(1100, 1100)])):
        with pytest.raises(ValueError):
            muon_step(*args[:3], lr=args[3] if len(args) > 3 else 0.1)
    for args in (([t(4, 4, dtype=torch.float64)], [t(4, 4)], [t(4, 4)]), ([w], [g.bfloat16()], [m])):
        with pytest.raises(TypeError):
            muon_step(*args, lr=0.1)
    with pytest.raises(ValueError, match="one device"):
        orthogonalize([w, w.cpu()])
    with pytest.raises(TypeError):
        orthogonalize(t(4, 4, dtype=torch.float64))
    with pytest.raises(ValueError, match="at most"):
        orthogonalize(t(1030, 1030))
    with pytest.raises(nat.EgnnError, match="grow"):
        orthogonalize(w, coefficients=(5.0, 0.0, 0.0))
    muon_step([], [], [], lr=0.1)
    assert not any(x.any() for x in (w, g, m, store))
