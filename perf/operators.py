"""Timed cases of the training-step operators around the E_GCL layers.

Three operators: layer normalisation of node features (forward, and forward
with backward), orthogonalisation of matrices by Newton-Schulz products, and
the momentum step that orthogonalises its update (Muon).  ``run`` computes a
case in plain torch operations, or, with ``own`` set, through
``pymolecular_b200``.  ``exact`` is the same from the definitions in float64.

Sizes: the node counts and widths of the package's workloads (config 1: 96
molecules, H = 64, 4 layers; config 2: 512 molecules, H = 128, 7 layers;
config 4: 256 slabs, H = 256, 6 layers; config 5: one graph of 2^20 nodes,
H = 128) and odd ones between and around them.
"""
from __future__ import annotations

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
NS_EPS = 1e-7
NORM_EPS = 1e-5
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01


def layer_shapes(hidden: int, layers: int, width: int = 0, edge_attr: int = 0) -> str:
    """The weight matrices of `layers` E_GCL layers, as "RxC*count,..."; `width`
    is the node feature width next to `hidden` (0: the same)."""
    w = width or hidden
    one = [(hidden, 2 * w + 1 + edge_attr), (hidden, hidden), (hidden, w + hidden), (w, hidden), (hidden, hidden)]
    return ",".join("%dx%d*%d" % (r, c, layers) for r, c in one)


def matrices(shapes: str) -> list:
    """[(rows, cols), ...] of "RxC*count,RxC,..."."""
    found = []
    for part in shapes.split(","):
        size, _, count = part.partition("*")
        r, c = size.split("x")
        found += [(int(r), int(c))] * int(count or 1)
    return found


def listed() -> list:
    return [
        # inference on config 1's batch: the smallest call, where latency counts
        {"name": "norm infer 96 molecules", "op": "norm", "rows": 1850, "cols": 64, "dtype": "f32", "train": False, "pad": 0},
        # a training step's normalisation on config 2's batch, the default workload
        {"name": "norm train 512 molecules", "op": "norm", "rows": 9939, "cols": 128, "dtype": "f32", "train": True, "pad": 0},
        # config 4's batch (about 125 nodes in each of 256 slabs)
        {"name": "norm train 256 slabs", "op": "norm", "rows": 32117, "cols": 256, "dtype": "f32", "train": True, "pad": 0},
        # config 5's single graph: the largest
        {"name": "norm train 2^20 nodes", "op": "norm", "rows": 1 << 20, "cols": 128, "dtype": "f32", "train": True, "pad": 0},
        # odd width, half the bytes, rows that are a slice of wider ones
        {"name": "norm train odd bf16 slice", "op": "norm", "rows": 30011, "cols": 321, "dtype": "bf16", "train": True, "pad": 7},
        # few wide rows, as of a wide feature table
        {"name": "norm infer wide f16", "op": "norm", "rows": 2053, "cols": 4096, "dtype": "f16", "train": False, "pad": 0},
        # one weight's update: the smallest call
        {"name": "orthogonalize one", "op": "ortho", "shapes": "64x129", "dtype": "f32"},
        # every weight matrix of config 2's model
        {"name": "orthogonalize 7 layers H128", "op": "ortho", "shapes": layer_shapes(128, 7), "dtype": "f32"},
        # every weight matrix of config 4's model
        {"name": "orthogonalize 6 layers H256", "op": "ortho", "shapes": layer_shapes(256, 6), "dtype": "f32"},
        # embeddings, odd widths and edge attributes, tall and wide, bf16 gradients
        {"name": "orthogonalize ragged bf16", "op": "ortho", "shapes": "128x5,1x128,77x31*2,200x333,64x1100,513x97,3x3", "dtype": "bf16"},
        # the whole update of config 1's and config 2's models
        {"name": "muon 4 layers H64", "op": "muon", "shapes": layer_shapes(64, 4), "nesterov": True},
        {"name": "muon 7 layers H128", "op": "muon", "shapes": layer_shapes(128, 7), "nesterov": True},
    ]


def draw(rng) -> dict:
    def log_int(lo, hi):
        return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))

    op = rng.choice(["norm", "norm", "ortho", "muon"])
    if op == "norm":
        cols = log_int(8, 8192)
        rows = log_int(1, max(2, min(1 << 19, (1 << 25) // cols)))
        return {"op": "norm", "rows": rows, "cols": cols, "dtype": rng.choice(["f32", "f32", "bf16", "f16"]),
                "train": rng.random() < 0.7, "pad": rng.choice([0, 0, rng.randint(1, 64)])}
    hidden = rng.choice([32, 64, 128, 256, log_int(8, 256)])
    shapes = layer_shapes(hidden, rng.randint(1, 6), rng.choice([0, log_int(8, 256)]), rng.choice([0, rng.randint(1, 16)]))
    if rng.random() < 0.4:
        shapes += ",%dx%d,%dx%d" % (hidden, log_int(1, 64), log_int(1, 600), log_int(1, 600))
    if op == "ortho":
        return {"op": "ortho", "shapes": shapes, "dtype": rng.choice(["f32", "f32", "bf16", "f16"])}
    return {"op": "muon", "shapes": shapes, "nesterov": rng.random() < 0.7}


def generator(seed: int):
    return torch.Generator(device="cuda").manual_seed(seed)


def gradient(rows: int, cols: int, g) -> torch.Tensor:
    """A weight gradient's spectrum: sums of outer products of rank half the
    smaller side, and noise of half their size; its own overall scale."""
    k = max(1, min(rows, cols) // 2)
    u = torch.randn(rows, k, device="cuda", generator=g)
    v = torch.randn(k, cols, device="cuda", generator=g)
    e = torch.randn(rows, cols, device="cuda", generator=g)
    scale = torch.exp(2 * torch.randn((), device="cuda", generator=g) - 5)
    return scale * ((u @ v) / k ** 0.5 + 0.5 * e)


def prepare(case: dict, seed: int) -> dict:
    g = generator(seed)
    if case["op"] == "norm":
        rows, cols, dt = case["rows"], case["cols"], DTYPES[case["dtype"]]
        wide = cols + case["pad"]
        # node features: rows of different sizes around a common offset
        x = torch.randn(rows, wide, device="cuda", generator=g)
        x.mul_(torch.exp(0.5 * torch.randn(rows, 1, device="cuda", generator=g))).add_(0.5)
        layer = torch.nn.LayerNorm(cols, eps=NORM_EPS, device="cuda")
        with torch.no_grad():
            layer.weight.copy_(1 + 0.2 * torch.randn(cols, device="cuda", generator=g))
            layer.bias.copy_(0.2 * torch.randn(cols, device="cuda", generator=g))
        state = {"op": "norm", "train": case["train"], "layer": layer,
                 "x": x.to(dt)[:, :cols].detach().requires_grad_(case["train"])}
        if case["train"]:
            state["dy"] = torch.randn(rows, cols, device="cuda", generator=g).to(dt)
        return state
    sizes = matrices(case["shapes"])
    if case["op"] == "ortho":
        return {"op": "ortho", "grads": [gradient(r, c, g).to(DTYPES[case["dtype"]]) for r, c in sizes]}
    # the weights of a model lie one after another in one buffer
    flat = 0.1 * torch.randn(sum(r * c for r, c in sizes), device="cuda", generator=g)
    params = [w.view(r, c) for w, (r, c) in zip(flat.split([r * c for r, c in sizes]), sizes)]
    grads = [gradient(r, c, g) for r, c in sizes]
    buffers = [0.3 * a + gradient(r, c, g) * (a.norm() / (r * c) ** 0.5) for a, (r, c) in zip(grads, sizes)]
    return {"op": "muon", "flat": flat, "params": params, "grads": grads, "buffers": buffers, "nesterov": case["nesterov"]}


# -- the plain forms ----------------------------------------------------------

def plain_norm(x, weight, bias, dy=None):
    x32, w = x.detach().float(), weight.detach()
    centred = x32 - x32.mean(1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + NORM_EPS)
    unit = centred * rstd
    y = (unit * w + bias.detach()).to(x.dtype)
    if dy is None:
        return [y]
    d = dy.float()
    gw = d * w
    dx = rstd * (gw - gw.mean(1, keepdim=True) - unit * (gw * unit).mean(1, keepdim=True))
    return [y, dx.to(x.dtype), (d * unit).sum(0), d.sum(0)]


def plain_newton_schulz(batch):
    """(B, m, n) float32 -> the orthogonalised batch, float32."""
    a, b, c = COEFFICIENTS
    turn = batch.shape[1] > batch.shape[2]
    x = batch.mT if turn else batch
    x = x / (torch.sqrt((x * x).sum((1, 2), keepdim=True)) + NS_EPS)
    for _ in range(STEPS):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.mT if turn else x


def plain_orthogonalize(mats):
    """Matrices of one size go through one batched product."""
    sizes = {}
    for i, t in enumerate(mats):
        sizes.setdefault(tuple(t.shape), []).append(i)
    done = [None] * len(mats)
    for where in sizes.values():
        x = plain_newton_schulz(torch.stack([mats[i].float() for i in where]))
        for k, i in enumerate(where):
            done[i] = x[k].to(mats[i].dtype)
    return done


def plain_muon(params, grads, buffers, nesterov):
    torch._foreach_mul_(buffers, MOMENTUM)
    torch._foreach_add_(buffers, grads, alpha=1 - MOMENTUM)
    updates = buffers
    if nesterov:
        updates = torch._foreach_mul(buffers, MOMENTUM)
        torch._foreach_add_(updates, grads, alpha=1 - MOMENTUM)
    turned = plain_orthogonalize(updates)
    torch._foreach_mul_(params, 1 - LR * DECAY)
    torch._foreach_mul_(turned, [-LR * max(1.0, p.shape[0] / p.shape[1]) ** 0.5 for p in params])
    torch._foreach_add_(params, turned)


def run(state: dict):
    if own:
        import pymolecular_b200 as pm
    if state["op"] == "norm":
        x, layer = state["x"], state["layer"]
        if own:
            if not state["train"]:
                with torch.no_grad():
                    return [pm.layer_norm(x, layer)]
            y = pm.layer_norm(x, layer)
            return [y, *torch.autograd.grad(y, [x, layer.weight, layer.bias], state["dy"])]
        return plain_norm(x, layer.weight, layer.bias, state.get("dy"))
    if state["op"] == "ortho":
        return pm.orthogonalize(state["grads"]) if own else plain_orthogonalize(state["grads"])
    params, grads, buffers = state["params"], state["grads"], state["buffers"]
    if own:
        pm.muon_step(params, grads, buffers, lr=LR, momentum=MOMENTUM, nesterov=state["nesterov"], weight_decay=DECAY)
    else:
        plain_muon(params, grads, buffers, state["nesterov"])
    return [state["flat"], *buffers]


def work(case: dict) -> dict:
    if case["op"] == "norm":
        n, s = case["rows"] * case["cols"], SIZE[case["dtype"]]
        # x in, y out; with the backward also dy in, dx out
        return {"bytes": n * s * (4 if case["train"] else 2) + case["cols"] * (16 if case["train"] else 8),
                "flops": n * (20 if case["train"] else 8)}
    sizes = matrices(case["shapes"])
    # both symmetric products at half their multiplications
    flops = sum(STEPS * (3 * min(r, c) ** 2 * max(r, c) + min(r, c) ** 3) for r, c in sizes)
    n = sum(r * c for r, c in sizes)
    # gradient in, result out; the step: gradient, momentum and weight in, both written
    return {"bytes": n * (2 * SIZE[case["dtype"]] if case["op"] == "ortho" else 20), "flops": flops}


# -- the definitions in float64 -----------------------------------------------

def exact_norm(state):
    x, layer = state["x"].detach().double(), state["layer"]
    w, b = layer.weight.detach().double(), layer.bias.detach().double()
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    unit = x.sub_(mean).div_((var + NORM_EPS).sqrt())
    y = unit * w + b
    if not state["train"]:
        return [y]
    dy = state["dy"].double()
    dw, db = torch.einsum("ij,ij->j", dy, unit), torch.einsum("ij->j", dy)
    # the Jacobian of one row: (I - 1 1^T / C - u u^T / C) diag(w) / sigma
    h = dy.mul_(w)
    h = h - unit * (torch.einsum("ij,ij->i", h, unit) / h.shape[1])[:, None] - (torch.einsum("ij->i", h) / h.shape[1])[:, None]
    return [y, h.div_((var + NORM_EPS).sqrt()), dw, db]


def exact_orthogonal(mat):
    """The odd polynomial, STEPS times, on the singular values."""
    a, b, c = COEFFICIENTS
    x = mat.double()
    u, s, vt = torch.linalg.svd(x / (torch.linalg.matrix_norm(x) + NS_EPS), full_matrices=False)
    for _ in range(STEPS):
        s = s * (a + s.square() * (b + c * s.square()))
    return (u * s) @ vt


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["op"] == "norm":
        return exact_norm(state)
    if case["op"] == "ortho":
        return [exact_orthogonal(t) for t in state["grads"]]
    moved, buffers = [], []
    for p, g, m in zip(state["params"], state["grads"], state["buffers"]):
        g, m = g.double(), m.double()
        m = MOMENTUM * m + (1 - MOMENTUM) * g
        o = exact_orthogonal(MOMENTUM * m + (1 - MOMENTUM) * g if case["nesterov"] else m)
        gain = max(1.0, p.shape[0] / p.shape[1]) ** 0.5
        moved.append(((1 - LR * DECAY) * p.double() - LR * gain * o).reshape(-1))
        buffers.append(m)
    return [torch.cat(moved), *buffers]
