"""Timed cases of the normalisation operators of training: layer norm (with the
SiLU that follows it in a radial MLP) and its gradients, and the norm and the
clipping of a model's gradients.

``run`` computes each operator in its plain form (elementary torch operations
in 32 bits, sums over a whole model in 64) or, with ``own``, through
``mace_mlx_b200.norms``.

Definitions, for rows x of C channels:

    mean = sum x / C,  var = sum (x - mean)^2 / C,  xhat = (x - mean) / sqrt(var + eps)
    y = f(w xhat + b)          f: the identity, or f(z) = z / (1 + exp(-z))

    norm = sqrt(sum over all tensors of g^2)
    clipped g = g min(1, max_norm / (norm + 1e-6))
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
FLOAT = {"float32": torch.float32, "bfloat16": torch.bfloat16}
SIZE = {"float32": 4, "bfloat16": 2}


def _rows(name, op, n, c, **more):
    base = {"name": name, "op": op, "n": n, "c": c, "silu": False, "dtype": "float32", "param": "float32", "slot": 0}
    return base | more


def _grads(name, op, channels, elements, layers, ells, **more):
    base = {"name": name, "op": op, "channels": channels, "elements": elements, "layers": layers, "ells": ells,
            "dtype": "float32", "out": "", "flat": False}
    return base | more


def listed():
    return [
        # scalar features of the 1000-atom headline cell: a call whose time is launch latency
        _rows("norm-rows-cell-1000", "rows", 1000, 128),
        # a hidden layer of the radial MLP (64 wide, SiLU behind the norm) over the edges of that cell
        _rows("norm-silu-edges-46k", "rows", 46_348, 64, silu=True),
        # the same over a box of about 90 000 atoms at 45 neighbours
        _rows("norm-silu-edges-4m", "rows", 4_000_003, 64, silu=True),
        # scalar slot of a (0e + 1o) node table in 16 bits, parameters kept in 32
        _rows("norm-slot-bf16", "rows", 400_000, 128, dtype="bfloat16", slot=3),
        # gradients of the smallest call
        _rows("norm-grad-cell-1000", "rows_grad", 1000, 128),
        # gradients of the radial MLP's hidden layer: long sums over the edges for each of 64 channels
        _rows("norm-silu-grad-edges-2m", "rows_grad", 2_000_001, 64, silu=True),
        # odd width in 16 bits: rows that begin at any 2-byte address
        _rows("norm-silu-grad-odd-bf16", "rows_grad", 300_007, 97, silu=True, dtype="bfloat16", param="bfloat16"),
        # a whole node row, 128 channels of l <= 3 (16 components), taken as one vector
        _rows("norm-grad-wide", "rows_grad", 20_011, 2048),
        # gradient norm of a small model: tens of small tensors
        _grads("grad-norm-small", "norm", 32, 4, 1, 1),
        # the same of a large one in 16 bits, its gradients one behind the other in one buffer
        _grads("grad-norm-large-bf16", "norm", 256, 89, 4, 3, dtype="bfloat16", flat=True),
        # an ordinary step of the headline architecture: below the bound, so the gradients stay as they are
        _grads("clip-idle-medium", "clip", 128, 89, 2, 2),
        # accumulated 16-bit gradients of a large model, clipped into the 32-bit gradients of its optimiser
        _grads("clip-large-bf16-f32", "clip", 256, 89, 4, 3, dtype="bfloat16", out="float32"),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _drawn(case):
    del case["name"]
    return case


def draw(rng):
    op = rng.choice(["rows", "rows", "rows_grad", "rows_grad", "rows_grad", "norm", "clip"])
    dtype = rng.choice(["float32", "float32", "bfloat16"])
    if op in ("rows", "rows_grad"):
        c = rng.choice([64, 96, 128, _log_uniform(rng, 8, 512), _log_uniform(rng, 512, 8192)])
        slot = rng.choice([0, 0, 0, 1, 3])
        # at most the values of the largest listed case, gaps between the rows of a slot among them
        most = (256_000_000 if op == "rows" else 128_000_000) // (c * (1 + slot))
        return _drawn(_rows("", op, _log_uniform(rng, 1, min(4_000_000, most)), c, silu=rng.random() < 0.5, dtype=dtype,
                            param=rng.choice(["float32", dtype]), slot=slot))
    shape = (_log_uniform(rng, 4, 256), _log_uniform(rng, 1, 89), rng.randint(1, 4), rng.randint(1, 3))
    out = rng.choice(["", "float32", dtype]) if op == "clip" else ""
    return _drawn(_grads("", op, *shape, dtype=dtype, out=out, flat=rng.random() < 0.3))


# ------------------------------------------------------------------ inputs
def _parameters(case):
    """Shapes of the parameters of an equivariant message-passing model: embedding, and per layer the linear maps of
    each degree, a radial MLP with its layer norms, species-indexed matrices, contraction weights and a readout."""
    c, e = case["channels"], case["elements"]
    shapes = [(e, c)]
    for layer in range(case["layers"]):
        ells = 1 if layer == 0 else case["ells"]
        shapes += [(c, c)] * ells
        for wide, deep in ((64, 8), (64, 64), (64, 64)):
            shapes += [(wide, deep), (wide,), (wide,), (wide,)]
        shapes += [(4 * ells * c, 64)]
        shapes += [(c, c)] * 4 * ells
        shapes += [(c, e, c)] * ells
        shapes += [(e, paths, c) for paths in (23, 4, 1, 51, 6, 1)]
        shapes += [(c, c)] * ells + [(c, 1)]
    return shapes + [(c, 16), (16, 1)]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    if case["op"] in ("rows", "rows_grad"):
        n, c, dt = case["n"], case["c"], FLOAT[case["dtype"]]
        # pre-activations: channels of their own scale and offset
        wide = normal(n, c * (1 + case["slot"]))
        wide = (wide * (0.5 + torch.rand(wide.shape[1], generator=gen, device=dev)) + normal(wide.shape[1])).to(dt)
        s["x"] = wide[:, :c]
        s["weight"] = (1.0 + 0.1 * normal(c)).to(FLOAT[case["param"]])
        s["bias"] = (0.1 * normal(c)).to(FLOAT[case["param"]])
        if case["op"] == "rows_grad":
            s["dy"] = (0.01 * normal(n, c)).to(dt)
        return s
    shapes, dt = _parameters(case), FLOAT[case["dtype"]]
    rough = [10.0 ** -(1 + i % 3) for i in range(len(shapes))]  # tensors of unlike magnitude
    s["grad_buffer"], s["grads"] = _buffer(case, dt, dev)
    for g, r in zip(s["grads"], rough):
        g.copy_(r * normal(*g.shape))
    s["clipped_buffer"], s["clipped"] = _buffer(case, FLOAT[case["out"]], dev) if case["out"] else (None, None)
    # the bound lies far above the norm where gradients stay in place, at half of it where they are clipped
    expected = math.sqrt(sum(math.prod(shape) * r * r for shape, r in zip(shapes, rough)))
    s["max_norm"] = expected * (0.5 if case["out"] else 10.0)
    return s


def _buffer(case, dtype, dev):
    """One buffer of zeros and a tensor for every parameter in it: with ``flat`` one behind the other, else each at a
    multiple of 128 values, as an allocator places them."""
    shapes = _parameters(case)
    sizes = [math.prod(shape) for shape in shapes]
    steps = sizes if case["flat"] else [-(-size // 128) * 128 for size in sizes]
    buffer = torch.zeros(sum(steps), dtype=dtype, device=dev)
    parts = buffer.split(steps)
    return buffer, [part[:size].view(shape) for part, size, shape in zip(parts, sizes, shapes)]


# -------------------------------------------------------------- plain forms
def _normalised(s):
    x = s["x"].float()
    centred = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt(centred.square().mean(-1, keepdim=True) + EPS)
    return centred * rstd, rstd


def _plain_rows(s):
    xhat, _ = _normalised(s)
    z = xhat * s["weight"].float() + s["bias"].float()
    if s["silu"]:
        z = z / (1.0 + torch.exp(-z))
    return z.to(s["x"].dtype)


def _plain_rows_grad(s):
    xhat, rstd = _normalised(s)
    w, dz = s["weight"].float(), s["dy"].float()
    if s["silu"]:
        z = xhat * w + s["bias"].float()
        sig = 1.0 / (1.0 + torch.exp(-z))
        dz = dz * sig * (1.0 + z * (1.0 - sig))
    dw = (dz * xhat).sum(0)
    db = dz.sum(0)
    dxhat = dz * w
    dx = rstd * (dxhat - dxhat.mean(-1, keepdim=True) - xhat * (dxhat * xhat).mean(-1, keepdim=True))
    return {"x": dx.to(s["x"].dtype), "weight": dw.to(s["weight"].dtype), "bias": db.to(s["bias"].dtype)}


def _plain_norm(s):
    squares = [torch.sum(g.float().square(), dtype=torch.float64) for g in s["grads"]]
    return torch.stack(squares).sum().sqrt()


def _plain_clip(s):
    norm = _plain_norm(s)
    scale = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    into = s["grads"] if s["clipped"] is None else s["clipped"]
    for g, clipped in zip(s["grads"], into):
        clipped.copy_((g.float() * scale).to(clipped.dtype))
    return {"norm": norm.float(), "grads": s["grad_buffer"] if s["clipped"] is None else s["clipped_buffer"]}


def _plain(s):
    op = s["op"]
    if op == "rows":
        return _plain_rows(s)
    if op == "rows_grad":
        return _plain_rows_grad(s)
    return _plain_norm(s).float() if op == "norm" else _plain_clip(s)


def _own(s):
    from mace_mlx_b200 import norms

    op = s["op"]
    if op in ("rows", "rows_grad"):
        more = {"eps": EPS, "activation": "silu" if s["silu"] else None}
        if op == "rows":
            return norms.layer_norm(s["x"], s["weight"], s["bias"], **more)
        dx, dw, db = norms.layer_norm_grad(s["x"], s["dy"], s["weight"], s["bias"], **more)
        return {"x": dx, "weight": dw, "bias": db}
    if op == "norm":
        return norms.grad_norm(s["grads"])
    norm = norms.clip_grads(s["grads"], s["max_norm"], out=s["clipped"])
    return {"norm": norm, "grads": s["grad_buffer"] if s["clipped"] is None else s["clipped_buffer"]}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------- definitions
def work(case):
    op, b = case["op"], SIZE[case["dtype"]]
    if op in ("rows", "rows_grad"):
        n, c, p = case["n"], case["c"], SIZE[case["param"]]
        act = 4 if case["silu"] else 0
        if op == "rows":
            return {"bytes": 2 * b * n * c + 2 * p * c, "flops": (8 + act) * n * c}
        return {"bytes": 3 * b * n * c + 4 * p * c, "flops": (18 + 2 * act) * n * c}
    values = sum(math.prod(shape) for shape in _parameters(case))
    if op == "norm" or not case["out"]:  # below the bound nothing has to be written
        return {"bytes": b * values + 4, "flops": 2 * values}
    return {"bytes": (b + SIZE[case["out"]]) * values + 4, "flops": 3 * values}


def _define_rows(x, w, b, silu):
    var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
    z = torch.addcmul(b, (x - mean) / torch.sqrt(var + EPS), w)
    return z * torch.special.expit(z) if silu else z


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "rows":
        return _define_rows(s["x"].double(), s["weight"].double(), s["bias"].double(), s["silu"])
    if op == "rows_grad":
        w, b = (s[k].double().requires_grad_() for k in ("weight", "bias"))
        parts = []
        for x, dy in zip(s["x"].split(500_000), s["dy"].split(500_000)):  # rows do not meet: gradients of w and b add up
            x = x.double().requires_grad_()
            _define_rows(x, w, b, s["silu"]).backward(dy.double())
            parts.append(x.grad)
        return {"x": torch.cat(parts), "weight": w.grad, "bias": b.grad}
    every = s["grad_buffer"].double()  # (zeros between the tensors)
    norm = torch.linalg.vector_norm(every)
    if op == "norm":
        return norm
    scale = torch.minimum(norm.new_ones(()), s["max_norm"] / (norm + 1e-6))
    return {"norm": norm, "grads": every * scale}
