"""Timed cases of the species operators: grouping atoms (or edges) by species,
the species embedding with its table gradient, the species-indexed linear map
with its gradients, and the 8-bit row checkpoint with the weight gradient that
reads it.

``run`` computes each operator in its plain form (elementary torch operations
in 32 bits) or, with ``own``, through ``mace_mlx_b200.species``.  A species
index outside ``[0, g)`` marks a padding row: it belongs to no group, its
outputs are zero and it adds nothing to a gradient.
"""

from __future__ import annotations

import math

import torch

own = False

BLOCK8 = 128  # channels that share one scale of an 8-bit checkpoint
FLOAT = {"float32": torch.float32, "bfloat16": torch.bfloat16}
LIPSO = (3.0, 1.0, 4.0, 0.5)  # Li : P : S : O of the four-species box


def _case(name, op, n, g, mix, **more):
    base = {"name": name, "op": op, "n": n, "g": g, "mix": mix, "pad": 0.0, "d": 1, "k": 0, "m": 0,
            "dtype": "float32", "slot": False}
    return base | more


def listed():
    return [
        # one small cell: a call whose time is launch latency
        _case("group-cell-1000", "group", 1000, 89, "even"),
        # the species pair (89 x 89) of every directed edge of about 90 000 atoms at 45 neighbours
        _case("group-edge-pairs-4m", "group", 4_000_003, 7921, "even", pad=0.01),
        # node embedding of the 1000-atom headline cell, 128 channels
        _case("embed-cell-1000", "embed", 1000, 89, "even", k=128),
        # node embedding of the 1 000 000-atom system
        _case("embed-1m", "embed", 1_000_000, 89, "even", k=128, pad=0.001),
        # its table gradient where four species hold all atoms (long sums over few rows)
        _case("embed-grad-1m-lipso", "embed_grad", 1_000_000, 4, "lipso", k=128),
        # a table of species pairs read per edge: many short sums, 64 radial features in 16 bits
        _case("embed-grad-pairs-bf16", "embed_grad", 1_500_007, 7921, "even", k=64, dtype="bfloat16", pad=0.01),
        # skip connection of the 1000-atom cell: one species of 89 present, vectors in a (0e + 1o) table
        _case("linear-si-1000", "linear", 1000, 89, "one", d=3, k=128, m=128, slot=True),
        # the same map over a large four-species system
        _case("linear-lipso-200k", "linear", 200_000, 4, "lipso", d=3, k=128, m=128, slot=True),
        # both gradients on the 8000-atom box, l = 2 features
        _case("linear-grad-lipso-8000", "linear_grad", 8000, 4, "lipso", d=5, k=128, m=128),
        # both gradients of 96-channel scalars in 16 bits over all elements: ragged groups
        _case("linear-grad-89-bf16", "linear_grad", 300_007, 89, "even", k=96, m=96, dtype="bfloat16", pad=0.01),
        # writing the 8-bit checkpoint of a layer's (0e + 1o) features and reading it back
        _case("checkpoint-400k", "checkpoint", 400_000, 1, "one", d=4, k=128),
        # weight gradient from an 8-bit checkpoint, odd channel counts
        _case("checkpoint-grad-odd", "checkpoint_grad", 60_013, 10, "even", d=3, k=97, m=61, pad=0.02),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["group", "embed", "embed_grad", "linear", "linear", "linear_grad", "linear_grad", "checkpoint",
                     "checkpoint_grad"])
    pad = rng.choice([0.0, 0.0, 0.001, 0.05])
    dtype = rng.choice(["float32", "float32", "bfloat16"])
    if op == "group":
        return _drawn(op, _log_uniform(rng, 64, 4_000_000), _log_uniform(rng, 1, 8000), rng.choice(["even", "zipf"]),
                      pad=pad)
    if op in ("embed", "embed_grad"):
        mix = rng.choice(["even", "lipso", "one"])
        g = 4 if mix == "lipso" else _log_uniform(rng, 1, 8000)
        k = rng.choice([64, 96, 128, _log_uniform(rng, 1, 256)])
        # at most the 128 million values of the largest listed case
        return _drawn(op, _log_uniform(rng, 64, min(1_000_000, 100_000_000 // k)), g, mix, k=k, dtype=dtype, pad=pad)
    d = rng.choice([1, 3, 5, 7])
    k = rng.choice([64, 96, 128, _log_uniform(rng, 8, 256)])
    m = rng.choice([k, 64, 128, _log_uniform(rng, 8, 256)])
    mix = rng.choice(["even", "lipso", "one", "zipf"])
    g = 4 if mix == "lipso" else rng.choice([1, 10, 89, 119])
    if op == "checkpoint":
        return _drawn(op, _log_uniform(rng, 64, max(65, 150_000_000 // (d * k))), 1, "one", d=d, k=k, dtype=dtype)
    # the padded plain form multiplies up to 40 times the rows of a zipf mix
    rows = (4_000_000_000 if mix != "zipf" else 200_000_000) // (k * m)
    rows = min(rows, 50_000_000 // (k + m))
    return _drawn(op, _log_uniform(rng, 64, max(65, rows // d)), g, mix, d=d, k=k, m=m, dtype=dtype, pad=pad,
                  slot=rng.random() < 0.3)


def _drawn(*a, **more):
    c = _case("", *a, **more)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs
def _species(case, gen, dev):
    n, g, mix = case["n"], case["g"], case["mix"]
    u = torch.rand(n, generator=gen, device=dev)
    if mix == "one":
        z = torch.full((n,), min(13, g - 1), device=dev, dtype=torch.int64)  # one element of the table
    else:
        share = {"lipso": lambda: torch.tensor(LIPSO[:g], device=dev),
                 "even": lambda: torch.ones(g, device=dev),
                 "zipf": lambda: 1.0 / torch.arange(1, g + 1, device=dev)}[mix]()
        z = torch.searchsorted(torch.cumsum(share.double() / share.double().sum(), 0).float(), u).clamp(max=g - 1)
    if case["pad"] > 0:
        z = torch.where(torch.rand(n, generator=gen, device=dev) < case["pad"], -1, z)
    return z.to(torch.int32)


def _rows(case, width, gen, dev, slot):
    """(n, d, width) features; with ``slot`` the l > 0 slot of a wider node table."""
    n, d, dt = case["n"], case["d"], FLOAT[case["dtype"]]
    if not slot:
        return torch.randn(n, d, width, generator=gen, device=dev).to(dt)
    table = torch.randn(n, (d + 1) * width, generator=gen, device=dev).to(dt)
    return table[:, width:].view(n, d, width)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    op, g, k, m, dt = case["op"], case["g"], case["k"], case["m"], FLOAT[case["dtype"]]
    s = {"op": op, "g": g, "n": case["n"], "k": k, "m": m, "d": case["d"], "dtype": dt}
    s["species"] = _species(case, gen, dev)
    if op != "group":
        # the grouping that a program makes once per structure, and its composition
        key = torch.where(s["species"] < 0, g, s["species"].long())
        s["order"] = torch.argsort(key, stable=True).to(torch.int32)
        counts = torch.bincount(key, minlength=g + 1)[:g]
        s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        s["present"] = counts.nonzero().flatten()
        s["most"] = int(counts.max())
    if op in ("embed", "embed_grad"):
        s["scale"] = 1.0 / math.sqrt(g)
        if op == "embed":
            s["table"] = torch.randn(g, k, generator=gen, device=dev).to(dt)
        else:
            s["dy"] = torch.randn(case["n"], k, generator=gen, device=dev).to(dt)
    if op in ("linear", "linear_grad"):
        s["weight"] = torch.randn(g, k, m, generator=gen, device=dev).to(dt)
    if op in ("linear", "linear_grad", "checkpoint_grad"):
        s["alpha"] = 1.0 / math.sqrt(k)
    if op in ("linear", "linear_grad", "checkpoint"):
        s["x"] = _rows(case, k, gen, dev, case["slot"])
    if op in ("linear_grad", "checkpoint_grad"):
        s["dy"] = _rows(case, m, gen, dev, case["slot"])
    if op == "checkpoint_grad":
        s["q"], s["qscale"] = _quantise(_rows(case, k, gen, dev, False).float())
    return s


# -------------------------------------------------------------- plain forms
def _quantise(x):
    """Symmetric 8-bit rows: q = round(x / s), s = max |x| / 127 over blocks of 128 channels."""
    n, d, k = x.shape
    nb = -(-k // BLOCK8)
    xb = torch.nn.functional.pad(x, (0, nb * BLOCK8 - k)).view(n, d, nb, BLOCK8)
    scale = xb.abs().amax(-1) / 127.0
    safe = torch.where(scale > 0, scale, 1.0)
    q = torch.round(xb / safe[..., None]).to(torch.int8).view(n, d, nb * BLOCK8)[..., :k].contiguous()
    return q, scale


def _values(q, scale):
    k = q.shape[-1]
    return q.float() * scale.repeat_interleave(BLOCK8, dim=-1)[..., :k]


def _padded(s, rows):
    """(groups present, rows of the fullest group, ...) with zero rows after each group's end."""
    start = s["offsets"].long()
    j = torch.arange(s["most"], device=rows.device)
    at = start[s["present"]][:, None] + j
    inside = at < start[s["present"] + 1][:, None]
    node = s["order"].long()[at.clamp(max=s["n"] - 1)]
    picked = rows[node].float()
    return picked * inside.view(inside.shape + (1,) * (picked.dim() - 2))


def _unpadded(s, padded, tail):
    """The padded groups' rows back at their atoms; zeros at padding atoms."""
    z = s["species"].long()
    rank = torch.empty_like(z)
    rank[s["order"].long()] = torch.arange(s["n"], device=z.device)
    nth = torch.zeros(s["g"], dtype=torch.int64, device=z.device)
    nth[s["present"]] = torch.arange(s["present"].numel(), device=z.device)
    zc = z.clamp(min=0)
    at = nth[zc] * s["most"] + rank - s["offsets"].long()[zc]
    rows = padded.reshape((-1,) + tail)[at.clamp(0, s["present"].numel() * s["most"] - 1)]
    return rows * (z >= 0).view((-1,) + (1,) * len(tail))


def _by_group(s, rows, tail):
    out = torch.zeros((s["g"],) + tail, device=rows.device)
    out[s["present"]] = rows
    return out


def _plain(s):
    op, g, n, d, k, m, dt = s["op"], s["g"], s["n"], s["d"], s["k"], s["m"], s["dtype"]
    if op == "group":
        key = torch.where((s["species"] < 0) | (s["species"] >= g), g, s["species"])
        key, order = torch.sort(key, stable=True)
        bounds = torch.arange(g + 1, device=key.device, dtype=key.dtype)
        return {"order": order.to(torch.int32), "offsets": torch.searchsorted(key, bounds, out_int32=True)}
    if op == "embed":
        z = s["species"].long()
        rows = s["table"].float()[z.clamp(min=0)] * s["scale"]
        return (rows * (z >= 0)[:, None]).to(dt)
    if op == "embed_grad":
        sums = _padded(s, s["dy"]).sum(1) * s["scale"]
        return _by_group(s, sums, (k,)).to(dt)
    if op == "linear":
        rows = _padded(s, s["x"]).view(-1, s["most"] * d, k)
        y = torch.bmm(rows, s["weight"].float()[s["present"]]) * s["alpha"]
        return _unpadded(s, y, (d, m)).to(dt)
    if op == "linear_grad":
        dy = _padded(s, s["dy"]).view(-1, s["most"] * d, m)
        dx = torch.bmm(dy, s["weight"].float()[s["present"]].transpose(1, 2)) * s["alpha"]
        x = _padded(s, s["x"]).view(-1, s["most"] * d, k)
        dw = torch.bmm(x.transpose(1, 2), dy) * s["alpha"]
        return {"x": _unpadded(s, dx, (d, k)).to(dt), "weight": _by_group(s, dw, (k, m)).to(dt)}
    if op == "checkpoint":
        q, scale = _quantise(s["x"].float())
        return {"scale": scale, "values": _values(q, scale).to(dt)}
    dy = _padded(s, s["dy"]).view(-1, s["most"] * d, m)
    x = _padded(s, _values(s["q"], s["qscale"])).view(-1, s["most"] * d, k)
    return _by_group(s, torch.bmm(x.transpose(1, 2), dy) * s["alpha"], (k, m)).to(dt)


def _own(s):
    from mace_mlx_b200 import species as sp

    op = s["op"]
    if op == "group":
        groups = sp.group_species(s["species"], s["g"])
        return {"order": groups.order, "offsets": groups.offsets}
    if op == "embed":
        return sp.species_embedding(s["table"], s["species"], scale=s["scale"])
    if op == "checkpoint":
        kept = sp.checkpoint_rows(s["x"])
        return {"scale": kept.scale, "values": sp.restore_rows(kept, dtype=s["dtype"])}
    groups = sp.SpeciesGroups(s["order"], s["offsets"])
    if op == "embed_grad":
        return sp.species_embedding_grad(s["dy"], groups, scale=s["scale"])
    if op == "linear":
        return sp.species_linear(s["x"], s["weight"], groups, alpha=s["alpha"])
    if op == "linear_grad":
        dx, dw = sp.species_linear_grad(s["x"], s["dy"], s["weight"], groups, alpha=s["alpha"])
        return {"x": dx, "weight": dw}
    kept = sp.RowCheckpoint(s["q"], s["qscale"])
    return sp.species_linear_grad_weight(kept, s["dy"], groups, alpha=s["alpha"])


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------- definitions
def work(case):
    n, g, d, k, m = case["n"], case["g"], case["d"], case["k"], case["m"]
    b = 4 if case["dtype"] == "float32" else 2
    used = {"one": 1, "lipso": 4}.get(case["mix"], g)
    used = min(used, g, n)
    rows = n * d
    index = 4 * n + 4 * (g + 1)
    op = case["op"]
    if op == "group":
        return {"bytes": 4 * n + index, "flops": 0}
    if op == "embed":
        return {"bytes": 4 * n + b * used * k + b * n * k, "flops": n * k}
    if op == "embed_grad":
        return {"bytes": index + b * n * k + b * g * k, "flops": n * k}
    if op == "linear":
        return {"bytes": index + b * rows * (k + m) + b * used * k * m, "flops": 2 * rows * k * m}
    if op == "linear_grad":
        return {"bytes": index + b * rows * (2 * k + m) + b * (used + g) * k * m, "flops": 4 * rows * k * m}
    nb = -(-k // BLOCK8)
    if op == "checkpoint":
        return {"bytes": rows * (2 * b * k + 2 * k + 8 * nb), "flops": 4 * rows * k}
    return {"bytes": index + rows * (k + 4 * nb + b * m) + b * g * k * m, "flops": 2 * rows * k * m}


def exact(case, seed):
    s = prepare(case, seed)
    z, g, op = s["species"].long(), s["g"], s["op"]
    if op == "group":
        return None
    if op == "embed":
        ext = torch.cat([s["table"].double() * s["scale"], s["table"].new_zeros(1, s["k"]).double()])
        return ext[torch.where(z < 0, g, z)]
    if op == "checkpoint":
        x = s["x"].double()
        scales, values = [], []
        for part in x.split(BLOCK8, dim=-1):
            t = part.abs().amax(-1, keepdim=True) / 127.0
            scales.append(t)
            values.append(torch.round(part / t.masked_fill(t == 0, 1.0)) * t)
        return {"scale": torch.cat(scales, -1), "values": torch.cat(values, -1)}
    at = [(z == i).nonzero().flatten() for i in range(g)] if g <= 128 else None
    if op == "embed_grad":
        out = torch.zeros(g + 1, s["k"], dtype=torch.float64, device=z.device)
        return out.index_add_(0, torch.where(z < 0, g, z), s["dy"].double())[:g] * s["scale"]
    if op == "linear":
        y = torch.zeros(s["n"], s["d"], s["m"], dtype=torch.float64, device=z.device)
        for i, rows in enumerate(at):
            y[rows] = s["x"][rows].double() @ s["weight"][i].double() * s["alpha"]
        return y
    if op == "linear_grad":
        dx = torch.zeros(s["n"], s["d"], s["k"], dtype=torch.float64, device=z.device)
        dw = torch.zeros(g, s["k"], s["m"], dtype=torch.float64, device=z.device)
        for i, rows in enumerate(at):
            dy = s["dy"][rows].double()
            dx[rows] = dy @ s["weight"][i].double().T * s["alpha"]
            dw[i] = torch.einsum("ndk,ndm->km", s["x"][rows].double(), dy) * s["alpha"]
        return {"x": dx, "weight": dw}
    dw = torch.zeros(g, s["k"], s["m"], dtype=torch.float64, device=z.device)
    for i, rows in enumerate(at):
        q, t = s["q"][rows].double(), s["qscale"][rows].double()
        parts = [q[..., b * BLOCK8:(b + 1) * BLOCK8] * t[..., b:b + 1] for b in range(t.shape[-1])]
        dw[i] = torch.einsum("ndk,ndm->km", torch.cat(parts, -1), s["dy"][rows].double()) * s["alpha"]
    return dw
