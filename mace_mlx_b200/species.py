"""Species operators: the parts of a MACE model whose parameters are indexed by
an atom's species, by themselves and with their gradients, for programs that
train them.

* ``group_species``               -- stable grouping of atoms (or edges) by species
* ``species_embedding``           -- ``scale * table[species]`` (the node embedding)
* ``species_embedding_grad``      -- its table gradient
* ``species_linear``              -- ``alpha * x[n, m] @ W[species[n]]`` (the skip tensor product)
* ``species_linear_grad``         -- its input and weight gradients
* ``checkpoint_rows``, ``restore_rows`` -- feature rows kept in 8 bits between
  the forward and the backward, which ``species_linear_grad_weight`` reads

``species_embedding`` and ``species_linear`` take part in autograd when an
argument requires a gradient (once differentiable).

Every call runs hand-written kernels of ``libmace_b200`` on the current stream
of the tensors' device, allocates only its results and workspace through
torch, and neither synchronises nor reads device values, so it can be captured
into a CUDA graph.  Tensors last used on another stream need the caller's
``wait_stream``/``record_stream``, as for torch's own operators.

A species index outside ``[0, num_elements)`` (by convention -1) marks a
padding row: it belongs to no group, its outputs are zero and it adds nothing
to a gradient, whatever its features hold.

Reference: node embedding ``mace_mlx/model.py:373-438``, skip tensor product
``mace_mlx/tensor_product.py:1046-1305``; the reference has no training path.
"""

from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from . import native as nv

CHECKPOINT_BLOCK = nv.CHECKPOINT_BLOCK
MAX_GROUPS = nv.SPECIES_MAX_GROUPS
MAX_INDEX = nv.SPECIES_MAX_INDEX
_DTYPES = {torch.float32: nv.DTYPE_F32, torch.bfloat16: nv.DTYPE_BF16}

__all__ = [
    "SpeciesGroups", "RowCheckpoint", "group_species", "species_embedding", "species_embedding_grad",
    "species_linear", "species_linear_grad", "species_linear_grad_weight", "checkpoint_rows", "restore_rows",
    "error_flag",
]


class SpeciesGroups(NamedTuple):
    """Rows listed by species: group g is ``order[offsets[g]:offsets[g + 1]]``."""

    order: torch.Tensor  # (N,) int32; padding rows come last
    offsets: torch.Tensor  # (num_elements + 1,) int32, offsets[0] = 0


class RowCheckpoint(NamedTuple):
    """Feature rows in 8 bits: ``q * scale``, one scale per row and block of 128 channels."""

    q: torch.Tensor  # (N, d, C) int8
    scale: torch.Tensor  # (N, d, ceil(C / 128)) float32


# ---------------------------------------------------------------- checks
def _cuda(name: str, t: torch.Tensor) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path), got device {t.device}")
    return t


def _index(name: str, t: torch.Tensor) -> torch.Tensor:
    _cuda(name, t)
    if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 1-D int32 tensor, got {t.dtype} {tuple(t.shape)}")
    return t


def _dtype(name: str, t: torch.Tensor) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} must be float32 or bfloat16, got {t.dtype}")
    return code


def _same(name: str, t: torch.Tensor, other: torch.Tensor, dtype: bool = True) -> None:
    if t.device != other.device:
        raise ValueError(f"{name} is on {t.device}, expected {other.device}")
    if dtype and t.dtype != other.dtype:
        raise ValueError(f"{name} is {t.dtype}, expected {other.dtype}")


def _rows(name: str, t: torch.Tensor) -> tuple[int, int, int, int, int]:
    """(N, d, C, node stride, component stride) of (N, d, C) or (N, C) feature rows."""
    _cuda(name, t)
    shape = t.shape
    if len(shape) == 3:
        n, d, c = shape
        sn, sm, sc = t.stride()
    elif len(shape) == 2:
        n, c = shape
        d = 1
        sn, sc = t.stride()
        sm = c
    else:
        raise ValueError(f"{name} must be (N, d, C) or (N, C), got {tuple(shape)}")
    if not 1 <= c <= nv.SPECIES_MAX_CHANNELS or not 1 <= d <= 1024:
        raise ValueError(f"{name}: need 1..{nv.SPECIES_MAX_CHANNELS} channels and 1..1024 components, "
                         f"got {tuple(shape)}")
    if sc != 1 and c > 1:
        raise ValueError(f"{name}: channels must be contiguous (stride 1), got strides {t.stride()}")
    return n, d, c, sn, sm


def _groups(groups: SpeciesGroups, n: int, like: torch.Tensor) -> int:
    """Checks a grouping of n rows and returns its number of groups."""
    order, offsets = groups
    _index("groups.order", order)
    _index("groups.offsets", offsets)
    _same("groups.order", order, like, False)
    _same("groups.offsets", offsets, like, False)
    if order.shape[0] != n:
        raise ValueError(f"groups.order lists {order.shape[0]} rows, expected {n}")
    if offsets.shape[0] < 2:
        raise ValueError("groups.offsets needs num_elements + 1 entries")
    return offsets.shape[0] - 1


def _weight(weight: torch.Tensor, num_groups: int) -> tuple[int, int]:
    _cuda("weight", weight)
    if weight.dim() != 3 or not weight.is_contiguous():
        raise ValueError(f"weight must be a contiguous (num_elements, K, M) tensor, got {tuple(weight.shape)} "
                         f"with strides {weight.stride()}")
    if weight.shape[0] != num_groups:
        raise ValueError(f"weight has {weight.shape[0]} elements, the grouping {num_groups}")
    if num_groups > MAX_GROUPS:
        raise ValueError(f"species_linear takes at most {MAX_GROUPS} elements, got {num_groups}")
    return weight.shape[1], weight.shape[2]


def _out(out: torch.Tensor | None, shape: tuple[int, ...], like: torch.Tensor) -> torch.Tensor:
    """The result tensor: a new one, or ``out`` (a view into a wider table is fine)."""
    if out is None:
        return torch.empty(shape, dtype=like.dtype, device=like.device)
    _cuda("out", out)
    _same("out", out, like)
    if tuple(out.shape) != tuple(shape):
        raise ValueError(f"out must be {tuple(shape)}, got {tuple(out.shape)}")
    n, d, c, sn, sm = _rows("out", out)
    apart = d == 1 or sm >= c
    nested = n <= 1 or sn >= (d - 1) * sm + c
    turned = d > 1 and sn >= c and sm >= (n - 1) * sn + c
    if not ((apart and nested) or turned):
        raise ValueError(f"out rows overlap (strides {out.stride()})")
    return out


class _on:
    """The device of a call: makes it current if it is not, and gives its stream."""

    __slots__ = ("guard", "index")

    def __init__(self, t: torch.Tensor):
        self.index = t.device.index
        self.guard = None if self.index == torch.cuda.current_device() else torch.cuda.device(self.index)

    def __enter__(self) -> int:
        if self.guard is not None:
            self.guard.__enter__()
        return torch.cuda.current_stream().cuda_stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _workspace(size_fn, args: tuple, like: torch.Tensor) -> tuple[torch.Tensor, int]:
    need = C.c_int64()
    nv.check(size_fn(*args, C.byref(need)))
    return torch.empty(max(need.value, 16), dtype=torch.uint8, device=like.device), need.value


# ------------------------------------------------------------- operators
def group_species(species: torch.Tensor, num_elements: int) -> SpeciesGroups:
    """Stable grouping of rows by ``species`` (int32), up to 1 048 575 values.

    Pairs are grouped the same way: ``species[sender] * E + species[receiver]``.
    """
    _index("species", species)
    if not 1 <= num_elements <= MAX_INDEX:
        raise ValueError(f"num_elements must be 1..{MAX_INDEX}, got {num_elements}")
    n = species.shape[0]
    lib = nv.load_library()
    order = torch.empty(n, dtype=torch.int32, device=species.device)
    offsets = torch.empty(num_elements + 1, dtype=torch.int32, device=species.device)
    with _on(species) as stream:
        ws, nbytes = _workspace(lib.mace_species_group_workspace, (n, num_elements), species)
        nv.check(lib.mace_species_group(species.data_ptr(), n, num_elements, order.data_ptr(), offsets.data_ptr(),
                                        ws.data_ptr(), nbytes, stream))
    return SpeciesGroups(order, offsets)


def _embedding(table, species, scale, out):
    _cuda("table", table)
    _index("species", species)
    _same("species", species, table, False)
    code = _dtype("table", table)
    g, _, c, ts, _ = _rows("table", table)
    if table.dim() != 2 or not 1 <= g <= MAX_INDEX:
        raise ValueError(f"table must be (num_elements, C) with 1..{MAX_INDEX} rows, got {tuple(table.shape)}")
    n = species.shape[0]
    out = _out(out, (n, c), table)
    with _on(table) as stream:
        lib = nv.load_library()
        nv.check(lib.mace_species_embed(code, table.data_ptr(), ts, g, c, species.data_ptr(), n, scale,
                                        out.data_ptr(), max(out.stride(0), c), stream))
    return out


def species_embedding(table: torch.Tensor, species: torch.Tensor, *, scale: float = 1.0,
                      groups: SpeciesGroups | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``scale * table[species]`` (N, C); zero rows for padding.

    When ``table`` requires a gradient, its backward sums over ``groups``
    (made from ``species`` when not given).
    """
    if table.requires_grad and torch.is_grad_enabled():
        if out is not None:
            raise ValueError("out= cannot take part in autograd")
        return _EmbeddingFn.apply(table, species, scale, groups)
    return _embedding(table, species, scale, out)


def species_embedding_grad(grad: torch.Tensor, groups: SpeciesGroups, *, scale: float = 1.0) -> torch.Tensor:
    """Table gradient ``scale * sum of grad over each group`` (num_elements, C)."""
    code = _dtype("grad", grad)
    n, _, c, gs, _ = _rows("grad", grad)
    if grad.dim() != 2:
        raise ValueError(f"grad must be (N, C), got {tuple(grad.shape)}")
    g = _groups(groups, n, grad)
    lib = nv.load_library()
    out = torch.empty((g, c), dtype=grad.dtype, device=grad.device)
    with _on(grad) as stream:
        ws, nbytes = _workspace(lib.mace_species_embed_grad_workspace, (n, g, c), grad)
        nv.check(lib.mace_species_embed_grad(code, grad.data_ptr(), gs, groups.order.data_ptr(),
                                             groups.offsets.data_ptr(), n, g, c, scale, out.data_ptr(),
                                             ws.data_ptr(), nbytes, stream))
    return out


def _linear(x, weight, groups, alpha, transpose, out):
    code = _dtype("x", x)
    n, d, k, sn, sm = _rows("x", x)
    g = _groups(groups, n, x)
    k_in, k_out = _weight(weight, g)
    _same("weight", weight, x)
    if transpose:
        k_in, k_out = k_out, k_in
    if k != k_in:
        raise ValueError(f"x has {k} channels, the weight takes {k_in}")
    y = _out(out, x.shape[:-1] + (k_out,), x)
    ys = y.stride()
    with _on(x) as stream:
        lib = nv.load_library()
        nv.check(lib.mace_species_linear(code, x.data_ptr(), sn, sm, weight.data_ptr(), int(transpose), g, k_in, k_out,
                                         groups.order.data_ptr(), groups.offsets.data_ptr(), n, d, alpha,
                                         y.data_ptr(), ys[0], ys[1] if len(ys) == 3 else k_out, stream))
    return y


def species_linear(x: torch.Tensor, weight: torch.Tensor, groups: SpeciesGroups, *, alpha: float = 1.0,
                   transpose: bool = False, out: torch.Tensor | None = None,
                   checkpoint: bool = False) -> torch.Tensor:
    """``alpha * x[n, m] @ weight[species[n]]`` for (N, d, K) or (N, K) rows.

    ``weight`` is (num_elements, K, M); with ``transpose`` x has M channels and
    meets the transposed matrices (the input gradient).  x may be a slot of a
    node-feature table (any node and component stride, channels contiguous),
    and so may ``out``, which must not overlap x.  In autograd,
    ``checkpoint`` keeps x for the weight gradient in 8 bits
    (``checkpoint_rows``) instead of x itself.
    """
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        if out is not None or transpose:
            raise ValueError("out= and transpose= cannot take part in autograd")
        return _LinearFn.apply(x, weight, groups.order, groups.offsets, alpha, checkpoint)
    return _linear(x, weight, groups, alpha, transpose, out)


def species_linear_grad_weight(x: torch.Tensor | RowCheckpoint, grad: torch.Tensor, groups: SpeciesGroups, *,
                               alpha: float = 1.0) -> torch.Tensor:
    """Weight gradient (num_elements, K, M) from the rows x, or from their 8-bit checkpoint."""
    code = _dtype("grad", grad)
    n, d, m, gn, gm = _rows("grad", grad)
    scale = None
    if isinstance(x, RowCheckpoint):
        x, scale = _checkpoint(x)
        _same("x.q", x, grad, False)
    else:
        _dtype("x", x)
        _same("x", x, grad)
    xn, xd, k, sn, sm = _rows("x", x)
    if (xn, xd) != (n, d):
        raise ValueError(f"x rows {tuple(x.shape)} do not match grad rows {tuple(grad.shape)}")
    g = _groups(groups, n, grad)
    if g > MAX_GROUPS:
        raise ValueError(f"species_linear takes at most {MAX_GROUPS} elements, got {g}")
    lib = nv.load_library()
    dw = torch.empty((g, k, m), dtype=grad.dtype, device=grad.device)
    with _on(grad) as stream:
        ws, nbytes = _workspace(lib.mace_species_linear_wgrad_workspace, (n, d, g, k, m), grad)
        nv.check(lib.mace_species_linear_wgrad(
            code, x.data_ptr(), sn, sm, None if scale is None else scale.data_ptr(), grad.data_ptr(), gn, gm, g, k, m,
            groups.order.data_ptr(), groups.offsets.data_ptr(), n, d, alpha, dw.data_ptr(), ws.data_ptr(), nbytes,
            stream))
    return dw


def species_linear_grad(x: torch.Tensor | RowCheckpoint, grad: torch.Tensor, weight: torch.Tensor,
                        groups: SpeciesGroups, *, alpha: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """Input and weight gradients of ``species_linear`` for the output gradient ``grad``."""
    return (_linear(grad, weight, groups, alpha, True, None),
            species_linear_grad_weight(x, grad, groups, alpha=alpha))


def _checkpoint(ck: RowCheckpoint) -> tuple[torch.Tensor, torch.Tensor]:
    q, scale = ck
    _cuda("q", q)
    _cuda("scale", scale)
    if q.dtype != torch.int8 or not q.is_contiguous() or q.dim() not in (2, 3):
        raise ValueError(f"q must be contiguous int8 (N, d, C) or (N, C), got {q.dtype} {tuple(q.shape)}")
    want = tuple(q.shape[:-1]) + (-(-q.shape[-1] // CHECKPOINT_BLOCK),)
    if scale.dtype != torch.float32 or not scale.is_contiguous() or tuple(scale.shape) != want:
        raise ValueError(f"scale must be contiguous float32 {want}, got {scale.dtype} {tuple(scale.shape)}")
    _same("scale", scale, q, False)
    return q, scale


def checkpoint_rows(x: torch.Tensor) -> RowCheckpoint:
    """x (N, d, C) or (N, C) in 8 bits: per row and block of 128 channels
    ``scale = max |x| * (1 / 127)``, ``q = round(x / scale)`` (half to even), in fp32.

    The error of a value is at most half a scale.  A block that holds an
    infinity or NaN is restored as NaN.
    """
    code = _dtype("x", x)
    n, d, c, sn, sm = _rows("x", x)
    lib = nv.load_library()
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(x.shape[:-1] + (-(-c // CHECKPOINT_BLOCK),), dtype=torch.float32, device=x.device)
    with _on(x) as stream:
        nv.check(lib.mace_rows_checkpoint(code, x.data_ptr(), sn, sm, n, d, c, q.data_ptr(), scale.data_ptr(),
                                          stream))
    return RowCheckpoint(q, scale)


def restore_rows(checkpoint: RowCheckpoint, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values ``q * scale`` an 8-bit checkpoint stands for, rounded to ``dtype``."""
    q, scale = _checkpoint(checkpoint)
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"dtype must be float32 or bfloat16, got {dtype}")
    n, d, c, _, _ = _rows("q", q)
    x = torch.empty(q.shape, dtype=dtype, device=q.device)
    with _on(q) as stream:
        lib = nv.load_library()
        nv.check(lib.mace_rows_restore(code, q.data_ptr(), scale.data_ptr(), n, d, c, x.data_ptr(), stream))
    return x


def error_flag(device: int | str | torch.device | None = None) -> int:
    """Synchronise, return and clear the operators' device error flag (0: none;
    2: a bounded wait inside a kernel gave up and its outputs are incomplete)."""
    flag = C.c_int32()
    with torch.cuda.device(torch.cuda.current_device() if device is None else device):
        nv.check(nv.load_library().mace_species_error_flag(C.byref(flag)))
    return flag.value


# -------------------------------------------------------------- autograd
def _unit(grad: torch.Tensor) -> torch.Tensor:
    """The gradient with contiguous channels (sums hand back expanded ones)."""
    return grad if grad.stride(-1) == 1 else grad.contiguous()


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, species, scale, groups):
        if groups is None:
            groups = group_species(species, table.shape[0])
        elif groups.offsets.shape[0] != table.shape[0] + 1:
            raise ValueError(f"the grouping has {groups.offsets.shape[0] - 1} elements, the table {table.shape[0]}")
        ctx.save_for_backward(groups.order, groups.offsets)
        ctx.scale = scale
        return _embedding(table, species, scale, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return species_embedding_grad(_unit(grad), SpeciesGroups(*ctx.saved_tensors), scale=ctx.scale), None, None, None


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, order, offsets, alpha, checkpoint):
        groups = SpeciesGroups(order, offsets)
        y = _linear(x, weight, groups, alpha, False, None)
        need_x, need_w = ctx.needs_input_grad[:2]
        kept = (x,) if need_w else ()
        if need_w and checkpoint:
            kept = tuple(checkpoint_rows(x))
        ctx.save_for_backward(order, offsets, weight if need_x else None, *kept)
        ctx.alpha = alpha
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        order, offsets, weight, *kept = ctx.saved_tensors
        groups, grad = SpeciesGroups(order, offsets), _unit(grad)
        dx = dw = None
        if weight is not None:
            dx = _linear(grad, weight, groups, ctx.alpha, True, None)
        if kept:
            x = kept[0] if len(kept) == 1 else RowCheckpoint(*kept)
            dw = species_linear_grad_weight(x, grad, groups, alpha=ctx.alpha)
        return dx, dw, None, None, None, None
