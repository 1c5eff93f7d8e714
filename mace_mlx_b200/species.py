"""Species operators: the parts of a MACE model whose parameters are indexed by
an atom's species, by themselves and with their gradients, for programs that
train parts of this form (a head on a frozen model's features, a layer of their
own).

* ``group_species``               -- stable grouping of atoms (or edges) by species
* ``species_embedding``           -- ``scale * table[species]`` (the node embedding)
* ``species_embedding_grad``      -- its table gradient
* ``species_linear``              -- ``alpha * x[n, m] @ W[species[n]]`` (the skip tensor product)
* ``species_linear_grad``         -- its input and weight gradients
* ``checkpoint_rows``, ``restore_rows`` -- feature rows kept in 8 bits between
  the forward and the backward, which ``species_linear_grad_weight`` reads

``species_embedding`` and ``species_linear`` take part in autograd when an
argument requires a gradient (once differentiable, in reverse mode: a tensor
with a forward-mode tangent is refused).

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
import functools
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

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
# These run before every call and small calls are bound by them: device
# indices and raw streams, which cost a tenth of device and stream objects.
_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream


def _cuda(name: str, t: torch.Tensor) -> int:
    """Device index of a CUDA tensor."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path), got device {t.device}")
    if forward_ad._current_level >= 0 and t.is_floating_point() and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} carries a tangent: the species operators have no forward-mode derivative")
    return t.get_device()


def _on(name: str, t: torch.Tensor, dev: int) -> None:
    if _cuda(name, t) != dev:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{dev}")


def _index(name: str, t: torch.Tensor) -> int:
    dev = _cuda(name, t)
    if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 1-D int32 tensor, got {t.dtype} {tuple(t.shape)}")
    return dev


def _dtype(name: str, dtype: torch.dtype) -> int:
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"{name} must be float32 or bfloat16, got {dtype}")
    return code


def _same_dtype(name: str, t: torch.Tensor, other: torch.Tensor) -> None:
    if t.dtype != other.dtype:
        raise ValueError(f"{name} is {t.dtype}, expected {other.dtype}")


def _rows(name: str, t: torch.Tensor) -> tuple[int, int, int, int, int]:
    """(N, d, C, node stride, component stride) of (N, d, C) or (N, C) feature rows."""
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


def _groups(groups: SpeciesGroups, n: int, dev: int) -> tuple[int, int, int]:
    """(number of groups, pointers of order and offsets) of a grouping of n rows."""
    order, offsets = groups
    if _index("groups.order", order) != dev or _index("groups.offsets", offsets) != dev:
        raise ValueError(f"the grouping is on {order.device} and {offsets.device}, expected cuda:{dev}")
    if order.shape[0] != n:
        raise ValueError(f"groups.order lists {order.shape[0]} rows, expected {n}")
    g = offsets.shape[0] - 1
    if g < 1:
        raise ValueError("groups.offsets needs num_elements + 1 entries")
    return g, order.data_ptr(), offsets.data_ptr()


def _map_limits(n: int, d: int, num_groups: int) -> None:
    if num_groups > MAX_GROUPS:
        raise ValueError(f"species_linear takes at most {MAX_GROUPS} elements, got {num_groups}")
    if n * d > nv.SPECIES_MAX_ROWS:
        raise ValueError(f"species_linear takes at most {nv.SPECIES_MAX_ROWS} rows, got {n} x {d}")


def _out(out: torch.Tensor | None, shape, like: torch.Tensor, dev: int) -> torch.Tensor:
    """The result tensor: a new one, or ``out`` (a view into a wider table is fine)."""
    if out is None:
        return like.new_empty(shape)
    _on("out", out, dev)
    _same_dtype("out", out, like)
    if out.shape != shape:
        raise ValueError(f"out must be {tuple(shape)}, got {tuple(out.shape)}")
    n, d, c, sn, sm = _rows("out", out)
    apart = d == 1 or sm >= c
    nested = n <= 1 or sn >= (d - 1) * sm + c
    turned = d > 1 and sn >= c and sm >= (n - 1) * sn + c
    if not ((apart and nested) or turned):
        raise ValueError(f"out rows overlap (strides {out.stride()})")
    return out


def _launch(dev: int, fn, *args) -> None:
    """Calls a C entry on the current stream of device ``dev``."""
    if _current_device() == dev:
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    if rc:
        nv.check(rc)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(entry: str, dev: int, *sizes: int) -> int:
    """Workspace of a C entry: it depends on the sizes and the device's SM count only."""
    need = C.c_int64()
    with torch.cuda.device(dev):
        nv.check(getattr(nv.load_library(), entry)(*sizes, C.byref(need)))
    return need.value


def _workspace(entry: str, dev: int, like: torch.Tensor, *sizes: int) -> tuple[torch.Tensor | None, int | None, int]:
    nbytes = _workspace_bytes(entry, dev, *sizes)
    if nbytes == 0:
        return None, None, 0
    ws = like.new_empty(nbytes, dtype=torch.uint8)
    return ws, ws.data_ptr(), nbytes


# ------------------------------------------------------------- operators
def group_species(species: torch.Tensor, num_elements: int) -> SpeciesGroups:
    """Stable grouping of rows by ``species`` (int32), up to 1 048 575 values.

    Pairs are grouped the same way: ``species[sender] * E + species[receiver]``.
    """
    dev = _index("species", species)
    if not 1 <= num_elements <= MAX_INDEX:
        raise ValueError(f"num_elements must be 1..{MAX_INDEX}, got {num_elements}")
    n = species.shape[0]
    order = torch.empty_like(species)
    offsets = species.new_empty(num_elements + 1)
    ws, ptr, nbytes = _workspace("mace_species_group_workspace", dev, species, n, num_elements)
    _launch(dev, nv.load_library().mace_species_group, species.data_ptr(), n, num_elements, order.data_ptr(),
            offsets.data_ptr(), ptr, nbytes)
    return SpeciesGroups(order, offsets)


def _embedding(table, species, scale, out):
    dev = _cuda("table", table)
    if _index("species", species) != dev:
        raise ValueError(f"species is on {species.device}, expected cuda:{dev}")
    code = _dtype("table", table.dtype)
    g, _, c, ts, _ = _rows("table", table)
    if table.dim() != 2 or not 1 <= g <= MAX_INDEX:
        raise ValueError(f"table must be (num_elements, C) with 1..{MAX_INDEX} rows, got {tuple(table.shape)}")
    n = species.shape[0]
    out = _out(out, (n, c), table, dev)
    _launch(dev, nv.load_library().mace_species_embed, code, table.data_ptr(), ts, g, c, species.data_ptr(), n, scale,
            out.data_ptr(), max(out.stride(0), c))
    return out


def species_embedding(table: torch.Tensor, species: torch.Tensor, *, scale: float = 1.0,
                      groups: SpeciesGroups | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``scale * table[species]`` (N, C); zero rows for padding.

    When ``table`` requires a gradient, its backward sums over ``groups``
    (made from ``species`` when not given).
    """
    if torch.is_grad_enabled() and table.requires_grad:
        if out is not None:
            raise ValueError("out= cannot take part in autograd")
        _cuda("table", table)
        return _EmbeddingFn.apply(table, species, scale, groups)
    return _embedding(table, species, scale, out)


def species_embedding_grad(grad: torch.Tensor, groups: SpeciesGroups, *, scale: float = 1.0) -> torch.Tensor:
    """Table gradient ``scale * sum of grad over each group`` (num_elements, C)."""
    dev = _cuda("grad", grad)
    code = _dtype("grad", grad.dtype)
    n, _, c, gs, _ = _rows("grad", grad)
    if grad.dim() != 2:
        raise ValueError(f"grad must be (N, C), got {tuple(grad.shape)}")
    g, order, offsets = _groups(groups, n, dev)
    out = grad.new_empty((g, c))
    ws, ptr, nbytes = _workspace("mace_species_embed_grad_workspace", dev, grad, n, g, c)
    _launch(dev, nv.load_library().mace_species_embed_grad, code, grad.data_ptr(), gs, order, offsets, n, g, c, scale,
            out.data_ptr(), ptr, nbytes)
    return out


def _linear(x, weight, groups, alpha, transpose, out):
    dev = _cuda("x", x)
    code = _dtype("x", x.dtype)
    n, d, k, sn, sm = _rows("x", x)
    g, order, offsets = _groups(groups, n, dev)
    _on("weight", weight, dev)
    if weight.dim() != 3 or not weight.is_contiguous():
        raise ValueError(f"weight must be a contiguous (num_elements, K, M) tensor, got {tuple(weight.shape)} "
                         f"with strides {weight.stride()}")
    wg, k_in, k_out = weight.shape
    if wg != g:
        raise ValueError(f"weight has {wg} elements, the grouping {g}")
    _map_limits(n, d, g)
    _same_dtype("weight", weight, x)
    if transpose:
        k_in, k_out = k_out, k_in
    if k != k_in:
        raise ValueError(f"x has {k} channels, the weight takes {k_in}")
    shape = (n, d, k_out) if x.dim() == 3 else (n, k_out)
    if out is None:
        y = x.new_empty(shape)
        yn, ym = d * k_out, k_out
    else:
        y = _out(out, shape, x, dev)
        yn, ym = y.stride()[0], y.stride()[1] if d > 1 else k_out
    _launch(dev, nv.load_library().mace_species_linear, code, x.data_ptr(), sn, sm, weight.data_ptr(), transpose, g,
            k_in, k_out, order, offsets, n, d, alpha, y.data_ptr(), yn, ym)
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

    float32 products keep fp32 accuracy, here and in the gradients; infinities
    and NaN enter the results as they enter fp32 sums.
    """
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        if out is not None or transpose:
            raise ValueError("out= and transpose= cannot take part in autograd")
        _cuda("x", x), _cuda("weight", weight)
        return _LinearFn.apply(x, weight, groups.order, groups.offsets, alpha, checkpoint)
    return _linear(x, weight, groups, alpha, transpose, out)


def species_linear_grad_weight(x: torch.Tensor | RowCheckpoint, grad: torch.Tensor, groups: SpeciesGroups, *,
                               alpha: float = 1.0) -> torch.Tensor:
    """Weight gradient (num_elements, K, M) from the rows x, or from their 8-bit checkpoint."""
    dev = _cuda("grad", grad)
    code = _dtype("grad", grad.dtype)
    n, d, m, gn, gm = _rows("grad", grad)
    scale = None
    if isinstance(x, RowCheckpoint):
        x, scale = _checkpoint(x)
        scale = scale.data_ptr()
        _on("x.q", x, dev)
    else:
        _on("x", x, dev)
        _same_dtype("x", x, grad)
    xn, xd, k, sn, sm = _rows("x", x)
    if xn != n or xd != d:
        raise ValueError(f"x rows {tuple(x.shape)} do not match grad rows {tuple(grad.shape)}")
    g, order, offsets = _groups(groups, n, dev)
    _map_limits(n, d, g)
    dw = grad.new_empty((g, k, m))
    ws, ptr, nbytes = _workspace("mace_species_linear_wgrad_workspace", dev, grad, n, d, g, k, m)
    _launch(dev, nv.load_library().mace_species_linear_wgrad, code, x.data_ptr(), sn, sm, scale, grad.data_ptr(), gn,
            gm, g, k, m, order, offsets, n, d, alpha, dw.data_ptr(), ptr, nbytes)
    return dw


def species_linear_grad(x: torch.Tensor | RowCheckpoint, grad: torch.Tensor, weight: torch.Tensor,
                        groups: SpeciesGroups, *, alpha: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """Input and weight gradients of ``species_linear`` for the output gradient ``grad``."""
    return (_linear(grad, weight, groups, alpha, True, None),
            species_linear_grad_weight(x, grad, groups, alpha=alpha))


def _checkpoint(ck: RowCheckpoint) -> tuple[torch.Tensor, torch.Tensor]:
    q, scale = ck
    dev = _cuda("q", q)
    _on("scale", scale, dev)
    if q.dtype != torch.int8 or not q.is_contiguous() or q.dim() not in (2, 3):
        raise ValueError(f"q must be contiguous int8 (N, d, C) or (N, C), got {q.dtype} {tuple(q.shape)}")
    want = (*q.shape[:-1], -(-q.shape[-1] // CHECKPOINT_BLOCK))
    if scale.dtype != torch.float32 or not scale.is_contiguous() or scale.shape != want:
        raise ValueError(f"scale must be contiguous float32 {want}, got {scale.dtype} {tuple(scale.shape)}")
    return q, scale


def checkpoint_rows(x: torch.Tensor) -> RowCheckpoint:
    """x (N, d, C) or (N, C) in 8 bits: per row and block of 128 channels
    ``scale = max |x| * (1 / 127)``, ``q = round(x / scale)`` (half to even), in fp32.

    The error of a value is at most half a scale.  A block that holds an
    infinity or NaN is restored as NaN.
    """
    dev = _cuda("x", x)
    code = _dtype("x", x.dtype)
    n, d, c, sn, sm = _rows("x", x)
    q = x.new_empty(x.shape, dtype=torch.int8)
    scale = x.new_empty((*x.shape[:-1], -(-c // CHECKPOINT_BLOCK)), dtype=torch.float32)
    _launch(dev, nv.load_library().mace_rows_checkpoint, code, x.data_ptr(), sn, sm, n, d, c, q.data_ptr(),
            scale.data_ptr())
    return RowCheckpoint(q, scale)


def restore_rows(checkpoint: RowCheckpoint, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values ``q * scale`` an 8-bit checkpoint stands for, rounded to ``dtype``."""
    q, scale = _checkpoint(checkpoint)
    code = _dtype("dtype", dtype)
    n, d, c, _, _ = _rows("q", q)
    x = q.new_empty(q.shape, dtype=dtype)
    _launch(q.get_device(), nv.load_library().mace_rows_restore, code, q.data_ptr(), scale.data_ptr(), n, d, c,
            x.data_ptr())
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
        else:
            g, _, _ = _groups(groups, species.shape[0], table.get_device())
            if g != table.shape[0]:
                raise ValueError(f"the grouping has {g} elements, the table {table.shape[0]}")
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
