"""Normalisation operators of training, beside the species operators, for
programs that train parts of MACE's form on the GPU.

* ``layer_norm``       -- layer norm of feature rows, with the SiLU that follows
  it in the radial MLPs of the non-linear interaction block
* ``layer_norm_grad``  -- its input and parameter gradients
* ``grad_norm``        -- the 2-norm of a model's gradients taken as one vector
* ``clip_grads``       -- the same, and the gradients scaled down to a largest norm

``layer_norm`` takes part in autograd when an argument requires a gradient
(once differentiable, in reverse mode: a tensor with a forward-mode tangent is
refused).  It keeps x for its backward, and no statistics: the backward makes
them again from x.

Every call runs hand-written kernels of ``libmace_b200`` on the current stream
of the tensors' device, allocates only its results and workspace through
torch, and neither synchronises nor reads device values, so it can be captured
into a CUDA graph (a backward, as torch has it, while no eager graph of the
same leaves lives).  Tensors last used on another stream need the caller's
``wait_stream``/``record_stream``, as for torch's own operators.

Reference: Linear -> LayerNorm -> SiLU stacks ``mace_mlx/radial.py:344-357``;
the reference has no training path.
"""

from __future__ import annotations

import ctypes as C
import functools
import math
import operator
from array import array
from collections.abc import Iterable, Sequence

import torch
from torch.autograd import forward_ad

from . import native as nv
from .species import _DTYPES, _cuda, _dtype, _launch, _on, _workspace

MAX_CHANNELS = nv.LAYER_NORM_MAX_CHANNELS
_ACTIVATIONS = {None: nv.ACT_NONE, "silu": nv.ACT_SILU}

__all__ = ["layer_norm", "layer_norm_grad", "grad_norm", "clip_grads"]

# Small calls are bound by the host.  The library reads the tensor objects itself through DLPack's C interface (a forward
# of 1000 rows 7.5 us a call, 9.3 attribute by attribute, its gradients 11.4 and 14.3); what that interface has not, and
# what is to be refused, is looked at here.
_reader = nv.dlpack_reader(torch.Tensor)
_reading = functools.cache(nv.load_reading)


# ---------------------------------------------------------------- layer norm
def _rows(name: str, t: torch.Tensor) -> tuple[int, int, int]:
    """(rows, C, row stride) of (..., C) whose leading dimensions lie one row stride apart."""
    shape = t.shape
    if len(shape) != 2:
        if not shape:
            raise ValueError(f"{name} must be (..., C), got a scalar")
        try:
            t = t.view(math.prod(shape[:-1]), shape[-1])
        except RuntimeError:
            raise ValueError(f"{name}: rows must lie at one stride, got shape {tuple(shape)} with strides "
                             f"{t.stride()}") from None
    n, c = t.shape
    if not 1 <= c <= MAX_CHANNELS or n >= 2**31:
        raise ValueError(f"{name}: need 1..{MAX_CHANNELS} channels and fewer than 2**31 rows, got {tuple(shape)}")
    sn, sc = t.stride()
    if sc != 1 and c > 1:
        raise ValueError(f"{name}: channels must be contiguous (stride 1), got strides {t.stride()}")
    return n, c, sn


def _params(weight, bias, dev: int, c: int, dtype: torch.dtype) -> tuple[int, int | None, int | None]:
    """(type code, pointers of weight and bias): C contiguous values, both of x's type or both float32."""
    kind = None
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        _on(name, t, dev)
        if t.numel() != c or t.dim() != 1 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous ({c},) tensor, got {tuple(t.shape)} with strides {t.stride()}")
        if kind is None:
            kind = t.dtype
            if kind is not dtype and kind is not torch.float32:
                raise ValueError(f"{name} is {kind}, expected {dtype} or float32")
        elif t.dtype is not kind:
            raise ValueError(f"weight is {kind}, bias {t.dtype}: they must be of one type")
        if not t.data_ptr():  # (null stands for no parameter in the C entries)
            raise ValueError(f"{name} has no memory of its own (a wrapper of other tensors?)")
    return (_DTYPES[dtype if kind is None else kind], None if weight is None else weight.data_ptr(),
            None if bias is None else bias.data_ptr())


def _written(name: str, t: torch.Tensor) -> None:
    """Refuses to write, unseen by autograd, to a tensor that it follows."""
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, and what is written to it here has none: pass a tensor that needs "
                         "none (a parameter's .grad, a detached one), or call under torch.no_grad()")


def _like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _activation(activation: str | None) -> int:
    code = _ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"activation must be None or 'silu', got {activation!r}")
    return code


def _eps(eps: float) -> float:
    if not 0.0 <= eps < 3e38:
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    return eps


def _read_rows(x, grad, weight, bias) -> nv.NormRows | None:
    """The operands as the library takes them; None where they have to be looked at here."""
    if _reader is None or forward_ad._current_level >= 0:
        return None
    rows = nv.NormRows()
    try:
        rc = _reading("mace_norm_rows_read")(_reader, id(x), None if grad is None else id(grad),
                                             None if weight is None else id(weight), None if bias is None else id(bias),
                                             C.byref(rows))
    except Exception:  # noqa: BLE001 (of a type, or a layout, that DLPack has not)
        return None
    return rows if rc == nv.MACE_OK else None


def _operands(x, grad, weight, bias) -> nv.NormRows:
    rows = _read_rows(x, grad, weight, bias)
    if rows is not None:
        return rows
    dev = _cuda("x", x)
    rows = nv.NormRows(dtype=_dtype("x", x.dtype), device=dev, x=x.data_ptr())
    rows.n, rows.C, rows.x_stride = _rows("x", x)
    if grad is not None:
        _on("grad", grad, dev)
        if grad.dtype != x.dtype or grad.shape != x.shape:
            raise ValueError(f"grad must be {x.dtype} {tuple(x.shape)}, got {grad.dtype} {tuple(grad.shape)}")
        _, _, rows.dy_stride = _rows("grad", grad)
        rows.dy = grad.data_ptr()
    rows.param_dtype, rows.weight, rows.bias = _params(weight, bias, dev, rows.C, x.dtype)
    return rows


def _layer_norm(x, weight, bias, eps, activation, out):
    rows = _operands(x, None, weight, bias)
    act = _activation(activation)
    if out is None:
        y = _like(x)
        _launch(rows.device, nv.load_library().mace_norm_rows_forward, C.byref(rows), _eps(eps), act, y.data_ptr())
        return y
    _on("out", out, rows.device)
    _written("out", out)
    if out.dtype != x.dtype or out.shape != x.shape:
        raise ValueError(f"out must be {x.dtype} {tuple(x.shape)}, got {out.dtype} {tuple(out.shape)}")
    n, c, stride = _rows("out", out)
    if n > 1 and stride < c:
        raise ValueError(f"out rows overlap (strides {out.stride()})")
    _launch(rows.device, nv.load_library().mace_layer_norm, rows.dtype, rows.x, rows.x_stride, rows.param_dtype, rows.weight,
            rows.bias, n, c, _eps(eps), act, out.data_ptr(), stride)
    torch.autograd.graph.increment_version(out)
    return out


def _layer_norm_grad(x, grad, weight, bias, eps, activation, want_x, want_w, want_b):
    rows = _operands(x, grad, weight, bias)
    act = _activation(activation)
    dx = _like(x) if want_x else None
    dw = _like(weight) if want_w else None
    db = _like(bias) if want_b else None
    ws, ptr, nbytes = None, None, 0
    if want_w or want_b:
        ws, ptr, nbytes = _workspace("mace_layer_norm_grad_workspace", rows.device, x, rows.n, rows.C)
    _launch(rows.device, nv.load_library().mace_norm_rows_backward, C.byref(rows), _eps(eps), act,
            dx.data_ptr() if want_x else None, dw.data_ptr() if want_w else None, db.data_ptr() if want_b else None, ptr, nbytes)
    return dx, dw, db


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
               eps: float = 1e-5, activation: str | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``f(weight * (x - mean) / sqrt(var + eps) + bias)`` over the last dimension, of up to 8192 channels.

    ``activation`` is None (f the identity) or ``"silu"``.  x is float32 or
    bfloat16, (..., C) with contiguous channels and rows at one stride, so a
    slot of a node-feature table is passed in place; so may ``out``, which must
    not overlap x, weight or bias.  weight and bias (C,), either or both, are of
    x's type or float32; without them they are ones and zeros.

    Statistics and products are fp32, rounded once to x's type.  Sums are taken
    of x minus one of the row's first values: an offset common to a row costs no
    accuracy, such a value k standard deviations off costs k units in the last
    place.  Deviations from the mean are squared in fp32: rows whose values pass
    1e18 lose them, and with ``eps`` 0 rows whose deviations all stay below 1e-18.
    SiLU's exponential and reciprocal are approximate: its sigmoid is off by about
    2 + 1.2 |z| units of fp32's last place.
    """
    _cuda("x", x)
    if torch.is_grad_enabled() and (x.requires_grad or _requires_grad("weight", weight) or _requires_grad("bias", bias)):
        if out is not None:
            raise ValueError("out= cannot take part in autograd")
        for name, t in (("weight", weight), ("bias", bias)):
            if t is not None:
                _cuda(name, t)
        return _LayerNormFn.apply(x, weight, bias, eps, activation)
    return _layer_norm(x, weight, bias, eps, activation, out)


def _requires_grad(name: str, t: torch.Tensor | None) -> bool:
    if t is None:
        return False
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    return t.requires_grad


def layer_norm_grad(x: torch.Tensor, grad: torch.Tensor, weight: torch.Tensor | None = None,
                    bias: torch.Tensor | None = None, *, eps: float = 1e-5, activation: str | None = None
                    ) -> tuple[torch.Tensor, torch.Tensor | None, torch.Tensor | None]:
    """Gradients of ``layer_norm`` at x, weight and bias for the output gradient ``grad``.

    They have no graph, whatever the arguments require.  Those of weight and bias
    have their type (None without them); their sums over the rows are fp32, in an
    order that depends on the sizes, the types and the addresses modulo 16 alone,
    so equal calls give equal bits.
    """
    return _layer_norm_grad(x, grad, weight, bias, eps, activation, True, weight is not None, bias is not None)


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, activation):
        ctx.save_for_backward(x, weight, bias)
        ctx.more = eps, activation
        return _layer_norm(x, weight, bias, eps, activation, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, weight, bias = ctx.saved_tensors
        if grad.dim() != 2 or grad.stride(-1) != 1:  # sums hand back expanded gradients, others any order
            grad = grad.contiguous()
        return (*_layer_norm_grad(x, grad, weight, bias, *ctx.more, *ctx.needs_input_grad[:3]), None, None)


# ----------------------------------------------------------- gradient norms
def _dense(t: torch.Tensor) -> bool:
    """Whether the values fill their memory without gaps or repeats, in whatever order of the dimensions."""
    if t.layout is not torch.strided:
        return False
    if t.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != expected:
            return False
        expected *= size
    return True


# (153 tensors: 10 us through DLPack, 41 by these, which take no Python frame each)
_requires = operator.attrgetter("requires_grad")
_device, _pointer, _numel, _contiguous = (getattr(torch.Tensor, f) for f in
                                          ("get_device", "data_ptr", "numel", "is_contiguous"))


_ZERO_POINTERS, _ZERO_SIZES, _ZERO_CODES = array("Q", [0]), array("q", [0]), array("i", [0])
_list_item = nv.list_reader()


def _objects(items: list) -> tuple[array, bool]:
    """Addresses of a list's objects, and whether None is among them."""
    objects = _ZERO_POINTERS * len(items)
    return objects, bool(_reading("mace_list_items")(_list_item, id(items), len(items), id(None), objects.buffer_info()[0]))


def _flat(name: str, tensors: Sequence[torch.Tensor], dev: int, objects: array | None = None, refuse=None
          ) -> tuple[array, array, array, bool]:
    """Pointers, sizes and type codes of dense tensors on device ``dev``, and whether all are contiguous.

    ``objects`` are their addresses, where the caller has them; ``refuse`` looks at the tensors where, under grad mode,
    one requires a gradient.
    """
    if _reader is not None and forward_ad._current_level < 0:
        n = len(tensors)
        if objects is None:
            objects, _ = _objects(tensors)
        ptrs, sizes, codes = _ZERO_POINTERS * n, _ZERO_SIZES * n, _ZERO_CODES * n
        try:
            rc = _reading("mace_tensor_list")(_reader, n, objects.buffer_info()[0], dev, ptrs.buffer_info()[0], sizes.buffer_info()[0],
                                              codes.buffer_info()[0])
        except Exception:  # noqa: BLE001 (of a type, or a layout, that DLPack has not: told below)
            rc = nv.MACE_ERR_BAD_ARG
        if rc == nv.MACE_OK:
            if refuse is not None and torch.is_grad_enabled() and any(map(_requires, tensors)):
                refuse(name, tensors)
            return ptrs, sizes, codes, True
    try:
        elsewhere = set(map(_device, tensors)) - {dev}
    except TypeError:  # (no tensor)
        elsewhere = True
    if elsewhere or forward_ad._current_level >= 0:
        for i, t in enumerate(tensors):
            _on(f"{name}[{i}]", t, dev)
    try:
        contiguous = all(map(_contiguous, tensors))
    except RuntimeError:  # (not strided)
        contiguous = False
    if not contiguous:
        for i, t in enumerate(tensors):
            if not _dense(t):
                raise ValueError(f"{name}[{i}] has gaps or repeated values (strides {t.stride()}); use .contiguous()"
                                 if t.layout is torch.strided else f"{name}[{i}] is not strided, got {t.layout}")
    if refuse is not None and torch.is_grad_enabled() and any(map(_requires, tensors)):
        refuse(name, tensors)
    kinds = {dtype: _dtype(name, dtype) for dtype in {t.dtype for t in tensors}}
    codes = array("i", kinds.values()) * len(tensors) if len(kinds) == 1 else array("i", [kinds[t.dtype] for t in tensors])
    return array("Q", map(_pointer, tensors)), array("q", map(_numel, tensors)), codes, contiguous


def _grads(grads: Iterable[torch.Tensor | None]) -> tuple[list[torch.Tensor], array]:
    """The gradients without the entries that are None, and the objects' addresses."""
    if isinstance(grads, torch.Tensor):
        raise TypeError("grads must be a sequence of tensors, got one tensor")
    grads = list(grads)
    objects, gaps = _objects(grads)
    if gaps:
        grads = [g for g in grads if g is not None]
        objects, _ = _objects(grads)
    return grads, objects


def _written_to(name: str, tensors: Sequence[torch.Tensor]) -> None:
    for i, t in enumerate(tensors):
        _written(f"{name}[{i}]", t)


def _without_graph(name: str, grads: Sequence[torch.Tensor]) -> None:
    """Refuses gradients that have a graph themselves: what is made of them here would have none."""
    for i, g in enumerate(grads):
        if not g.is_leaf:
            raise ValueError(f"{name}[{i}] has a graph (create_graph=True?), which would end here without a word: detach it "
                             "or call under torch.no_grad(); a norm to differentiate is torch.linalg.vector_norm's")


def _norm_of(grads: list[torch.Tensor], dev: int, flat, fn, *more) -> torch.Tensor:
    ptrs, sizes, codes, _ = flat
    norm = (grads[0].new_empty((), dtype=torch.float32) if grads
            else torch.empty((), dtype=torch.float32, device=torch.device("cuda", dev)))
    # (the number of values tells few tensors from small ones)
    values = sum(sizes) if len(grads) <= nv.GRAD_FEW_TENSORS else 0
    ws, wptr, nbytes = _workspace("mace_grad_norm_workspace", dev, norm, len(grads), values)
    _launch(dev, fn, len(grads), ptrs.buffer_info()[0], sizes.buffer_info()[0], codes.buffer_info()[0], *more,
            norm.data_ptr(), wptr, nbytes)
    return norm


def grad_norm(grads: Iterable[torch.Tensor | None]) -> torch.Tensor:
    """The 2-norm of all gradients taken as one vector: a float32 scalar on their device.

    The gradients are float32 or bfloat16 (mixed as they come), on one device,
    without gaps in their memory; entries that are None (parameters without a
    gradient) are passed over.  Squares are summed in fp64.  The norm has no
    graph: leaves are taken by their values, and gradients with a graph of their
    own (``create_graph=True``) are refused under grad mode.
    """
    grads, objects = _grads(grads)
    dev = _cuda("grads[0]", grads[0]) if grads else torch.cuda.current_device()
    flat = _flat("grads", grads, dev, objects, _without_graph)
    return _norm_of(grads, dev, flat, nv.load_library().mace_grad_norm)


def clip_grads(grads: Iterable[torch.Tensor | None], max_norm: float, *,
               out: Sequence[torch.Tensor | None] | None = None) -> torch.Tensor:
    """Scales the gradients by ``min(1, max_norm / (norm + 1e-6))``, in place, and returns their ``grad_norm``.

    Gradients below the bound are left untouched, and nothing waits for the
    norm on the host.  With ``out`` (a tensor for every gradient, with as many
    values in the same order in memory, float32 or bfloat16) the results go there
    and the gradients stay, unless ``out`` holds the gradient itself.  No tensor
    that is written may overlap another one of the call, so none may be listed
    twice, and under grad mode none may require a gradient (pass the parameters'
    gradients, not the parameters), nor gradients have a graph of their own.

    A norm that is NaN makes every gradient NaN, and infinities among the
    gradients make the finite values zero and themselves NaN: test the norm where
    that can occur.  One of finite gradients that passes fp32's range is returned
    as infinity, and the gradients are scaled by it all the same, in fp64.
    """
    if isinstance(max_norm, torch.Tensor):
        raise TypeError("max_norm must be a number: a tensor's value would be waited for")
    max_norm = float(max_norm)
    if not 0.0 <= max_norm < math.inf:
        raise ValueError(f"max_norm must be finite and not negative, got {max_norm}")
    every = grads if out is None or isinstance(grads, torch.Tensor) else list(grads)
    grads, objects = _grads(every)
    dev = _cuda("grads[0]", grads[0]) if grads else torch.cuda.current_device()
    flat = _flat("grads", grads, dev, objects, _written_to if out is None else _without_graph)
    into, ptrs, codes = grads, flat[0], flat[2]
    if out is not None:
        if len(out) != len(every):
            raise ValueError(f"out has {len(out)} tensors, grads {len(every)}")
        into = list(out) if len(grads) == len(every) else [o for o, g in zip(out, every) if g is not None]
        ptrs, sizes, codes, contiguous = _flat("out", into, dev, None, _written_to)
        if sizes.tobytes() != flat[1].tobytes() or not (contiguous and flat[3]):
            for i, (g, o) in enumerate(zip(grads, into)):
                if o.numel() != g.numel() or o.stride() != g.stride() and not (o.is_contiguous() and g.is_contiguous()):
                    raise ValueError(f"out[{i}] must be {tuple(g.shape)} with strides {g.stride()}, got {tuple(o.shape)} "
                                     f"with strides {o.stride()}")
    norm = _norm_of(grads, dev, flat, nv.load_library().mace_grad_clip, ptrs.buffer_info()[0], codes.buffer_info()[0],
                    max_norm)
    torch.autograd.graph.increment_version(into)
    return norm
