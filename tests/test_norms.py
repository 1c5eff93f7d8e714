"""Normalisation operators without a GPU: refusals of the Python entry points and of
the C ABI (host-side argument checks only, no launch)."""

import ctypes as C
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import mace_mlx_b200
from mace_mlx_b200 import native as nv
from mace_mlx_b200 import norms


def test_operators_are_public():
    for name in norms.__all__:
        assert hasattr(norms, name)
    assert mace_mlx_b200.norms is norms


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 8), torch.ones(8)
    for call in (lambda: norms.layer_norm(x, w, w), lambda: norms.layer_norm(x.requires_grad_(), w),
                 lambda: norms.layer_norm_grad(x, x, w, w), lambda: norms.grad_norm([x]),
                 lambda: norms.clip_grads([x, w], 1.0), lambda: norms.clip_grads([None, x], 1.0, out=[None, x])):
        with pytest.raises(ValueError, match="no CPU path"):
            call()


def test_bounds_of_the_norm_are_checked_first():
    for bad in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="max_norm"):
            norms.clip_grads([torch.zeros(2)], bad)
    with pytest.raises(TypeError, match="max_norm"):
        norms.clip_grads([torch.zeros(2)], torch.ones(()))
    for call in (lambda: norms.grad_norm(torch.zeros(2)), lambda: norms.clip_grads(torch.zeros(2), 1.0),
                 lambda: norms.grad_norm([1.0])):
        with pytest.raises(TypeError):
            call()


@pytest.mark.parametrize("t,dense", [
    (torch.zeros(3, 4), True), (torch.zeros(3, 4).T, True), (torch.zeros(2, 3, 4).permute(1, 2, 0), True),
    (torch.zeros(3, 4)[:, :2], False), (torch.zeros(3, 4)[:2], True), (torch.zeros(3, 4)[::2], False),
    (torch.zeros(1).expand(5), False), (torch.zeros(4, 1).expand(4, 3), False), (torch.zeros(0, 4), True),
    (torch.zeros(()), True), (torch.zeros(3, 1, 4)[:, :, :1], False), (torch.zeros(5, 2)[:, 0], False),
    (torch.zeros(1, 9)[:, ::2][:, :1], True), (torch.zeros(3, 4).to_sparse(), False),
])  # fmt: skip
def test_dense_tensors_are_told_apart(t, dense):
    assert norms._dense(t) == dense


def test_c_entries_check_their_arguments():
    lib = nv.load_library()
    one, odd = C.c_void_p(32), C.c_void_p(33)  # never dereferenced: every call below is refused on the host

    def refused(f, args, changes, match=""):
        for at, value in changes:
            call = list(args)
            call[at] = value
            assert f(*call) == nv.MACE_ERR_BAD_ARG and match in nv.last_error(lib), (f, at, value)

    rows = (0, one, 8, 0, one, one, 4, 8, 1e-5, 0, one, 8, None)
    refused(lib.mace_layer_norm, rows, [
        (0, 2), (1, None), (2, -1), (3, 2), (6, -1), (6, 2**31), (7, 0), (7, nv.LAYER_NORM_MAX_CHANNELS + 1), (8, -1.0),
        (8, float("inf")), (8, float("nan")), (9, 2), (9, -1), (10, None), (11, 7)])
    refused(lib.mace_layer_norm, rows, [(1, odd), (4, odd), (5, odd), (10, odd)], "values' size")
    assert lib.mace_layer_norm(0, None, 8, 0, None, None, 0, 8, 1e-5, 0, None, 8, None) == nv.MACE_OK  # no rows

    need = C.c_int64(-1)
    assert lib.mace_layer_norm_grad_workspace(100_000, 128, C.byref(need)) == nv.MACE_OK and need.value > 0
    assert lib.mace_layer_norm_grad_workspace(1000, 128, C.byref(need)) == nv.MACE_OK and need.value == 0  # one cluster
    for args in ((-1, 8), (2**31, 8), (1, 0), (1, nv.LAYER_NORM_MAX_CHANNELS + 1)):
        assert lib.mace_layer_norm_grad_workspace(*args, C.byref(need)) == nv.MACE_ERR_BAD_ARG
    assert lib.mace_layer_norm_grad_workspace(1, 8, None) == nv.MACE_ERR_BAD_ARG
    grad = (0, one, 8, one, 8, 0, one, one, 4, 8, 1e-5, 0, one, 8, one, one, one, 1 << 20, None)
    refused(lib.mace_layer_norm_grad, grad, [(0, 7), (1, None), (2, -1), (3, None), (4, -1), (5, 7), (8, -1), (9, 0),
                                             (10, -1.0), (11, 5), (13, 7)])
    refused(lib.mace_layer_norm_grad, grad, [(k, odd) for k in (1, 3, 6, 7, 12, 14, 15)], "values' size")
    many = (*grad[:8], 100_000, *grad[9:])
    refused(lib.mace_layer_norm_grad, many, [(16, None), (16, C.c_void_p(40)), (17, 3)], "workspace")


def test_c_entries_check_lists_of_tensors():
    lib = nv.load_library()
    need = C.c_int64(-1)
    assert lib.mace_grad_norm_workspace(0, 0, C.byref(need)) == nv.MACE_OK and need.value == 0
    assert lib.mace_grad_norm_workspace(8, 1000, C.byref(need)) == nv.MACE_OK and need.value == 0  # one cluster
    assert lib.mace_grad_norm_workspace(8, 10**7, C.byref(need)) == nv.MACE_OK and need.value > 0
    assert lib.mace_grad_norm_workspace(5000, 5000, C.byref(need)) == nv.MACE_OK and need.value > 0
    for args in ((-1, 0), (0, -1)):
        assert lib.mace_grad_norm_workspace(*args, C.byref(need)) == nv.MACE_ERR_BAD_ARG
    assert lib.mace_grad_norm_workspace(1, 1, None) == nv.MACE_ERR_BAD_ARG
    one = C.c_void_p(4096)

    def call(ptrs, sizes, types, out=None, out_types=None, max_norm=1.0, norm=one, ws=one, nbytes=1 << 20):
        n = len(ptrs)
        a = ((C.c_void_p * n)(*ptrs), (C.c_int64 * n)(*sizes), (C.c_int32 * n)(*types))
        if out is None:
            rc = lib.mace_grad_norm(n, *a, norm, ws, nbytes, None)
        else:
            rc = lib.mace_grad_clip(n, *a, (C.c_void_p * n)(*out), (C.c_int32 * n)(*(out_types or types)), max_norm, norm,
                                    ws, nbytes, None)
        return rc, nv.last_error(lib)

    bad = [
        call([64], [-1], [0]), call([64], [8], [2]), call([None], [8], [0]), call([66], [8], [0]), call([65], [8], [1]),
        call([64], [8], [0], norm=None), call([64], [10**7], [0], ws=None), call([64], [10**7], [0], nbytes=8),
        call([64], [10**7], [0], ws=C.c_void_p(4)), call([64], [2**41], [0]),
        call([64], [8], [0], out=[64], max_norm=-1.0), call([64], [8], [0], out=[64], max_norm=float("inf")),
        call([64], [8], [0], out=[64], max_norm=float("nan")), call([64], [8], [0], out=[None]),
        call([64], [8], [0], out=[64], out_types=[1]), call([64], [8], [0], out=[63], out_types=[1]),
    ]
    assert [rc for rc, _ in bad] == [nv.MACE_ERR_BAD_ARG] * len(bad)
    # outputs over other tensors: one listed twice, a later one inside an earlier, an output that begins in its own
    # input, or reaches into another's input or output
    overlaps = [
        call([64, 64], [8, 8], [0, 0], out=[64, 64]), call([64, 80], [8, 2], [0, 0], out=[64, 80]),
        call([64], [8], [0], out=[68]), call([64], [8], [0], out=[92]),
        call([64, 256], [8, 8], [0, 0], out=[252, 512]), call([64, 256], [8, 8], [0, 0], out=[512, 528]),
        call([64, 256], [8, 8], [1, 1], out=[1024, 1040], out_types=[0, 1]),
        call([4096, 64, 256], [100, 4, 4], [0, 0, 0], out=[4096, 4492, 256]),
    ]
    for rc, text in overlaps:
        assert rc == nv.MACE_ERR_BAD_ARG and "overlaps" in text


def test_kernels_read_their_inputs_by_plain_loads():
    """As the species operators' kernels: one may start while the kernel before it still writes its inputs."""
    for name in ("layer_norm.cu", "layer_norm_grad.cu", "layer_norm.cuh", "grad_norm.cu"):
        text = (Path(mace_mlx_b200.__file__).parent / "csrc" / name).read_text()
        for form in ("__ldg(", "global.nc", "__restrict__"):
            assert form not in text, (name, form)


def test_workspace_follows_the_shares_of_the_rows():
    """At most a row of sums (2 C values in whole 16 bytes) for every 256 rows of a CTA, or for each CTA of a full GPU."""
    lib, need = nv.load_library(), C.c_int64()
    for n, c in ((0, 64), (1, 1), (1000, 128), (50_000_000, 64), (2**31 - 1, 8), (20_000, 2048), (5, 8192), (10**6, 8192)):
        assert lib.mace_layer_norm_grad_workspace(n, c, C.byref(need)) == nv.MACE_OK
        pitch = (2 * c + 3) // 4 * 16
        assert need.value % pitch == 0 and need.value // pitch <= min(n, n // 256 + 148 * 32)


def test_lists_of_objects_are_read_through_dlpack():
    """On tensors of the host: refused for their device, as are other objects (their reader's exception is raised)."""
    from array import array

    reader = nv.dlpack_reader(torch.Tensor)
    if reader is None:
        pytest.skip("this torch has no DLPack C exchange API")
    read = nv.load_reading("mace_tensor_list")

    def call(objects, device=0, reader=reader):
        n = len(objects)
        ids, out = array("Q", map(id, objects)), [array("Q", bytes(8 * n)), array("q", bytes(8 * n)), array("i", bytes(4 * n))]
        return read(reader, n, ids.buffer_info()[0], device, *(a.buffer_info()[0] for a in out))

    assert call([]) == nv.MACE_OK
    assert call([torch.zeros(3)]) == nv.MACE_ERR_BAD_ARG
    assert call([torch.zeros(3)], reader=None) == nv.MACE_ERR_BAD_ARG
    for other in (1.0, None, "x"):
        with pytest.raises(Exception):  # noqa: B017 (whatever the reader sets)
            call([other])
    assert nv.dlpack_reader(int) is None


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_struct_of_operands_matches_the_header(tmp_path):
    fields = [name for name, _ in nv.NormRows._fields_]
    prints = "".join(f'printf("%zu ", offsetof(mace_norm_rows, {f}));' for f in fields)
    include = Path(mace_mlx_b200.__file__).resolve().parents[1] / "include"
    (tmp_path / "l.c").write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"mace_b200.h\"\n"
                                  f'int main(void){{{prints}printf("%zu", sizeof(mace_norm_rows)); return 0;}}')
    subprocess.run(["gcc", f"-I{include}", str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    got = subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in got] == [*(getattr(nv.NormRows, f).offset for f in fields), C.sizeof(nv.NormRows)]


def test_struct_entries_check_their_arguments():
    lib = nv.load_library()
    rows = nv.NormRows(dtype=0, param_dtype=0, C=8, device=0, n=4, x_stride=8, dy_stride=8, x=32, dy=32)
    assert lib.mace_norm_rows_forward(None, 1e-5, 0, 32, None) == nv.MACE_ERR_BAD_ARG
    assert lib.mace_norm_rows_backward(None, 1e-5, 0, 32, None, None, None, 0, None) == nv.MACE_ERR_BAD_ARG
    assert lib.mace_norm_rows_forward(C.byref(rows), -1.0, 0, 32, None) == nv.MACE_ERR_BAD_ARG
    assert lib.mace_norm_rows_backward(C.byref(rows), 1e-5, 7, 32, None, None, None, 0, None) == nv.MACE_ERR_BAD_ARG
    if nv.dlpack_reader(torch.Tensor) is not None:
        read, x = nv.load_reading("mace_norm_rows_read"), torch.zeros(4, 8)
        for reader, obj in ((nv.dlpack_reader(torch.Tensor), x), (None, x)):  # (of the host; no reader)
            assert read(reader, id(obj), None, None, None, C.byref(rows)) == nv.MACE_ERR_BAD_ARG


class Elsewhere(torch.Tensor):
    """A tensor without memory of its own, as the wrappers of distributed tensors are."""

    @staticmethod
    def __new__(cls, *shape, dtype=torch.float32):
        return torch.Tensor._make_wrapper_subclass(cls, shape, dtype=dtype, device=torch.device("cuda", 0))

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError(func)


def test_parameters_without_memory_are_refused():
    """A null address stands for no weight in the C entries: that of a parameter must not get there."""
    for pair in ((Elsewhere(8), None), (None, Elsewhere(8)), (Elsewhere(8, dtype=torch.bfloat16),) * 2):
        with pytest.raises(ValueError, match="no memory"):
            norms._params(*pair, 0, 8, torch.bfloat16)


def test_the_reader_of_operands_refuses_null_addresses():
    class Tensor(C.Structure):
        _fields_ = [("data", C.c_void_p), ("device_type", C.c_int32), ("device_id", C.c_int32), ("ndim", C.c_int32),
                    ("code", C.c_uint8), ("bits", C.c_uint8), ("lanes", C.c_uint16), ("shape", C.POINTER(C.c_int64)),
                    ("strides", C.POINTER(C.c_int64)), ("byte_offset", C.c_uint64)]

    shapes = {1: (4, 8), 2: (4, 8), 3: (8,), 4: (8,), 5: (0, 8)}
    memory = {k: ((C.c_int64 * len(s))(*s), s) for k, s in shapes.items()}
    null = set()

    @C.CFUNCTYPE(C.c_int, C.c_void_p, C.c_void_p)
    def read(key, tensor):  # fp32 tensors on CUDA device 0, at addresses that nothing reads
        shape, sizes = memory[key]
        t = Tensor.from_address(tensor)
        t.data, t.device_type, t.device_id, t.ndim = None if key in null else 4096 * key, 2, 0, len(sizes)
        t.code, t.bits, t.lanes, t.shape, t.strides, t.byte_offset = 2, 32, 1, shape, None, 0
        return 0

    entry = nv.load_reading("mace_norm_rows_read")
    fn, rows = C.cast(read, C.c_void_p), nv.NormRows()
    assert entry(fn, 1, 2, 3, 4, C.byref(rows)) == nv.MACE_OK
    assert (rows.x, rows.dy, rows.weight, rows.bias) == (4096, 8192, 12288, 16384)
    for key in (1, 2, 3, 4):
        null.clear()
        null.add(key)
        assert entry(fn, 1, 2, 3, 4, C.byref(rows)) == nv.MACE_ERR_BAD_ARG, key
    null.clear()
    null.add(5)
    assert entry(fn, 5, 5, 3, 4, C.byref(rows)) == nv.MACE_OK  # (no rows have no memory)


@pytest.mark.parametrize("default", [torch.float32, torch.float64, torch.bfloat16])
def test_the_norm_of_nothing_is_fp32(default, monkeypatch):
    """Four bytes are written whatever the program's default type is."""
    empty, launched = torch.empty, []
    monkeypatch.setattr(torch, "empty", lambda *a, device=None, **k: empty(*a, **k))  # (here on the host)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(norms, "_workspace", lambda *a: (None, None, 0))
    monkeypatch.setattr(norms, "_launch", lambda *a: launched.append(a))
    before = torch.get_default_dtype()
    try:
        torch.set_default_dtype(default)
        for norm in (norms.grad_norm([]), norms.grad_norm([None]), norms.clip_grads([], 1.0), norms.clip_grads([None], 1.0)):
            assert norm.dtype == torch.float32
    finally:
        torch.set_default_dtype(before)
    assert len(launched) == 4


def test_results_over_operands_are_refused():
    """Rows that lie between each other without meeting are told from rows that meet (the calls that are taken, as slots
    of one table, run on the GPU)."""
    lib = nv.load_library()

    def forward(x, xs, y, ys, n=5, c=8, w=None, b=None, dtype=0, param=0):
        rc = lib.mace_layer_norm(dtype, x, xs, param, w, b, n, c, 1e-5, 0, y, ys, None)
        return rc == nv.MACE_ERR_BAD_ARG and "overlaps" in nv.last_error(lib)

    def backward(x, xs, dy, ds, dx, dxs, n=5, c=8, w=None, b=None):
        rc = lib.mace_layer_norm_grad(0, x, xs, dy, ds, 0, w, b, n, c, 1e-5, 0, dx, dxs, None, None, None, 0, None)
        return rc == nv.MACE_ERR_BAD_ARG and "overlaps" in nv.last_error(lib)

    at = 1 << 20
    size = 4 * 8  # of a row
    assert forward(at, 8, at, 8) and forward(at, 8, at + 4, 8) and forward(at + 4, 8, at, 8)
    assert forward(at, 8, at + 5 * size - 4, 8) and forward(at, 20, at + 28, 20) and forward(at, 20, at + 4 * 80 + 28, 20)
    assert forward(at + 3 * size, 0, at, 8) and forward(at, 8, at, 20) and forward(at, 8, at + 8, 20, n=1)
    assert forward(at, 12, at + 32, 8) and forward(at, 16, at + 32, 24)  # unlike strides: x meets the second row of y
    assert forward(at, 16, at + 16 * 6 - 2, 16, dtype=1) and forward(at, 16, at + 16, 16, c=9, dtype=1)
    assert forward(at, 8, at + (1 << 16), 8, w=at + (1 << 16) + 4 * size + 4) and forward(at, 8, at + 4096, 20, b=at + 4096 + 76)
    assert forward(at, 8, at + 4096, 8, w=at + 4096 - 4, dtype=1, param=0)
    other = at + (1 << 16)
    assert backward(at, 8, other, 8, at, 8) and backward(at, 8, other, 8, other + 16, 8) and backward(at, 0, other, 0, other - 64, 8)
    assert backward(at, 8, at, 8, other, 8, w=other) and backward(at, 8, at, 8, other, 8, b=other + 4 * size + 28)


def test_arrays_read_as_vectors_are_aligned():
    """A local array whose values go out as one word of 8 or 16 bytes is declared with that alignment: in memory, where a
    compiler may place it, the word would else be misaligned."""
    import re

    csrc, found = Path(mace_mlx_b200.__file__).parent / "csrc", 0
    for name in ("layer_norm.cu", "layer_norm_grad.cu", "layer_norm.cuh", "grad_norm.cu", "species.cuh"):
        text = (csrc / name).read_text()
        for use in re.finditer(r"reinterpret_cast<const (?:uint|float)([24])\*>\((\w+)\)", text):
            declared = list(re.finditer(rf"^\s*(alignas\((\d+)\) )?(?:T|bf16|float) {use[2]}\[\w+\];", text[:use.start()], re.M))
            if declared and text.count("\n", declared[-1].start(), use.start()) < 12:
                found += 1
                assert declared[-1][1] and int(declared[-1][2]) == 4 * int(use[1]), (name, use[0])
    assert found >= 3


def test_what_host_threads_share_is_atomic():
    """Statics of the C entries, which two host threads may call at once, are atomic (or constant)."""
    import re

    for name in ("layer_norm.cu", "layer_norm_grad.cu", "layer_norm.cuh", "grad_norm.cu", "tensor_list.cu"):
        text = (Path(mace_mlx_b200.__file__).parent / "csrc" / name).read_text()
        kinds = set(re.findall(r"^ +static (?!constexpr|__device__|const |inline)([\w:]+)[^;()]*[;=]", text, re.M))
        assert kinds <= {"DeviceFlags", "ClusterSizes"}, (name, kinds)


def test_a_lane_adds_256_rows_at_most_wherever_rows_start():
    """Rows that start anywhere can take twice the lanes of aligned ones (fp32 of 62 to 64 channels 16, bf16 of 122 to 128
    32), and a CTA then half the rows at once: the workspace holds the sums of as many more CTAs."""
    lib, need = nv.load_library(), C.c_int64()
    for c, lanes in ((16, 4), (62, 16), (64, 16), (122, 32), (128, 32), (256, 32), (300, 32)):
        for n in (5_000_000, 50_000_000):
            assert lib.mace_layer_norm_grad_workspace(n, c, C.byref(need)) == nv.MACE_OK
            shares = need.value // ((2 * c + 3) // 4 * 16)
            assert shares * 256 * (256 // lanes) >= n, (c, n)


def test_lists_are_read_as_they_stand():
    one, two = torch.zeros(1), torch.zeros(2)
    for items, gaps in (([], False), ([one], False), ([one, two, one], False), ([None], True), ([one, None, two], True), ([one] * 300, False)):
        objects, none = norms._objects(items)
        assert list(objects) == [id(item) for item in items] and none == gaps
    read, room, short = nv.load_reading("mace_list_items"), (C.c_void_p * 3)(), [one]
    with pytest.raises(IndexError):
        read(nv.list_reader(), id(short), 3, id(None), room)
