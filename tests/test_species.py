"""Species operators without a GPU: refusals of the Python entry points and of
the C ABI (host-side argument checks only, no launch)."""

import ctypes as C

import pytest
import torch

import mace_mlx_b200
from mace_mlx_b200 import native as nv
from mace_mlx_b200 import species as sp


def test_operators_are_public():
    for name in sp.__all__:
        assert hasattr(sp, name)
    assert mace_mlx_b200.species is sp


def test_cpu_tensors_are_refused():
    z = torch.zeros(4, dtype=torch.int32)
    groups = sp.SpeciesGroups(z, torch.zeros(2, dtype=torch.int32))
    x, w = torch.zeros(4, 1, 8), torch.zeros(1, 8, 8)
    for call in (lambda: sp.group_species(z, 1), lambda: sp.species_embedding(w[0], z),
                 lambda: sp.species_embedding_grad(x[:, 0], groups), lambda: sp.species_linear(x, w, groups),
                 lambda: sp.species_linear_grad(x, x, w, groups), lambda: sp.species_linear_grad_weight(x, x, groups),
                 lambda: sp.checkpoint_rows(x),
                 lambda: sp.restore_rows(sp.RowCheckpoint(x.to(torch.int8), torch.zeros(4, 1, 1)))):
        with pytest.raises(ValueError, match="no CPU path"):
            call()


def test_c_entries_check_their_arguments():
    lib = nv.load_library()
    need = C.c_int64(-1)
    one = C.c_void_p(16)  # never dereferenced: every call below is refused on the host
    assert lib.mace_species_group_workspace(1000, 89, C.byref(need)) == nv.MACE_OK and need.value == 0  # one CTA
    assert lib.mace_species_group_workspace(100000, 89, C.byref(need)) == nv.MACE_OK and need.value > 0
    assert lib.mace_species_group_workspace(-1, 89, C.byref(need)) == nv.MACE_ERR_BAD_ARG
    assert lib.mace_species_group_workspace(1, 0, C.byref(need)) == nv.MACE_ERR_BAD_ARG
    assert lib.mace_species_group_workspace(1, nv.SPECIES_MAX_INDEX + 1, C.byref(need)) == nv.MACE_ERR_BAD_ARG
    assert lib.mace_species_group_workspace(2**31, 1, C.byref(need)) == nv.MACE_ERR_BAD_ARG
    assert lib.mace_species_group_workspace(1, 1, None) == nv.MACE_ERR_BAD_ARG
    assert lib.mace_species_group(one, 5, 2, one, None, one, 1 << 20, None) == nv.MACE_ERR_BAD_ARG
    assert lib.mace_species_group(one, 100000, 2, one, one, one, 3, None) == nv.MACE_ERR_BAD_ARG
    assert "workspace" in nv.last_error(lib)
    assert lib.mace_species_embed(2, one, 8, 1, 8, one, 1, 1.0, one, 8, None) == nv.MACE_ERR_BAD_ARG
    assert lib.mace_species_embed(0, one, 8, 1, 8, one, 1, 1.0, one, 7, None) == nv.MACE_ERR_BAD_ARG
    assert lib.mace_species_embed(0, None, 8, 1, 8, one, 1, 1.0, one, 8, None) == nv.MACE_ERR_BAD_ARG
    assert lib.mace_species_embed_grad_workspace(1, 1, 0, C.byref(need)) == nv.MACE_ERR_BAD_ARG
    assert lib.mace_species_embed_grad(0, None, 8, one, one, 4, 1, 8, 1.0, one, one, 1 << 20, None) == nv.MACE_ERR_BAD_ARG
    lin = (0, one, 8, 8, one, 0, 1, 8, 8, one, one, 4, 1, 1.0, one, 8, 8, None)
    for at, value in ((0, 7), (1, None), (4, None), (6, 0), (6, nv.SPECIES_MAX_GROUPS + 1), (7, 0), (8, 0), (9, None),
                      (10, None), (11, -1), (12, 0), (12, 5000), (14, None), (2, -1)):
        args = list(lin)
        args[at] = value
        assert lib.mace_species_linear(*args) == nv.MACE_ERR_BAD_ARG, at
    wg = (0, one, 8, 8, None, one, 8, 8, 1, 8, 8, one, one, 4, 1, 1.0, one, one, 1 << 30, None)
    for at, value in ((0, 7), (1, None), (5, None), (8, 0), (9, 0), (10, 0), (11, None), (12, None), (13, -1), (14, 0),
                      (16, None), (3, -1)):
        args = list(wg)
        args[at] = value
        assert lib.mace_species_linear_wgrad(*args) == nv.MACE_ERR_BAD_ARG, at
    assert lib.mace_species_linear_wgrad_workspace(-1, 1, 1, 1, 1, C.byref(need)) == nv.MACE_ERR_BAD_ARG
    assert lib.mace_rows_checkpoint(0, None, 8, 8, 1, 1, 8, one, one, None) == nv.MACE_ERR_BAD_ARG
    assert lib.mace_rows_checkpoint(3, one, 8, 8, 1, 1, 8, one, one, None) == nv.MACE_ERR_BAD_ARG
    assert lib.mace_rows_restore(0, one, None, 1, 1, 8, one, None) == nv.MACE_ERR_BAD_ARG
    assert lib.mace_rows_restore(0, one, one, 1, 0, 8, one, None) == nv.MACE_ERR_BAD_ARG
    assert lib.mace_species_error_flag(None) == nv.MACE_ERR_BAD_ARG


def test_c_entries_refuse_addresses_off_their_values():
    lib = nv.load_library()
    one, odd, half = C.c_void_p(32), C.c_void_p(33), C.c_void_p(34)  # never dereferenced

    def refused(f, args, *at):
        for k in at:
            for address in (odd, half) if k >= 0 else (odd,):
                call = list(args)
                call[abs(k)] = address
                assert f(*call) == nv.MACE_ERR_BAD_ARG and "values' size" in nv.last_error(lib), (f, k)

    # (0: fp32; a negative place may be any multiple of two)
    refused(lib.mace_species_group, (one, 5, 2, one, one, None, 0, None), 0, 3, 4)
    refused(lib.mace_species_embed, (0, one, 8, 1, 8, one, 1, 1.0, one, 8, None), 1, 5, 8)
    refused(lib.mace_species_embed, (1, one, 8, 1, 8, one, 1, 1.0, one, 8, None), -1, 5, -8)
    refused(lib.mace_species_embed_grad, (0, one, 8, one, one, 4, 1, 8, 1.0, one, one, 1 << 20, None), 1, 3, 4, 9, 10)
    refused(lib.mace_species_linear, (0, one, 8, 8, one, 0, 1, 8, 8, one, one, 4, 1, 1.0, one, 8, 8, None), 1, 4, 9, 10, 14)
    refused(lib.mace_species_linear, (1, one, 8, 8, one, 0, 1, 8, 8, one, one, 4, 1, 1.0, one, 8, 8, None), -1, -4, -14)
    refused(lib.mace_species_linear_wgrad, (0, one, 8, 8, None, one, 8, 8, 1, 8, 8, one, one, 4, 1, 1.0, one, one, 1 << 30,
                                            None), 1, 4, 5, 11, 12, 16)
    refused(lib.mace_rows_checkpoint, (0, one, 8, 8, 1, 1, 8, one, one, None), 1, 8)
    refused(lib.mace_rows_restore, (0, one, one, 1, 1, 8, one, None), 2, 6)


def test_c_entries_refuse_workspaces_off_their_alignment():
    """Every kernel that reads its workspace in 16-byte pieces (the weight gradient's is held to 32)."""
    lib = nv.load_library()
    one, size = C.c_void_p(32), 1 << 20  # never dereferenced
    # a list of one row leaves one share with partial rows: the smallest call that has a workspace
    grad = [0, one, 8, one, one, 1, 1, 8, 1.0, one, None, size, None]
    group = [one, 100000, 2, one, one, None, size, None]
    wgrad = [0, one, 8, 8, None, one, 8, 8, 1, 8, 8, one, one, 4, 1, 1.0, one, None, 1 << 30, None]
    for f, args, at, offsets in ((lib.mace_species_embed_grad, grad, 10, (4, 8, 12)),
                                 (lib.mace_species_group, group, 5, (4, 8, 12)),
                                 (lib.mace_species_linear_wgrad, wgrad, 17, (4, 8, 16))):
        for offset in offsets:
            call = list(args)
            call[at] = C.c_void_p(64 + offset)
            assert f(*call) == nv.MACE_ERR_BAD_ARG and "aligned" in nv.last_error(lib), (f, offset)


def test_kernels_read_their_inputs_by_plain_loads():
    """A kernel of these operators may start while the one before it still writes its inputs, so none goes through the
    read-only path, which is for data that nothing writes while a kernel lives."""
    from pathlib import Path

    sources = sorted((Path(mace_mlx_b200.__file__).parent / "csrc").glob("species*.cu*"))
    assert len(sources) == 5
    for path in sources:
        text = path.read_text()
        for form in ("__ldg(", "global.nc", "__restrict__"):
            assert form not in text, (path.name, form)


def test_weight_gradient_workspace_follows_its_shares():
    """Two partial tiles a share and none for one share, however many groups there are."""
    lib, need = nv.load_library(), C.c_int64()

    def bytes_of(n, d, g, k, m):
        assert lib.mace_species_linear_wgrad_workspace(n, d, g, k, m, C.byref(need)) == nv.MACE_OK
        return need.value

    for g, k, m in ((89, 4096, 4096), (512, 2048, 2048), (1, 32768, 32768)):  # a tile to every SM: one share
        assert bytes_of(10_000, 3, g, k, m) <= 4 * g
    tile = 4 * 128 * 128
    for n, g, k, m in ((1_000_000, 512, 512, 512), (1000, 4, 128, 128), (100, 300, 128, 128), (5, 512, 300, 257)):
        tiles = -(-k // 128) * -(-m // 128)
        units = n // 64 + 1 + min(g, n)
        assert bytes_of(n, 1, g, k, m) <= 4 * g + tiles * 2 * min(units, -(-148 // tiles)) * tile
