"""Normalisation operators on the GPU against their definitions in 64 bits.

Bounds (u = 2^-24, the unit roundoff of fp32; every step's rounding carried
through to first order, with whole numbers rounded up):

* forward, with R = max |x - x[0]| of a row: x - x[0] rounds by u R, its mean
  by 24 u R (8 values of a lane, then sums of at most 2^10 lanes), so a
  deviation from the mean is off by D = 28 u R; the sum of its squares rounds
  by 26 u, so rstd is off by D rstd + 18 u of itself and xhat by
  E = D rstd (1 + |xhat|) + 19 u |xhat|.
  z = w xhat + b is one fma: |w| E + u |z|.  SiLU has a slope below 1.1, and
  its sigmoid is off by (12 + 2.4 |z|) u of itself (exp within 2 + 1.17 |z|
  units, a sum, a quotient within 2 units, a product) or by 1e-36.
* backward: the slope of SiLU, f' = s (1 + z (1 - s)), is off by half of z's
  error (|f''| <= 1/2) and by (16 + 10 |z|) u; then dz, g = w dz, and the means of
  g and g xhat (26 u of the mean magnitude) enter dx = rstd (g - c1 - xhat c2)
  as they stand, with 4 u for its own three operations.
* a sum over rows adds at most 256 rows a lane, then warps, then shares: its
  rounding stays below (min(n, 512) + 16) u of the terms' magnitudes.
* those errors are random, so over a whole result of unit-scale inputs the
  relative error in the 2-norm also stays below 2^-19;
* a bf16 result adds half a unit in its last place, at most 2^-8 of it.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
F32, BF16 = torch.float32, torch.bfloat16
DTYPES = [F32, BF16]


@pytest.fixture(scope="module")
def nm():
    from mace_mlx_b200 import norms

    return norms


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0, dtype=F32):
    return torch.randn(shape, generator=gen(seed), device="cuda").to(dtype)


def inputs(n, c, dtype, param, seed=0):
    """x with channels of their own scale and offset, dy, weight and bias."""
    x = (randn(n, c, seed=seed) * (0.5 + randn(c, seed=seed + 1).abs()) + randn(c, seed=seed + 2)).to(dtype)
    return (x, randn(n, c, seed=seed + 3, dtype=dtype), (1.0 + 0.3 * randn(c, seed=seed + 4)).to(param),
            (0.3 * randn(c, seed=seed + 5)).to(param))


class Rows64:
    """The definition in 64 bits, and how far fp32 may be off."""

    def __init__(self, x, weight, bias, eps, silu):
        x = x.double()
        x = x - x[:, :1]  # (the mean of equal large ones would round in 64 bits too)
        self.n, self.c = x.shape
        one = torch.ones(self.c, dtype=torch.float64, device=x.device)
        self.w = one if weight is None else weight.double()
        b = 0 * one if bias is None else bias.double()
        mean = x.mean(1, keepdim=True)
        eps = float(torch.tensor(eps, dtype=F32))  # the kernel gets it in fp32
        self.rstd = 1.0 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + eps)
        self.xhat = (x - mean) * self.rstd
        self.D = 28 * U * x.abs().amax(1, keepdim=True) * self.rstd
        self.E = self.D * (1 + self.xhat.abs()) + 19 * U * self.xhat.abs()
        self.z = self.w * self.xhat + b
        self.E_z = self.w.abs() * self.E + U * self.z.abs()
        self.silu = silu
        self.sig = torch.sigmoid(self.z)

    def forward(self):
        if not self.silu:
            return self.z, self.E_z
        y = self.z * self.sig
        return y, 1.1 * self.E_z + (12 + 2.4 * self.z.abs()) * U * y.abs() + 1e-36 * (1 + self.z.abs())

    def backward(self, dy):
        dz, E_dz = dy.double(), torch.zeros_like(self.z)
        if self.silu:
            slope = self.sig * (1 + self.z * (1 - self.sig))
            E_dz = dz.abs() * (0.5 * self.E_z + (16 + 10 * self.z.abs()) * U)
            dz = dz * slope
            E_dz = E_dz + U * dz.abs()
        depth = (min(self.n, 512) + 16) * U
        dw, mass = (dz * self.xhat).sum(0), (dz * self.xhat).abs().sum(0)
        E_dw = (E_dz * self.xhat.abs() + dz.abs() * self.E).sum(0) + depth * mass
        db, E_db = dz.sum(0), E_dz.sum(0) + depth * dz.abs().sum(0)
        g = dz * self.w
        E_g = E_dz * self.w.abs() + U * g.abs()
        c1, c2 = g.mean(1, keepdim=True), (g * self.xhat).mean(1, keepdim=True)
        E_c1 = E_g.mean(1, keepdim=True) + 26 * U * g.abs().mean(1, keepdim=True)
        E_c2 = ((E_g * self.xhat.abs() + g.abs() * self.E).mean(1, keepdim=True)
                + 27 * U * (g * self.xhat).abs().mean(1, keepdim=True))
        dx = self.rstd * (g - c1 - self.xhat * c2)
        E_dx = self.rstd * (E_g + E_c1 + self.E * c2.abs() + self.xhat.abs() * E_c2
                            + 4 * U * (g.abs() + c1.abs() + (self.xhat * c2).abs()))
        return (dx, E_dx + dx.abs() * (self.D + 18 * U)), (dw, E_dw), (db, E_db)


def assert_close(got, want, bound, what="", norm=True):
    bound = bound * 1.01 + 1e-37
    if got.dtype == BF16:
        bound = bound * (1 + 2.0**-8) + 2.0**-8 * want.abs()
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} values off, worst {float(off.max()):.3e}, {float((off / bound).max()):.2f} of its bound"
    if norm:
        rel, size = float(off.norm()), float(want.norm())
        assert rel <= (2.0**-19 if got.dtype == F32 else 2.0**-8 + 2.0**-19) * size, f"{what}: relative error {rel / size:.3e}"


def check_rows(nm, x, dy, w, b, eps=1e-5, silu=False, norm=True):
    act = "silu" if silu else None
    ref = Rows64(x, w, b, eps, silu)
    y = nm.layer_norm(x, w, b, eps=eps, activation=act)
    assert y.dtype == x.dtype and y.shape == x.shape
    assert_close(y, *ref.forward(), "y", norm)
    got = nm.layer_norm_grad(x, dy, w, b, eps=eps, activation=act)
    for name, value, (want, bound), like in zip(("dx", "dw", "db"), got, ref.backward(dy), (x, w, b)):
        if like is None:
            assert value is None
            continue
        assert value.dtype == like.dtype and value.shape == like.shape
        assert_close(value, want, bound, name, norm)


# ----------------------------------------------------------------- layer norm
@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("dtype,param", [(F32, F32), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("n,c", [(1, 1), (5, 1), (3, 2), (40, 3), (1, 8), (70, 16), (33, 31), (1000, 32), (129, 33),
                                 (4097, 64), (1, 64), (300, 61), (1003, 97), (500, 96), (1, 128), (777, 128), (64, 130),
                                 (100, 250), (31, 255), (1000, 256), (65, 257), (50, 264), (20, 511), (200, 512),
                                 (7, 1000), (33, 2048), (3, 4097), (2, 8191), (5, 8192)])  # fmt: skip
def test_layer_norm_and_its_gradients(nm, n, c, dtype, param, silu):
    x, dy, w, b = inputs(n, c, dtype, param, seed=n + c)
    # (two or three channels leave dx as the small difference of large terms, one none at all)
    check_rows(nm, x, dy, w, b, silu=silu, norm=c >= 8)


@pytest.mark.parametrize("n", [200_003, 1_500_001])
@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_of_many_rows(nm, n, dtype):
    x, dy, w, b = inputs(n, 64, dtype, F32, seed=1)
    check_rows(nm, x, dy, w, b, silu=True)


def test_sums_of_one_sign_over_many_rows(nm):
    n, c = 3_000_001, 40
    x, _, w, b = inputs(n, c, F32, F32, seed=2)
    dy = randn(n, c, seed=3).abs_() + 0.5
    check_rows(nm, x, dy, w, b)


@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("c", [64, 97, 700])
def test_layer_norm_without_parameters(nm, c, silu):
    x, dy, w, b = inputs(100, c, F32, F32, seed=4)
    for weight, bias in ((None, None), (w, None), (None, b)):
        check_rows(nm, x, dy, weight, bias, silu=silu)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c,pitch,at", [(64, 192, 64), (64, 65, 0), (64, 72, 3), (97, 200, 5), (128, 512, 128),
                                        (512, 1030, 1), (2048, 2052, 4), (300, 300, 0)])
def test_rows_in_a_wider_table(nm, dtype, c, pitch, at):
    n = 111
    x, dy, w, b = inputs(n, pitch, dtype, F32, seed=5)
    table, grads = x.clone(), dy.clone()
    x, dy, w, b = x[:, at:at + c], dy[:, at:at + c], w[at:at + c].clone(), b[at:at + c].clone()
    check_rows(nm, x, dy, w, b, silu=True)
    node = torch.full((n + 2, pitch), 7.0, dtype=dtype, device="cuda")
    out = node[1:n + 1, at:at + c]
    got = nm.layer_norm(x, w, b, activation="silu", out=out)
    assert got.data_ptr() == out.data_ptr()
    assert_close(out, *Rows64(x, w, b, 1e-5, True).forward(), "out")
    assert (node[0] == 7.0).all() and (node[n + 1:] == 7.0).all()
    assert (node[:, :at] == 7.0).all() and (node[:, at + c:] == 7.0).all()
    if pitch >= 2 * c + at:  # a table's slot into another slot of the same table
        into = table[:, at + c:at + 2 * c]
        before = table.clone()
        nm.layer_norm(table[:, at:at + c], w, b, activation="silu", out=into)
        # (the order of a row's sums follows its address modulo 16: within the bound, not equal bits)
        assert_close(into, *Rows64(x, w, b, 1e-5, True).forward(), "slot")
        before[:, at + c:at + 2 * c] = into
        assert torch.equal(table, before)
    assert torch.equal(grads[:, at:at + c], dy)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", [3, 9, 17, 33, 65, 96, 97, 250, 257, 500, 511, 1001, 8189])
def test_rows_among_neighbours_that_are_not_numbers(nm, dtype, c):
    """Rows at every address modulo 16, one behind the other or with gaps: what lies around them does not enter, and
    nothing but the rows is written."""
    for n, gap, at in ((1, 0, 1), (2, 0, 0), (9, 0, 3), (21, 0, 5), (21, 1, 0), (17, 5, 7), (40, 8, 2)):
        if c > 1000:
            n = min(n, 9)
        size = at + n * (c + gap) + 16

        def rows(values, fill):
            t = torch.full((size,), fill, dtype=dtype, device="cuda")
            v = t.as_strided((n, c), (c + gap, 1), at)
            v.copy_(values)
            return t, v

        x, dy, w, b = inputs(n, c, dtype, F32, seed=c + n)
        x, dy = rows(x, float("nan"))[1], rows(dy, float("nan"))[1]
        check_rows(nm, x, dy, w, b, silu=True, norm=False)
        table, out = rows(torch.zeros(n, c), 7.0)
        nm.layer_norm(x, w, b, activation="silu", out=out)
        assert_close(out, *Rows64(x, w, b, 1e-5, True).forward(), "out", norm=False)
        out.fill_(7.0)
        assert (table == 7.0).all()


def test_repeated_rows_and_other_shapes(nm):
    c = 64
    x, dy, w, b = inputs(1, c, F32, F32, seed=6)
    many = x.expand(50, c)
    assert torch.equal(nm.layer_norm(many, w, b), nm.layer_norm(x, w, b).expand(50, c))
    dx, dw, db = nm.layer_norm_grad(many, dy.expand(50, c), w, b)
    one = nm.layer_norm_grad(x, dy, w, b)
    assert torch.equal(dx, one[0].expand(50, c))
    ref = Rows64(many, w, b, 1e-5, False).backward(dy.expand(50, c))
    assert_close(dw, *ref[1])
    assert_close(db, *ref[2])
    x, dy, w, b = inputs(24, c, F32, F32, seed=7)
    want, grads = nm.layer_norm(x, w, b), nm.layer_norm_grad(x, dy, w, b)
    for shape in ((2, 3, 4, c), (24, 1, c), (1, 24, c)):
        assert torch.equal(nm.layer_norm(x.view(shape), w, b), want.view(shape))
        got = nm.layer_norm_grad(x.view(shape), dy.view(shape), w, b)
        assert torch.equal(got[0], grads[0].view(shape)) and torch.equal(got[1], grads[1])
    assert torch.equal(nm.layer_norm(x[0], w, b), want[0])  # one row without leading dimensions


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(0, 64), (0, 97), (0, 2048), (3, 0, 64)])
def test_no_rows(nm, dtype, shape):
    x, w = torch.zeros(shape, dtype=dtype, device="cuda"), torch.ones(shape[-1], device="cuda")
    assert nm.layer_norm(x, w, w).shape == shape
    dx, dw, db = nm.layer_norm_grad(x, x, w, w, activation="silu")
    assert dx.shape == shape and not dw.any() and not db.any()


@pytest.mark.parametrize("c", [8, 64, 97, 300, 2048])
@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_and_offset_rows(nm, dtype, c):
    """A row of equal values is b (or its SiLU) exactly, whatever the value; an offset common to a row changes nothing
    but what it rounds in x itself."""
    _, dy, w, b = inputs(6, c, dtype, dtype, seed=8)
    value = torch.tensor([0.0, 1.0, -3.7, 1e6 + 3, 1e-20, -2e17], device="cuda")
    x = value[:, None].expand(6, c).to(dtype).contiguous()
    assert torch.equal(nm.layer_norm(x, w, b), b.expand(6, c))
    check_rows(nm, x, dy, w, b, norm=False)
    x = (randn(6, c, seed=9) + torch.tensor([0.0, 10, 1e3, 1e4, -1e5, 3e5], device="cuda")[:, None]).to(dtype)
    check_rows(nm, x, dy, w, b, silu=True, norm=False)
    if dtype == F32:
        # the bound holds for the spread of a row, which no offset enters: as accurate as without it
        for eps in (1e-5, 0.0):
            check_rows(nm, x, dy, w, b, eps=eps, norm=True)


def test_scales_from_1e_minus_15_to_1e15(nm):
    x, dy, w, b = inputs(31, 64, F32, F32, seed=10)
    for scale in (1e-15, 1e-6, 1e6, 1e15):
        check_rows(nm, x * scale, dy, w, b, eps=0.0)
        check_rows(nm, x * scale, dy * scale, w, b, eps=1e-5, norm=False)


@pytest.mark.parametrize("c", [31, 64, 97, 256, 520])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_are_not_finite_stay_by_themselves(nm, dtype, c):
    n = 45
    x, dy, w, b = inputs(n, c, dtype, F32, seed=11)
    want = nm.layer_norm(x, w, b, activation="silu"), nm.layer_norm_grad(x, dy, w, b, activation="silu")[0]
    bad = [3, 17, 18, 44]
    x[3, 0], x[17, c - 1], x[18, c // 2], x[44] = float("nan"), float("inf"), -float("inf"), float("inf")
    good = torch.ones(n, dtype=torch.bool, device="cuda")
    good[bad] = False
    y = nm.layer_norm(x, w, b, activation="silu")
    dx, dw, db = nm.layer_norm_grad(x, dy, w, b, activation="silu")
    for got, expected in zip((y, dx), want):
        assert torch.equal(got[good], expected[good])
        assert got[~good].isnan().all()
    assert dw.isnan().all() and db.isnan().all()
    # rows behind the last of a warp's are no rows: eps 0 leaves no trace of them
    x, dy, w, b = inputs(5, c, dtype, F32, seed=12)
    assert all(t.isfinite().all() for t in nm.layer_norm_grad(x, dy, w, b, eps=0.0, activation="silu"))


def test_large_pre_activations(nm):
    """SiLU far from zero: neither exp(-z) nor its reciprocal spoils the result."""
    x, dy, w, b = inputs(50, 64, F32, F32, seed=13)
    b = torch.linspace(-200, 200, 64, device="cuda")
    check_rows(nm, x, dy, w, b, silu=True)
    check_rows(nm, x, dy, 30 * w, b, silu=True)


def test_offsets_past_32_bits(nm):
    n, c = 33_600_011, 64  # 2.15e9 values of 2 bytes
    x = torch.empty(n, c, dtype=BF16, device="cuda").normal_(generator=gen(14))
    dy = torch.empty(n, c, dtype=BF16, device="cuda").normal_(generator=gen(15))
    w, b = 1 + 0.1 * randn(c, seed=16), randn(c, seed=17)
    y = nm.layer_norm(x, w, b, activation="silu")
    for at in (0, n // 2, 2**25 - 7, n - 1001):
        assert torch.equal(y[at:at + 1001], nm.layer_norm(x[at:at + 1001], w, b, activation="silu"))
    del y
    dx, dw, db = nm.layer_norm_grad(x, dy, w, b, activation="silu")
    for at in (0, n // 2, 2**25 - 7, n - 1001):
        want = nm.layer_norm_grad(x[at:at + 1001], dy[at:at + 1001], w, b, activation="silu")[0]
        assert torch.equal(dx[at:at + 1001], want)
    del dx
    sums = torch.zeros(2, c, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(sums)
    for xs, ds in zip(x.split(2_000_000), dy.split(2_000_000)):
        _, (pw, ew), (pb, eb) = Rows64(xs, w, b, 1e-5, True).backward(ds)
        sums += torch.stack([pw, pb])
        bound += torch.stack([ew, eb])
    assert_close(dw, sums[0], bound[0], "dw", norm=False)
    assert_close(db, sums[1], bound[1], "db", norm=False)


@pytest.mark.parametrize("c", [1, 2, 13, 64, 300])
def test_gradients_against_differences(nm, c):
    """The gradients' product with a step is the definition's change along it, in 64 bits."""
    n = 9
    x, dy, w, b = inputs(n, c, F32, F32, seed=18)
    dx, dw, db = (t.double() for t in nm.layer_norm_grad(x, dy, w, b, activation="silu", eps=1e-2))
    step = [randn(*t.shape, seed=19 + i).double() for i, t in enumerate((x, w, b))]

    def loss(h):
        moved = [t.double() + h * s for t, s in zip((x, w, b), step)]
        eps = float(torch.tensor(1e-2))
        return float((Rows64(*moved, eps, True).forward()[0] * dy.double()).sum())

    def slope(h):  # central differences, error of the order h^4
        return (8 * (loss(h) - loss(-h)) - (loss(2 * h) - loss(-2 * h))) / (12 * h)

    want = slope(1e-3)
    dot = float((dx * step[0]).sum() + (dw * step[1]).sum() + (db * step[2]).sum())
    ref = Rows64(x, w, b, 1e-2, True).backward(dy)
    bound = sum(float((e * s.abs()).sum()) for (_, e), s in zip(ref, step)) + 10 * abs(want - slope(2e-3)) + 1e-9
    assert abs(dot - want) <= bound, (dot, want, bound)
    assert bound < 0.05 * abs(want) or c == 1


# ------------------------------------------------------------------- autograd
@pytest.mark.parametrize("dtype,param", [(F32, F32), (BF16, F32)])
def test_autograd(nm, dtype, param):
    n, c = 300, 96
    x, dy, w, b = inputs(n, c, dtype, param, seed=20)
    want = nm.layer_norm_grad(x, dy, w, b, activation="silu")
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = nm.layer_norm(*leaves, activation="silu")
    assert torch.equal(y.detach(), nm.layer_norm(x, w, b, activation="silu"))
    y.backward(dy)
    assert all(torch.equal(t.grad, g) for t, g in zip(leaves, want))
    for frozen in range(3):  # what needs no gradient gets none, the others the same bits
        leaves = [t.clone().requires_grad_(i != frozen) for i, t in enumerate((x, w, b))]
        nm.layer_norm(*leaves, activation="silu").backward(dy)
        for i, (t, g) in enumerate(zip(leaves, want)):
            assert t.grad is None if i == frozen else torch.equal(t.grad, g)
    only = x.clone().requires_grad_()
    nm.layer_norm(only).backward(dy)
    assert torch.equal(only.grad, nm.layer_norm_grad(x, dy)[0])
    with torch.no_grad():
        assert not nm.layer_norm(leaves[0], leaves[1]).requires_grad


def test_autograd_of_expanded_and_permuted_gradients(nm):
    n, c = 200, 33
    x, _, w, b = inputs(n, c, F32, F32, seed=21)
    x, w, b = x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    nm.layer_norm(x, w, b).sum().backward()
    want = nm.layer_norm_grad(x.detach(), torch.ones(n, c, device="cuda"), w.detach(), b.detach())
    assert all(torch.equal(t.grad, g) for t, g in zip((x, w, b), want))
    x.grad = w.grad = b.grad = None
    v = randn(c, n, seed=22)
    (nm.layer_norm(x, w, b).T * v).sum().backward()
    want = nm.layer_norm_grad(x.detach(), v.T.contiguous(), w.detach(), b.detach())
    assert all(torch.equal(t.grad, g) for t, g in zip((x, w, b), want))
    x.grad = w.grad = b.grad = None
    # parameters shared by two uses add up
    (nm.layer_norm(x, w, b) + nm.layer_norm(x, w, b)).sum().backward()
    once = nm.layer_norm_grad(x.detach(), torch.ones(n, c, device="cuda"), w.detach(), b.detach())
    assert all(torch.equal(t.grad, g + g) for t, g in zip((x, w, b), once))
    # a slot of a table, several leading dimensions
    table = randn(6, 7, 3 * c, seed=23).requires_grad_()
    dy = randn(6, 7, c, seed=24)
    nm.layer_norm(table[..., c:2 * c], w, b).backward(dy)
    want = nm.layer_norm_grad(table.detach()[..., c:2 * c], dy, w.detach(), b.detach())[0]
    assert torch.equal(table.grad[..., c:2 * c], want) and not table.grad[..., :c].any()


def test_second_derivatives_are_refused(nm):
    x = randn(4, 8, seed=25).requires_grad_()
    (g,) = torch.autograd.grad(nm.layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_a_changed_input_is_noticed(nm):
    x = randn(4, 8, seed=26).requires_grad_()
    h = x * 1.0
    y = nm.layer_norm(h)
    with torch.no_grad():
        nm.layer_norm(randn(4, 8, seed=27), out=h)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# ------------------------------------------------------------- gradient norms
def lists_of_gradients():
    return {
        "one": [(1,)], "scalar": [()], "empty among others": [(0,), (5, 3), (0, 7)], "odd": [(1,), (7, 3), (129,), (33, 5)],
        "around a tile": [(4095,), (4096,), (4097,), (8191,), (8192,), (8193,)], "many small": [(3,)] * 300,
        "large": [(1000, 1001), (17,), (3_000_001,)], "65": [(10,)] * 65, "257": [(64, 9)] * 257,
        "thousands": [(1 + i % 50,) for i in range(2500)],
    }  # fmt: skip


def norm64(grads):
    return torch.cat([g.double().flatten() for g in grads]).norm()


def assert_norm(got, grads):
    assert got.dtype == F32 and got.shape == ()
    want = norm64(grads)
    # the fp64 sum is off by far less than fp32's half unit
    assert abs(got.double() - want) <= U * (1 + 2.0**-10) * want + 2.0**-150


@pytest.mark.parametrize("dtype", [F32, BF16, "mixed"])
@pytest.mark.parametrize("name", list(lists_of_gradients()))
def test_gradient_norm(nm, name, dtype):
    grads = [randn(*s, seed=i, dtype=(F32, BF16)[i % 2] if dtype == "mixed" else dtype)
             for i, s in enumerate(lists_of_gradients()[name])]
    before = [g.clone() for g in grads]
    got = nm.grad_norm(grads)
    assert_norm(got, grads)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    assert torch.equal(nm.grad_norm([None, *grads, None]), got)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_norm_of_every_alignment(nm, dtype):
    flat = randn(20_000, seed=30, dtype=dtype)
    for at in range(9):
        for size in (1, 2, 7, 8, 9, 15, 16, 17, 4090, 4096, 4100, 8200):
            assert_norm(nm.grad_norm([flat[at:at + size]]), [flat[at:at + size]])


def test_gradient_norm_of_extreme_values(nm):
    for scale in (1e-40, 1e-30, 1e-20, 1e10, 1e25, 1e35):
        grads = [randn(1000, seed=31).clamp(-3, 3) * scale, torch.zeros(5, device="cuda")]
        assert_norm(nm.grad_norm(grads), grads)
    assert float(nm.grad_norm([torch.zeros(10, device="cuda")])) == 0.0
    assert float(nm.grad_norm([])) == 0.0 and float(nm.grad_norm([None])) == 0.0
    assert float(nm.grad_norm([torch.zeros(0, device="cuda")])) == 0.0
    big = torch.full((4,), 3e38, device="cuda")  # the norm itself lies past fp32
    assert float(nm.grad_norm([big])) == float("inf")
    for value in (float("inf"), -float("inf"), float("nan")):
        for dtype in DTYPES:
            for more in (0, 1_000_000):
                grads = [randn(100, seed=32, dtype=dtype), randn(5000 + more, seed=33, dtype=dtype)]
                grads[1][4321] = value
                got = float(nm.grad_norm(grads))
                assert got != got if value != value else got == float("inf")


@pytest.mark.parametrize("size", [777, 2_000_000])
def test_gradient_norm_of_16_bit_values_at_the_ends_of_their_range(nm, size):
    zeros = torch.zeros(size, dtype=BF16, device="cuda")
    assert float(nm.grad_norm([zeros, -zeros])) == 0.0
    for value in (2.0**-133, 2.0**-126, 1.5 * 2.0**-127, 2.0**-60, 1.0, 2.0**127, float(torch.finfo(BF16).max)):
        for where in (slice(0, 1), slice(5, 9), slice(size - 1, size)):  # subnormals, the least normal, the largest
            g = zeros.clone()
            g[where] = value
            got, want = float(nm.grad_norm([g])), abs(value) * (where.stop - where.start) ** 0.5
            assert got == float(torch.tensor(want, dtype=torch.float64).float()), (value, where)  # (2^128 rounds to inf)
    both = zeros.clone()
    both[3], both[4] = 2.0**-133, 3 * 2.0**-132
    assert_norm(nm.grad_norm([both]), [both])


def test_gradient_norm_in_any_order_of_dimensions(nm):
    g = randn(30, 7, 11, seed=34)
    for t in (g.permute(2, 0, 1), g.transpose(0, 2), g[:, :, :, None], g[5:20]):
        assert_norm(nm.grad_norm([t]), [t])


def test_operands_are_read_the_same_both_ways(nm, monkeypatch):
    base, w = randn(24, 4, 96, seed=37), 1 + 0.1 * randn(96, seed=38)
    b = randn(96, seed=39)
    cases = [(t, w, b) for t in (base, base[:, 1], base[..., :96], base[0, 0], base[:1], base[::3, 2], base[:0], base[3:, :1],
                                 base[:, :, None], base[2:3, 1:2], base[0, :1].expand(7, 96), base.view(6, 4, 4, 96)[:, :, 1])]
    cases += [(base[..., 5:9], w[5:9], None), (base[..., :1], None, b[:1]), (base.bfloat16(), w, b), (base[:, 0, 7:8], w[:1], b[:1]),
              (base.bfloat16()[:, 0], w.bfloat16(), b.bfloat16()), (torch.nn.Parameter(base[0].clone()), None, None)]
    readers = [nm._reader, None]
    assert nm._read_rows(base, base, w, b) is not None or readers[0] is None
    for x, weight, bias in cases:
        got = []
        for reader in readers:
            monkeypatch.setattr(nm, "_reader", reader)
            assert reader is None or nm._read_rows(x, x, weight, bias) is not None
            with torch.no_grad():
                y = nm.layer_norm(x, weight, bias, activation="silu")
                got.append([y, *nm.layer_norm_grad(x, x, weight, bias, activation="silu")])
        assert got[0][0].shape == x.shape and got[0][0].is_contiguous()
        for p, q in zip(*got):
            assert (p is None and q is None) or (torch.equal(p, q) and p.dtype == q.dtype and p.stride() == q.stride())


@pytest.mark.parametrize("reader", ["dlpack", "attributes"])
def test_lists_are_read_the_same_both_ways(nm, reader, monkeypatch):
    base = randn(40, 50, seed=36)
    tensors = [base, base[3:7], base[5], base.T, base[:, :1].contiguous(), base[:1, :1], base[2, 3], base[:0], base.view(-1)[7:],
               base.bfloat16(), torch.nn.Parameter(base.clone()), base.view(40, 1, 50), base.view(-1)[1:1]]
    if reader == "attributes":
        monkeypatch.setattr(nm, "_reader", None)
    ptrs, sizes, codes, contiguous = nm._flat("grads", tensors, 0)
    assert not contiguous and list(sizes) == [t.numel() for t in tensors]
    assert all(p == t.data_ptr() for p, t in zip(ptrs, tensors) if t.numel())
    assert list(codes) == [int(t.dtype == BF16) for t in tensors]
    tensors = [t for t in tensors if t.is_contiguous()]
    ptrs, sizes, codes, contiguous = nm._flat("grads", tensors, 0)
    assert contiguous and list(sizes) == [t.numel() for t in tensors]
    assert all(p == t.data_ptr() for p, t in zip(ptrs, tensors) if t.numel())
    assert_norm(nm.grad_norm(tensors), [t.detach() for t in tensors])
    out = [torch.empty_like(t, requires_grad=False) for t in tensors]
    want = clipped64([t.detach() for t in tensors], 3.0)
    nm.clip_grads(tensors, 3.0, out=out)
    assert_clipped(out, want)
    for bad in (base.half(), base.double(), base.cpu(), base[:, ::2], base.to_sparse(), base[:1].expand(3, 50)):
        with pytest.raises(ValueError):
            nm.grad_norm([base, bad])
    with pytest.raises(TypeError):
        nm.grad_norm([base, 1.0])


def test_gradient_norm_past_32_bits(nm):
    g = torch.empty(2**31 + 12345, dtype=BF16, device="cuda").normal_(generator=gen(35))
    want = sum(float(part.double().square().sum()) for part in g.split(2**28)) ** 0.5
    assert abs(float(nm.grad_norm([g, g[:1]])) - (want**2 + float(g[0]) ** 2) ** 0.5) <= 2 * U * want
    guard = g[-1].clone()
    nm.clip_grads([g[:-1]], want / 2)
    assert g[-1] == guard
    after = sum(float(part.double().square().sum()) for part in g[:-1].split(2**28)) ** 0.5
    assert abs(after - want / 2) <= 2.0**-8 * want


def clipped64(grads, max_norm):
    norm = norm64(grads)
    return [g.double() * torch.clamp(max_norm / (norm + 1e-6), max=1.0) for g in grads]


def assert_clipped(got, want):
    for a, b in zip(got, want, strict=True):
        # the factor rounds once, the product once, a 16-bit result once more
        bound = 2.01 * U * b.abs() + 2.0**-150 + (2.0**-8 * b.abs() if a.dtype == BF16 else 0.0)
        assert not ((a.double() - b).abs() > bound).any()


@pytest.mark.parametrize("dtype", [F32, BF16, "mixed"])
@pytest.mark.parametrize("name", list(lists_of_gradients()))
def test_clipping_in_place(nm, name, dtype):
    grads = [randn(*s, seed=i, dtype=(F32, BF16)[i % 2] if dtype == "mixed" else dtype)
             for i, s in enumerate(lists_of_gradients()[name])]
    norm = norm64(grads)
    before = [g.clone() for g in grads]
    got = nm.clip_grads(grads, float(norm) * 1.5)
    assert_norm(got, before)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    got = nm.clip_grads([None, *grads], float(norm) * 0.3)
    assert_norm(got, before)
    assert_clipped(grads, clipped64(before, float(norm) * 0.3))


@pytest.mark.parametrize("ins", DTYPES)
@pytest.mark.parametrize("outs", DTYPES)
def test_clipping_into_other_tensors(nm, ins, outs):
    shapes = [(1,), (7, 3), (0,), (4097,), (64, 64), (8193,), (100_003,)]
    sizes = [torch.Size(s).numel() for s in shapes]
    for shift in range(9):  # outputs one behind the other, at every address relative to the inputs'
        grads = [randn(*s, seed=i, dtype=ins) for i, s in enumerate(shapes)]
        before = [g.clone() for g in grads]
        buffer = torch.full((shift + sum(sizes) + 3,), 7.0, dtype=outs, device="cuda")
        out = [part.view(s) for part, s in zip(buffer[shift:shift + sum(sizes)].split(sizes), shapes)]
        for factor in (0.5, 2.0):
            max_norm = float(norm64(grads)) * factor
            assert_norm(nm.clip_grads([None, *grads], max_norm, out=[None, *out]), grads)
            assert_clipped(out, clipped64(grads, max_norm))
            if factor == 2.0:
                assert all(torch.equal(o, g.to(outs)) for o, g in zip(out, grads))
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
        assert (buffer[:shift] == 7.0).all() and (buffer[-3:] == 7.0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_clipping_packed_gradients(nm, dtype):
    """Gradients one behind the other in one buffer, each at any address: the gaps keep their values."""
    sizes = [5, 1, 4096, 33, 2, 8191, 16, 3, 1000]
    flat = randn(sum(sizes) + 9 * len(sizes), seed=40, dtype=dtype)
    at, grads, kept = 0, [], torch.ones(len(flat), dtype=torch.bool, device="cuda")
    for i, size in enumerate(sizes):
        grads.append(flat[at:at + size])
        kept[at:at + size] = False
        at += size + i % 3
    before = flat.clone()
    want = clipped64([g.clone() for g in grads], 3.0)
    nm.clip_grads(grads, 3.0)
    assert_clipped(grads, want)
    assert torch.equal(flat[kept], before[kept])


def test_clipping_of_some_in_place_and_some_elsewhere(nm):
    a, b, c = randn(100, seed=41), randn(40, 50, seed=42).T, randn(77, seed=43, dtype=BF16)
    into = [a, torch.empty_like(b), torch.empty(77, device="cuda")]
    assert into[1].stride() == b.stride()
    want = clipped64([a, b, c], 5.0)
    nm.clip_grads([a, b, c], 5.0, out=into)
    assert_clipped(into, want)
    again = clipped64([a, b, c], 1e9)
    nm.clip_grads([a, b, c], 1e9, out=into)
    assert_clipped(into, again)


def test_clipping_to_zero_and_of_infinities(nm):
    g = randn(5000, seed=44)
    nm.clip_grads([g], 0.0)
    assert not g.any()
    nm.clip_grads([g], 0.0)  # a zero norm: 0 / 1e-6
    assert not g.any()
    assert float(nm.clip_grads([], 1.0)) == 0.0 and float(nm.clip_grads([None], 1.0, out=[None])) == 0.0
    g = randn(5000, seed=45)
    g[17] = float("inf")
    assert float(nm.clip_grads([g], 1.0)) == float("inf")
    assert g[17].isnan() and not g[:17].any() and not g[18:].any()
    g = randn(5000, seed=46)
    g[17] = float("nan")
    nm.clip_grads([g], 1.0)
    assert g.isnan().all()


def test_clipping_counts_as_a_change(nm):
    g = randn(10, seed=47)
    version = g._version
    nm.grad_norm([g])
    assert g._version == version
    nm.clip_grads([g], 1.0)
    assert g._version > version


# ------------------------------------------------------------ streams, graphs
def everything(nm, x, dy, w, b, grads, out):
    y = nm.layer_norm(x, w, b, activation="silu")
    more = nm.layer_norm_grad(x, dy, w, b, activation="silu")
    wide = nm.layer_norm_grad(x.view(-1, 1536), dy.view(-1, 1536), activation="silu")[0]
    return [y, *more, wide, nm.grad_norm([*grads, more[1]]), nm.clip_grads([*grads, more[2]], 2.0, out=out), *out]


# one cluster each, or several launches with workspaces
SIZES = {"small": (64, 5000), "large": (9008, 2_000_000)}


def step_inputs(seed, size):
    n, values = SIZES[size]
    x, dy, w, b = inputs(n, 96, F32, F32, seed=seed)
    grads = [randn(values, seed=seed + 7), randn(33, 3, seed=seed + 8, dtype=BF16)]
    return x, dy, w, b, grads


def step_outputs(size):
    return [torch.empty(SIZES[size][1], device="cuda"), torch.empty(33, 3, device="cuda"), torch.empty(96, device="cuda")]


@pytest.mark.parametrize("size", list(SIZES))
def test_other_streams_and_cuda_graphs(nm, size):
    def outputs():
        return step_outputs(size)

    x, dy, w, b, grads = step_inputs(50, size)
    want = [t.clone() for t in everything(nm, x, dy, w, b, grads, outputs())]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = everything(nm, x, dy, w, b, grads, outputs())
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    graphs, results = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        out = outputs()
        with torch.cuda.graph(graph):
            results.append(everything(nm, x, dy, w, b, grads, out))
    for factor in (2.0, 0.01):  # (clipped, and below the bound)
        x.mul_(factor)
        dy.mul_(factor)
        for g in grads:
            g.mul_(factor)
        want = everything(nm, x, dy, w, b, grads, outputs())
        for graph, got in zip(graphs, results):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_in_place_clipping_in_a_graph(nm):
    source, g = randn(100_000, seed=60), torch.zeros(100_000, device="cuda")
    nm.clip_grads([g], 1.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g.copy_(source)
        norm = nm.clip_grads([g], 10.0)
    for factor in (1.0, 1e-3, 50.0):
        source.copy_(randn(100_000, seed=61) * factor)
        graph.replay()
        torch.cuda.synchronize()
        assert_norm(norm, [source])
        assert_clipped([g], clipped64([source], 10.0))


def test_training_step_in_a_graph(nm):
    """Forward, backward and clipping captured as one step, replayed on new inputs."""
    n, c = 500, 64
    x, _, w, b = inputs(n, c, F32, F32, seed=62)
    leaves = [t.clone().requires_grad_() for t in (w, b)]
    target = randn(n, c, seed=63)

    def step():
        loss = (nm.layer_norm(x, *leaves, activation="silu") - target).square().sum()
        got = torch.autograd.grad(loss, leaves)
        return [*got, nm.clip_grads(got, 1.0)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    x.copy_(randn(n, c, seed=64))
    graph.replay()
    want = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, d) for a, d in zip(got, want))


@pytest.mark.parametrize("size", list(SIZES))
def test_calls_from_two_host_threads(nm, size):
    import threading

    def outputs():
        return step_outputs(size)

    data = {seed: step_inputs(seed, size) for seed in (70, 80)}
    want = {seed: [t.clone() for t in everything(nm, *d, outputs())] for seed, d in data.items()}
    torch.cuda.synchronize()
    got, errors = {}, []

    def thread(seed):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[seed] = everything(nm, *data[seed], outputs())
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=thread, args=(seed,)) for seed in data]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for seed, values in want.items():
        assert all(torch.equal(a, b) for a, b in zip(got[seed], values, strict=True))


@pytest.mark.parametrize("dtype", DTYPES)
def test_calls_in_a_row_on_buffers_used_again(nm, dtype):
    """Each call reads what the call before it has just written to memory that earlier calls had read."""
    n, c = 3000, 64
    sources = [inputs(n, c, dtype, F32, seed=90 + 10 * k) for k in range(6)]

    def chain(k, x, rows, again):
        source, dy, w, b = sources[k]
        x.copy_(source)
        nm.layer_norm(x, w, b, activation="silu", out=rows)
        nm.layer_norm(rows, w, b, out=again)
        grads = nm.layer_norm_grad(rows, again, w, b, activation="silu")
        norm = nm.clip_grads(list(grads), 1.0)
        return [rows.clone(), again.clone(), *grads, norm]

    def buffers():
        return [torch.empty(n, c, dtype=dtype, device="cuda") for _ in range(3)]

    want = []
    for k in range(6):
        want.append(chain(k, *buffers()))
        torch.cuda.synchronize()
    shared = buffers()
    for _ in range(10):
        got = [chain(k, *shared) for k in range(6)]
        for a, b in zip(sum(got, []), sum(want, []), strict=True):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,n,c", [(F32, 30_011, 64), (BF16, 30_011, 97), (F32, 3001, 2048), (F32, 777, 129)])
def test_equal_calls_give_equal_bits(nm, dtype, n, c):
    x, dy, w, b = inputs(n, c, dtype, F32, seed=100)
    first = [nm.layer_norm(x, w, b), *nm.layer_norm_grad(x, dy, w, b), nm.grad_norm([x, dy, w])]
    for _ in range(5):
        again = [nm.layer_norm(x, w, b), *nm.layer_norm_grad(x, dy, w, b), nm.grad_norm([x, dy, w])]
        assert all(torch.equal(p, q) for p, q in zip(first, again))


# ------------------------------------------------------------------ refusals
@pytest.mark.parametrize("reader", ["dlpack", "attributes"])
def test_refusals(nm, reader, monkeypatch):
    if reader == "attributes":
        monkeypatch.setattr(nm, "_reader", None)
    x, w, b = torch.zeros(8, 16, device="cuda"), torch.ones(16, device="cuda"), torch.zeros(16, device="cuda")
    leaf = torch.zeros(8, 16, device="cuda", requires_grad=True)
    g, h = torch.zeros(40, device="cuda"), torch.zeros(40, device="cuda")
    bad = [
        lambda: nm.layer_norm(x.half(), w, b), lambda: nm.layer_norm(x.double()), lambda: nm.layer_norm(x.T, b[:8]),
        lambda: nm.layer_norm(x[:, ::2], w[:8]), lambda: nm.layer_norm(x, w[:8]), lambda: nm.layer_norm(x, w, b[:8]),
        lambda: nm.layer_norm(x, w[None]), lambda: nm.layer_norm(x, w.cpu(), b), lambda: nm.layer_norm(x, w, b.cpu()),
        lambda: nm.layer_norm(x, w.bfloat16()), lambda: nm.layer_norm(x.bfloat16(), w.bfloat16(), b),
        lambda: nm.layer_norm(x, torch.ones(32, device="cuda")[::2]), lambda: nm.layer_norm(x, w.double()),
        lambda: nm.layer_norm(x, w, b, eps=-1.0), lambda: nm.layer_norm(x, w, b, eps=float("nan")),
        lambda: nm.layer_norm(x, w, b, eps=float("inf")), lambda: nm.layer_norm(x, activation="relu"),
        lambda: nm.layer_norm(x, out=torch.zeros(7, 16, device="cuda")), lambda: nm.layer_norm(x, out=x.bfloat16()),
        lambda: nm.layer_norm(x, out=torch.zeros(16, device="cuda").expand(8, 16)),
        lambda: nm.layer_norm(x, out=torch.zeros(8, 16)), lambda: nm.layer_norm(leaf, out=torch.zeros_like(x)),
        lambda: nm.layer_norm(torch.zeros((), device="cuda")), lambda: nm.layer_norm(torch.zeros(4, 0, device="cuda")),
        lambda: nm.layer_norm(torch.zeros(2, 8193, device="cuda")),
        lambda: nm.layer_norm(torch.zeros(4, 6, 16, device="cuda")[:, :5]),  # no one stride between the rows
        lambda: nm.layer_norm_grad(x, x[:4]), lambda: nm.layer_norm_grad(x, x.bfloat16()),
        lambda: nm.layer_norm_grad(x, torch.ones(1, device="cuda").expand(8, 16)), lambda: nm.layer_norm_grad(x, x.cpu()),
        lambda: nm.layer_norm_grad(x, x, w[:4]), lambda: nm.layer_norm_grad(x, x, activation="gelu"),
        lambda: nm.grad_norm([g.half()]), lambda: nm.grad_norm([g.double()]), lambda: nm.grad_norm([g, g.cpu()]),
        lambda: nm.grad_norm([g[::2]]), lambda: nm.grad_norm([g[:1].expand(5)]), lambda: nm.grad_norm([g.to_sparse()]),
        lambda: nm.grad_norm([x[:, :8]]), lambda: nm.grad_norm([g.int()]),
        lambda: nm.clip_grads([g], -1.0), lambda: nm.clip_grads([g], float("inf")),
        lambda: nm.clip_grads([g], 1.0, out=[]), lambda: nm.clip_grads([g], 1.0, out=[h[:39]]),
        lambda: nm.clip_grads([g], 1.0, out=[h.half()]), lambda: nm.clip_grads([g], 1.0, out=[h.cpu()]),
        lambda: nm.clip_grads([x], 1.0, out=[torch.zeros(16, 8, device="cuda").T]),
        lambda: nm.clip_grads([x[:, :8]], 1.0), lambda: nm.clip_grads([g, h], 1.0, out=[h[:40], None][:1]),
    ]  # fmt: skip
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")
    from mace_mlx_b200.native import NativeError

    for call in (lambda: nm.clip_grads([g, g], 1.0), lambda: nm.clip_grads([g, g[3:7]], 1.0),
                 lambda: nm.clip_grads([g, h], 1.0, out=[h, torch.zeros_like(h)]),
                 lambda: nm.clip_grads([g[:39]], 1.0, out=[g[1:]]),
                 lambda: nm.clip_grads([g, h], 1.0, out=[torch.zeros(40, device="cuda")] * 2)):
        with pytest.raises(NativeError, match="overlaps"):
            call()
    for call in (lambda: nm.layer_norm([1.0]), lambda: nm.grad_norm([1.0]), lambda: nm.grad_norm(g),
                 lambda: nm.clip_grads([g], 1.0, out=[None]), lambda: nm.clip_grads([g], torch.ones((), device="cuda"))):
        with pytest.raises(TypeError):
            call()
    nm.grad_norm([g, g])  # only read: twice is twice
    torch.cuda.synchronize()


@pytest.mark.parametrize("requires_grad", [False, True])
def test_tangents_are_refused(nm, requires_grad):
    from torch.autograd import forward_ad

    plain = {"x": torch.zeros(8, 16, device="cuda"), "w": torch.ones(16, device="cuda")}
    with forward_ad.dual_level():
        dual = {k: forward_ad.make_dual(v.clone().requires_grad_(requires_grad), torch.ones_like(v))
                for k, v in plain.items()}
        for i, call in enumerate((
            lambda: nm.layer_norm(dual["x"], plain["w"]), lambda: nm.layer_norm(plain["x"], dual["w"]),
            lambda: nm.layer_norm(plain["x"], plain["w"], dual["w"]), lambda: nm.layer_norm_grad(dual["x"], plain["x"]),
            lambda: nm.layer_norm_grad(plain["x"], dual["x"]), lambda: nm.layer_norm_grad(plain["x"], plain["x"], dual["w"]),
            lambda: nm.grad_norm([plain["x"], dual["w"]]), lambda: nm.clip_grads([dual["w"]], 1.0),
        )):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
                pytest.fail(f"call {i} was accepted")
        nm.layer_norm(plain["x"], plain["w"])  # without a tangent: as ever
        nm.grad_norm([plain["w"]])


# ------------------------------------------------------------------- together
def example(name):
    import importlib.util
    import pathlib

    path = pathlib.Path(__file__).resolve().parents[1] / "examples" / f"{name}.py"
    spec = importlib.util.spec_from_file_location(name, path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_radial_mlp_has_the_plain_gradients(nm):
    ex = example("radial_mlp")
    x = ex.edge_features(6, seed=1)
    mlp = ex.RadialMLP([8, 64, 64, 97], gen(110))
    out = mlp(x)
    v = randn(*out.shape, seed=111)
    (out * v).sum().backward()
    p = {k: q.detach().double().requires_grad_() for k, q in mlp.named_parameters()}
    h = x.double()
    for i in range(3):
        h = h @ p[f"weights.{i}"].T + p[f"biases.{i}"]
        if i < 2:
            z = Rows64(h, p[f"gains.{i}"], p[f"shifts.{i}"], 1e-5, True).z
            h = z * torch.sigmoid(z)
    (h * v.double()).sum().backward()
    # fp32 sums of a few thousand terms each way: 2^-16 of the largest value covers their roundings and torch's
    assert (out.double() - h).abs().max() <= 2.0**-16 * h.abs().max()
    grads = []
    for name, q in mlp.named_parameters():
        assert (q.grad.double() - p[name].grad).abs().max() <= 2.0**-16 * p[name].grad.abs().max(), name
        grads.append(q.grad)
    before = [g.clone() for g in grads]
    want = clipped64(before, 0.1 * float(norm64(before)))
    assert_norm(nm.clip_grads([q.grad for q in mlp.parameters()], 0.1 * float(norm64(before))), before)
    assert_clipped(grads, want)


def test_examples_run_with_clipping(nm):
    losses, sizes = example("radial_mlp").train(n_structures=4, steps=5, max_norm=1e-3)
    assert len(losses) == len(sizes) == 5 and all(s > 0 for s in sizes)
    losses = example("species_head").train(n_structures=4, steps=5, max_norm=1e-3)
    assert len(losses) == 5 and all(x == x for x in losses)


# --------------------------------------------- tensors that only look like some
class Elsewhere(torch.Tensor):
    """A tensor without memory of its own, as the wrappers of distributed tensors are."""

    @staticmethod
    def __new__(cls, *shape):
        return torch.Tensor._make_wrapper_subclass(cls, shape, dtype=F32, device=torch.device("cuda", 0))

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError(func)


@pytest.mark.parametrize("reader", ["dlpack", "attributes"])
def test_tensors_without_memory_are_refused(nm, reader, monkeypatch):
    if reader == "attributes":
        monkeypatch.setattr(nm, "_reader", None)
    x, w = randn(8, 16, seed=120), Elsewhere(16)
    for call in (lambda: nm.layer_norm(x, w), lambda: nm.layer_norm(x, None, w), lambda: nm.layer_norm(x, w, out=x.clone()),
                 lambda: nm.layer_norm_grad(x, x, w), lambda: nm.layer_norm_grad(x, x, x[0], w)):
        with pytest.raises(ValueError, match="no memory"):
            call()


@pytest.mark.parametrize("default", [torch.float64, BF16])
def test_the_norm_of_nothing_under_other_default_types(nm, default):
    before = torch.get_default_dtype()
    try:
        torch.set_default_dtype(default)
        got = [nm.grad_norm([]), nm.grad_norm([None]), nm.clip_grads([], 1.0), nm.clip_grads([None], 1.0, out=[None])]
    finally:
        torch.set_default_dtype(before)
    assert all(t.dtype == F32 and float(t) == 0.0 for t in got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", [16, 33])
def test_results_beside_operands(nm, dtype, c):
    """Slots of one table, rows with a row between them and rows behind the last are taken; what overlaps is refused."""
    from mace_mlx_b200.native import NativeError

    n = 12
    table, w, b = randn(n, 3 * c, seed=121, dtype=dtype), 1 + 0.1 * randn(c, seed=122), randn(c, seed=123)
    flat = table.view(-1)
    rows = table.view(3 * n, c)
    for x, out in ((table[:, :c], table[:, c:2 * c]), (table[:, :c], table[:, 2 * c:]), (table[:, 2 * c:], table[:, c:2 * c]),
                   (rows[::6], rows[1::3][:6]), (rows[::6], rows[3::6]), (rows[:6], rows[6:12]), (rows[6:12], rows[:6]),
                   (rows[5], rows[6]), (rows[:1].expand(6, c), rows[1:7])):
        ref = Rows64(x.reshape(-1, c).clone(), w, b, 1e-5, False).forward()
        assert_close(nm.layer_norm(x, w, b, out=out).reshape(-1, c), *ref)
    for x, out in ((rows, rows), (rows[:6], rows[5:11]), (table[:, :c], table[:, 1:c + 1]), (table[:, 1:c + 1], table[:, :c]),
                   (table[:, :c], table[:, c - 1:2 * c - 1]),
                   (rows[:1].expand(6, c), rows[:6]), (rows[5], rows[5]), (flat[:6 * c].view(6, c), flat[3:6 * c + 3].view(6, c))):
        before = table.clone()
        with pytest.raises(NativeError, match="overlaps x"):
            nm.layer_norm(x, w, b, out=out)
        assert torch.equal(before, table)
    with pytest.raises(NativeError, match="overlaps a parameter"):
        nm.layer_norm(table[:, :c], table[1, c:2 * c], out=table[:, c:2 * c])
    nm.layer_norm(table[:, :c], table[1, 2 * c:], out=table[:, c:2 * c])


# ------------------------------------------- tensors that autograd follows
def test_writes_unseen_by_autograd_are_refused(nm):
    """Parameters in place of their gradients, results into parameters: refused under grad mode, as torch does."""
    leaf = torch.nn.Parameter(randn(40, seed=124))
    carried = leaf * 2.0  # (has a graph)
    g, h = randn(40, seed=125), torch.zeros(40, device="cuda")
    x, into = randn(8, 16, seed=126), torch.zeros(8, 16, device="cuda", requires_grad=True)
    before, kept = leaf.detach().clone(), g.clone()
    for call in (lambda: nm.clip_grads([leaf], 0.1), lambda: nm.clip_grads([g, leaf], 0.1), lambda: nm.clip_grads([carried], 0.1),
                 lambda: nm.clip_grads([None, g], 0.1, out=[None, leaf]), lambda: nm.clip_grads(iter([leaf]), 1e9),
                 lambda: nm.layer_norm(x, out=into)):
        with pytest.raises(ValueError, match="requires a gradient"):
            call()
    assert torch.equal(leaf, before) and torch.equal(g, kept) and not into.any()
    with torch.no_grad():
        nm.clip_grads([leaf], 0.1)
        nm.layer_norm(x, out=into)
    assert_clipped([leaf.detach()], clipped64([before], 0.1))
    assert torch.equal(into, nm.layer_norm(x))
    nm.clip_grads([g], 0.1, out=[h])
    now = leaf.detach().clone()
    nm.clip_grads([leaf.detach()], 0.01)
    assert_clipped([leaf.detach()], clipped64([now], 0.01))


def test_gradients_with_a_graph_are_refused(nm):
    """A gradient penalty on grad_norm would train nothing."""
    w = randn(30, seed=127).requires_grad_()
    (g,) = torch.autograd.grad((w**3).sum(), w, create_graph=True)
    h = torch.zeros(30, device="cuda")
    for call in (lambda: nm.grad_norm([g]), lambda: nm.grad_norm([h, g]), lambda: nm.clip_grads([h, g], 1.0, out=[h.clone(), h.clone()])):
        with pytest.raises(ValueError, match="graph"):
            call()
    want = [g.detach()]
    assert_norm(nm.grad_norm([g.detach()]), want)
    with torch.no_grad():
        assert_norm(nm.grad_norm([g]), want)
        assert_norm(nm.clip_grads([g], 1.0, out=[h]), want)
    assert_clipped([h], clipped64(want, 1.0))
    norm = nm.grad_norm([w])  # of a leaf: by its values
    assert_norm(norm, [w.detach()])
    assert not norm.requires_grad


# ------------------------------------------------ rows with one value far off
@pytest.mark.parametrize("c", [33, 61, 64, 97, 250, 257, 300, 513, 1001, 2049, 4097, 8191, 8192])
def test_one_hot_rows(nm, c):
    """One of a row's first values (all are subtracted from that, or from the one in its place) is alone in size, the
    others alike: differences and their sums are exact, the mean rounds twice in units of R, the value that is alone, a
    deviation once more: D = 3 u R.  The squares round by 26 u of their sum, those that
    are taken off again, of at most three places at each end of a row, by 8 u each, the deviations by 2 u, rstd's own
    steps by 4 u: 42 u of rstd with the half that the root leaves."""
    n = 40
    x, dy, w, b = torch.zeros(n, c, device="cuda"), randn(n, c, seed=130), 1 + 0.3 * randn(c, seed=131), 0.3 * randn(c, seed=132)
    rows = torch.arange(n, device="cuda")
    size = 1.0 + rows[:, None].double() / 64
    x[rows, rows % 8] = size[:, 0].float()
    table = torch.empty(n, 2 * c + 1, device="cuda")
    for silu in (False, True):
        act = "silu" if silu else None
        ref = Rows64(x, w, b, 1e-5, silu)
        ref.D = 42 * U + 3 * U * size * ref.rstd
        ref.E = 3 * U * size * ref.rstd + 42 * U * ref.xhat.abs()
        ref.E_z = ref.w.abs() * ref.E + U * ref.z.abs()
        assert_close(nm.layer_norm(x, w, b, activation=act), *ref.forward(), "y", norm=c < 1000)
        nm.layer_norm(x, w, b, activation=act, out=table[:, c:2 * c])  # (rows that start differently in x and out)
        assert_close(table[:, c:2 * c], *ref.forward(), "out", norm=c < 1000)
        grads = nm.layer_norm_grad(x, dy, w, b, activation=act)
        for name, value, (want, bound) in zip(("dx", "dw", "db"), grads, ref.backward(dy)):
            assert_close(value, want, bound, name, norm=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", [16, 97, 340, 513, 2048, 8191, 8192])
def test_values_up_to_1e18_in_rows_of_any_width(nm, dtype, c):
    x, dy, w, b = inputs(11, c, F32, F32, seed=141)
    x = (x / x.abs().max() * 0.99e18).to(dtype)
    x[3] = torch.where(torch.arange(c, device="cuda") % 2 == 0, 0.99e18, -0.99e18).to(dtype)  # as far apart as they go
    for eps in (0.0, 1e-5):
        check_rows(nm, x, dy.to(dtype), w, b, eps=eps, norm=False)
        check_rows(nm, x, (dy * 1e18).to(dtype), w, b, eps=eps, silu=True, norm=False)
    small = (x.double() * 1e-36).to(dtype)  # (deviations of 1e-18)
    check_rows(nm, small, (dy * 1e-18).to(dtype), w, b, eps=0.0, norm=False)


@pytest.mark.parametrize("n,c", [(1, 64), (50, 64), (33, 97), (7, 2048)])
def test_silu_where_its_result_nears_the_least_normal_number(nm, n, c):
    """z from -92 to -80: exp(-z) passes fp32's range from -88.7 on, z exp(z) stays a normal number to -91.9.  A relative error:
    that of the bounds above, of z with a slope of z exp(z) below 1.02 of the value for a unit of z, and half a unit of the
    subnormal numbers in the sigmoid."""
    x, dy, w, _ = inputs(n, c, F32, F32, seed=142)
    w = 0.01 * w
    b = torch.linspace(-91.8, -80.0, c, device="cuda")
    ref = Rows64(x, w, b, 1e-5, True)
    y = nm.layer_norm(x, w, b, activation="silu")
    want = ref.z * ref.sig
    rel = 1.02 * ref.E_z + (12 + 2.4 * ref.z.abs()) * U
    assert not ((y.double() - want).abs() > want.abs() * rel + (ref.z.abs() + 1) * 2.0**-149).any()
    assert (want.abs() > 2.0**-126).sum() > 0.9 * want.numel()
    dy = dy.abs() + 0.5
    slope = ref.sig * (1 + ref.z * (1 - ref.sig))
    db = nm.layer_norm_grad(x, dy, w, b, activation="silu")[2].double()
    want = (dy.double() * slope).sum(0)
    bound = (dy.double() * slope.abs() * (1.02 * ref.E_z + (16 + 10 * ref.z.abs()) * U)).sum(0)
    bound = bound + (dy.double() * (ref.z.abs() + 2) * 2.0**-149).sum(0) + (n + 16) * U * (dy.double() * slope.abs()).sum(0)
    assert not ((db - want).abs() > bound).any()


@pytest.mark.parametrize("size", [4, 3000, 2_000_003])
@pytest.mark.parametrize("ins,outs", [(F32, F32), (BF16, F32), (F32, BF16), (BF16, BF16)])
def test_clipping_of_norms_past_fp32(nm, size, ins, outs):
    """Factors below fp32's normal numbers, down to 1e-62: the product rounds twice (the factor's rest, the product), and below
    2^-123 by two units of 2^-149."""
    grads = [(randn(size, seed=143).clamp(-3, 3) * 1e38).to(ins), torch.full((4,), 3e38, device="cuda").to(ins), randn(50, seed=144, dtype=ins)]
    grads[0][0] = -3e38
    for max_norm in (1e20, 1.0, 1e-3, 1e-7, 1e-20):
        out = [torch.empty_like(g, dtype=outs) for g in grads]
        norm = nm.clip_grads(grads, max_norm, out=out)
        assert float(norm) == float(norm64(grads).float())
        for got, want in zip(out, clipped64(grads, max_norm)):
            bound = 2.01 * U * want.abs() + 2.0**-148 + (2.0**-8 * want.abs() + 2.0**-133 if outs == BF16 else 0.0)
            assert not ((got.double() - want).abs() > bound).any()
        assert (out[0] != 0).any()
    if ins == outs:
        want = clipped64(grads, 1e-7)
        nm.clip_grads(grads, 1e-7)
        for got, expected in zip(grads, want):
            bound = 2.01 * U * expected.abs() + 2.0**-148 + (2.0**-8 * expected.abs() + 2.0**-133 if outs == BF16 else 0.0)
            assert not ((got.double() - expected).abs() > bound).any()


@pytest.mark.parametrize("dtype,n,c", [(F32, 3_000_001, 63), (BF16, 1_500_003, 127), (F32, 1_300_001, 126)])
def test_sums_of_one_sign_over_many_rows_that_start_anywhere(nm, dtype, n, c):
    """Widths whose rows take twice the lanes where they start anywhere: still at most 256 rows a lane."""
    x, _, w, b = inputs(n, c, dtype, F32, seed=145)
    dy = (randn(n, c, seed=146).abs_() + 0.5).to(dtype)
    check_rows(nm, x, dy, w, b)
