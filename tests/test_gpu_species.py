"""Species operators on the GPU against their definitions in 64 bits.

Bounds (u = 2^-24, the unit roundoff of fp32):

* grouping, the embedding lookup and the 8-bit checkpoint are exact: the
  definition's own fp32 arithmetic, each operation rounded once, compared for
  equality;
* a sum of n products in fp32, in any order, is within (n + 16) 2u of the sum
  of the products' magnitudes (2u: the tensor core truncates where it adds;
  16: the roundings of the split operands, the partial sums and alpha);
  over a whole result those errors are random, so its relative error in the
  2-norm also stays below 2^-19, far below what one dropped bf16 term or a
  TF32 product would leave (2^-16, 2^-12);
* a bf16 result (8-bit significand) adds half a unit in its last place, at most
  2^-8 of its magnitude.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def sp():
    from mace_mlx_b200 import species

    return species


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=gen(seed), device="cuda").to(dtype)


def draw_species(n, g, seed, pad=0.0, only=None):
    """int32 species in [0, g), ``pad`` of them outside (below and above); ``only``: the groups used."""
    z = torch.randint(0, g, (n,), generator=gen(seed), device="cuda", dtype=torch.int32)
    if only is not None:
        z = torch.tensor(only, dtype=torch.int32, device="cuda")[z % len(only)]
    if pad:
        r = torch.rand(n, generator=gen(seed + 1), device="cuda")
        z = torch.where(r < pad / 2, -1, torch.where(r < pad, g + 3, z))
    return z


def valid(z, g):
    return (z >= 0) & (z < g)


def groups_of(z, g):
    """The grouping by its definition."""
    key = torch.where(valid(z, g), z, g).cpu()
    order = torch.tensor(sorted(range(len(key)), key=lambda i: int(key[i])), dtype=torch.int32)
    offsets = torch.tensor([int((key < v).sum()) for v in range(g + 1)], dtype=torch.int32)
    return order.cuda(), offsets.cuda()


def assert_sum(got, want, mass, n, what=""):
    """got (fp32 or bf16) against the 64-bit sum ``want`` of n products of total magnitude ``mass``."""
    got64 = got.double()
    bound = (n + 16) * 2 * U * mass
    if got.dtype == torch.bfloat16:
        bound = bound * (1 + 2.0**-8) + 2.0**-8 * want.abs()
    bad = (got64 - want).abs() > bound
    assert not bad.any(), f"{what}: {int(bad.sum())} values off, worst {float((got64 - want).abs().max()):.3e}"
    norm = float(want.norm())
    rel = float((got64 - want).norm())
    limit = 2.0**-19 if got.dtype == torch.float32 else 2.0**-8 + 2.0**-19
    assert rel <= limit * norm, f"{what}: relative error {rel / norm:.3e}"


# ------------------------------------------------------------------ grouping
@pytest.mark.parametrize("n", [0, 1, 2, 31, 33, 1000, 4096, 4097, 20011])
@pytest.mark.parametrize("g", [1, 2, 89, 511, 1023, 1024, 7921])
def test_grouping_is_the_stable_order(sp, n, g):
    z = draw_species(n, g, n + g, pad=0.1 if n > 1 else 0.0)
    got = sp.group_species(z, g)
    order = torch.argsort(torch.where(valid(z, g), z, g).cpu().long(), stable=True).to(torch.int32)
    counts = torch.bincount(z[valid(z, g)].cpu().long(), minlength=g)
    assert torch.equal(got.order.cpu(), order)
    assert torch.equal(got.offsets.cpu(), torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).int())


@pytest.mark.parametrize("z", [[], [-1, -1, -1], [2] * 5000, [5, 4, 3, 2, 1, 0], [2**31 - 1, -(2**31), 0, 6, 5]])
def test_grouping_of_special_lists(sp, z):
    z = torch.tensor(z, dtype=torch.int32, device="cuda")
    order, offsets = groups_of(z, 6)
    got = sp.group_species(z, 6)
    assert torch.equal(got.order, order) and torch.equal(got.offsets, offsets)


def test_grouping_of_many_rows(sp):
    n, g = 1_500_001, 300_007  # two counting passes, most groups with a few rows
    z = draw_species(n, g, 3, pad=0.01)
    got = sp.group_species(z, g)
    key = torch.where(valid(z, g), z, g)
    key, order = torch.sort(key, stable=True)
    assert torch.equal(got.order, order.int())
    assert torch.equal(got.offsets, torch.searchsorted(key, torch.arange(g + 1, device="cuda", dtype=torch.int32),
                                                       out_int32=True))


@pytest.mark.parametrize("n,g,used", [
    (30_001, 4095, 4095),    # the last group count of a 12-bit pass
    (30_001, 4096, 4096),    # the first of 13 bits
    (50_001, 8191, 8191),    # the last count of one pass
    (50_001, 8192, 8192),    # the first of two
    (50_001, 8191, 3),       # equal digits in every warp where they are expected to differ
    (50_001, 5000, 1),
    (9, 8191, 8191),         # fewer rows than a warp
    (10_000_019, 8191, 8191),  # the longest share of a CTA
    (10_000_019, 2, 1),
])  # fmt: skip
def test_grouping_at_the_limits_of_a_pass(sp, n, g, used):
    z = draw_species(n, g, n, pad=0.05, only=None if used == g else list(range(g - used, g)))
    got = sp.group_species(z, g)
    key, order = torch.sort(torch.where(valid(z, g), z, g), stable=True)
    assert torch.equal(got.order, order.int())
    assert torch.equal(got.offsets, torch.searchsorted(key, torch.arange(g + 1, device="cuda", dtype=torch.int32),
                                                       out_int32=True))


# ----------------------------------------------------------------- embedding
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,c", [(1, 1), (7, 3), (1000, 128), (333, 97), (65, 256), (130, 300), (2000, 8)])
def test_embedding_lookup(sp, dtype, n, c):
    g, scale = 11, 0.3
    table = randn(g, c, seed=1, dtype=dtype)
    z = draw_species(n, g, 2, pad=0.2)
    ok = valid(z, g)
    want = torch.where(ok[:, None], table.float()[z.clamp(0, g - 1).long()] * torch.tensor(scale), 0.0).to(dtype)
    assert torch.equal(sp.species_embedding(table, z, scale=scale), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c,pitch", [(64, 64), (33, 33), (33, 40)])
def test_embedding_of_padding_is_zero_whatever_the_scale(sp, dtype, c, pitch):
    n, g = 500, 7
    table, z = randn(g, c, seed=3, dtype=dtype), draw_species(n, g, 5, pad=0.3)
    for scale in (float("inf"), float("nan"), -2.0):
        out = torch.ones(n, pitch, dtype=dtype, device="cuda")[:, :c]
        got = sp.species_embedding(table, z, scale=scale, out=out)
        assert not got[~valid(z, g)].any()
        assert torch.equal(got[valid(z, g)].isfinite(), torch.full_like(got[valid(z, g)], scale == -2.0, dtype=torch.bool))


def test_embedding_of_strided_tables_and_outputs(sp):
    g, n = 5, 257
    z = draw_species(n, g, 4, pad=0.1)
    for c, off in [(64, 0), (64, 1), (33, 2)]:
        wide = randn(g, 200, seed=5)
        node = torch.full((n, 150), 7.0, device="cuda")
        out = node[:, off:off + c]
        got = sp.species_embedding(wide[:, off:off + c], z, scale=2.0, out=out)
        assert got.data_ptr() == out.data_ptr()
        want = torch.where(valid(z, g)[:, None], wide[z.clamp(0, g - 1).long(), off:off + c] * 2.0, 0.0)
        assert torch.equal(out, want)
        assert (node[:, :off] == 7.0).all() and (node[:, off + c:] == 7.0).all()
    one = randn(1, 16, seed=6).expand(g, 16)  # a broadcast table
    assert torch.equal(sp.species_embedding(one, z.clamp(0, g - 1)), one[z.clamp(0, g - 1).long()])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,g,c,pad", [(0, 3, 8, 0), (1, 1, 1, 0), (1, 4, 128, 0), (1000, 89, 128, 0.1), (5000, 4, 97, 0),
                                       (3001, 1, 64, 0.05), (700, 300, 33, 0.5), (40, 7, 16, 1.0),
                                       (9000, 2, 256, 0.01), (2000, 1500, 300, 0.1)])
def test_embedding_gradient(sp, dtype, n, g, c, pad):
    scale = 0.37
    z = draw_species(n, g, 7, pad=pad)
    dy = randn(n, c, seed=8, dtype=dtype)
    dy[~valid(z, g)] = float("nan")  # padding rows are never read
    got = sp.species_embedding_grad(dy, sp.group_species(z, g), scale=scale)
    want = torch.zeros(g, c, dtype=torch.float64, device="cuda")
    mass = torch.zeros_like(want)
    at = z[valid(z, g)].long()
    s = float(torch.tensor(scale))  # the fp32 scale the kernel gets
    want.index_add_(0, at, dy[valid(z, g)].double() * s)
    mass.index_add_(0, at, dy[valid(z, g)].double().abs() * s)
    assert got.shape == (g, c) and got.dtype == dtype
    assert_sum(got, want, mass, n)


def test_embedding_gradient_of_long_groups_and_strides(sp):
    n, g, c = 300_011, 3, 40
    z = draw_species(n, g, 9, only=[0, 2])
    dy = randn(n, 3 * c, seed=10)[:, c + 1:2 * c + 1]
    got = sp.species_embedding_grad(dy, sp.group_species(z, g))
    want = torch.zeros(g, c, dtype=torch.float64, device="cuda").index_add_(0, z.long(), dy.double())
    mass = torch.zeros(g, c, dtype=torch.float64, device="cuda").index_add_(0, z.long(), dy.double().abs())
    # blocks of rows are summed apart and joined: far fewer than n roundings meet in one sum
    assert_sum(got, want, mass, n)
    assert torch.equal(got[1], torch.zeros(c, device="cuda"))
    again = sp.species_embedding_grad(dy, sp.group_species(z, g))
    assert torch.equal(got, again)
    # every row the same: a broadcast gradient
    ones = torch.ones(1, c, device="cuda").expand(n, c)
    counts = torch.bincount(z.long(), minlength=g).float()
    assert torch.equal(sp.species_embedding_grad(ones, sp.group_species(z, g)), counts[:, None].expand(g, c))


@pytest.mark.parametrize("c", [8, 17])
def test_embedding_gradient_of_very_long_groups(sp, c):
    """The error stays where it is as the rows grow: no fp32 sum takes more than a stated number of rows."""
    n = 100_000_000
    groups = sp.SpeciesGroups(torch.arange(n, dtype=torch.int32, device="cuda"),
                              torch.tensor([0, n], dtype=torch.int32, device="cuda"))
    dy = randn(n, c, seed=15)
    want = torch.zeros(c, dtype=torch.float64, device="cuda")
    mass = torch.zeros_like(want)
    for part in dy.split(1 << 23):
        want += part.double().sum(0)
        mass += part.double().abs().sum(0)
    assert_sum(sp.species_embedding_grad(dy, groups)[0], want, mass, n)


# -------------------------------------------------------------------- linear
def linear64(x, w, z, alpha):
    """Output and product magnitudes of the map in 64 bits; x (n, d, k)."""
    g = w.shape[0]
    a = float(torch.tensor(alpha))
    y = torch.zeros(*x.shape[:-1], w.shape[2], dtype=torch.float64, device="cuda")
    mass = torch.zeros_like(y)
    for i in range(g):
        rows = (z == i).nonzero().flatten()
        if rows.numel():
            xi, wi = x[rows].double(), w[i].double()
            y[rows] = a * (xi @ wi)
            mass[rows] = abs(a) * (xi.abs() @ wi.abs())
    return y, mass


def wgrad64(x, dy, z, g, alpha):
    a = float(torch.tensor(alpha))
    dw = torch.zeros(g, x.shape[-1], dy.shape[-1], dtype=torch.float64, device="cuda")
    mass = torch.zeros_like(dw)
    for i in range(g):
        rows = (z == i).nonzero().flatten()
        if rows.numel():
            xi, yi = x[rows].double().flatten(0, 1), dy[rows].double().flatten(0, 1)
            dw[i] = a * (xi.T @ yi)
            mass[i] = abs(a) * (xi.abs().T @ yi.abs())
    return dw, mass


LINEAR = [
    # n, d, k, m, g, pad
    (1, 1, 1, 1, 1, 0.0), (1, 3, 128, 128, 4, 0.0), (2, 1, 16, 16, 89, 0.0), (5, 7, 9, 5, 3, 0.4),
    (127, 1, 128, 128, 1, 0.0), (128, 1, 128, 128, 1, 0.0), (129, 1, 128, 128, 2, 0.0), (1000, 3, 128, 128, 89, 0.0),
    (1000, 1, 96, 96, 4, 0.05), (333, 5, 97, 61, 10, 0.1), (400, 3, 65, 130, 6, 0.02), (300, 1, 129, 33, 5, 0.0),
    (257, 3, 256, 192, 3, 0.1), (100, 1, 300, 257, 2, 0.0), (64, 1, 64, 256, 7, 1.0), (700, 1, 48, 16, 500, 0.1),
    (210, 1, 520, 24, 2, 0.0), (4000, 1, 8, 8, 3, 0.0), (513, 7, 40, 72, 512, 0.3),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d,k,m,g,pad", LINEAR)
def test_linear_and_its_gradients(sp, dtype, n, d, k, m, g, pad):
    alpha = 1.0 / k**0.5
    z = draw_species(n, g, 11, pad=pad)
    x, w, dy = randn(n, d, k, seed=12, dtype=dtype), randn(g, k, m, seed=13, dtype=dtype), \
        randn(n, d, m, seed=14, dtype=dtype)
    out = ~valid(z, g)
    x[out], dy[out] = float("nan"), float("inf")  # padding rows are never read
    groups = sp.group_species(z, g)
    y, mass = linear64(x, w, z, alpha)
    assert_sum(sp.species_linear(x, w, groups, alpha=alpha), y, mass, k, "forward")
    dx, mass = linear64(dy, w.transpose(1, 2), z, alpha)
    dw, wmass = wgrad64(x, dy, z, g, alpha)
    got_x, got_w = sp.species_linear_grad(x, dy, w, groups, alpha=alpha)
    assert_sum(got_x, dx, mass, m, "input gradient")
    assert_sum(got_w, dw, wmass, n * d, "weight gradient")
    assert torch.equal(got_x, sp.species_linear(dy, w, groups, alpha=alpha, transpose=True))
    assert torch.equal(got_w, sp.species_linear_grad_weight(x, dy, groups, alpha=alpha))  # same order of sums
    assert sp.error_flag() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mix", ["one", "two of many", "none"])
def test_linear_over_many_tiles(sp, dtype, mix):
    """More row tiles than SMs, groups that start and end inside a CTA's share."""
    n, d, k, m, g = 30_011, 3, 64, 48, 20
    z = {"one": torch.full((n,), 13, dtype=torch.int32, device="cuda"), "two of many": draw_species(n, g, 20, only=[3, 17]),
         "none": torch.full((n,), -1, dtype=torch.int32, device="cuda")}[mix]
    x, w, dy = randn(n, d, k, seed=21, dtype=dtype), randn(g, k, m, seed=22, dtype=dtype), \
        randn(n, d, m, seed=23, dtype=dtype)
    groups = sp.group_species(z, g)
    y, mass = linear64(x, w, z, 0.5)
    assert_sum(sp.species_linear(x, w, groups, alpha=0.5), y, mass, k)
    dw, mass = wgrad64(x, dy, z, g, 0.5)
    got = sp.species_linear_grad_weight(x, dy, groups, alpha=0.5)
    assert_sum(got, dw, mass, n * d)
    assert torch.equal(got, sp.species_linear_grad_weight(x, dy, groups, alpha=0.5))


def test_weight_gradient_of_very_long_groups(sp):
    """The error stays where it is as the rows grow: no fp32 sum takes more than a stated number of steps."""
    n, k = 300_000_000, 8
    groups = sp.SpeciesGroups(torch.arange(n, dtype=torch.int32, device="cuda"),
                              torch.tensor([0, n], dtype=torch.int32, device="cuda"))
    x, dy = randn(n, k, seed=27), randn(1, k, seed=28)
    want = torch.zeros(k, dtype=torch.float64, device="cuda")
    mass = torch.zeros_like(want)
    for part in x.split(1 << 24):
        want += part.double().sum(0)
        mass += part.double().abs().sum(0)
    dw = sp.species_linear_grad_weight(x, dy.expand(n, k), groups)[0]  # (one row of dy, shared)
    assert_sum(dw, want[:, None] * dy.double(), mass[:, None] * dy.double().abs(), n)


def test_weight_gradient_of_the_widest_matrices(sp):
    """65 536 tiles of a matrix, and a group without rows."""
    n, k, g = 3, 32768, 2
    z = torch.zeros(n, dtype=torch.int32, device="cuda")
    x, dy = randn(n, k, seed=25, dtype=torch.bfloat16), randn(n, k, seed=26, dtype=torch.bfloat16)
    junk = torch.full((g, k, k), 7.0, dtype=torch.bfloat16, device="cuda")
    del junk  # (what the result is likely to be made in)
    dw = sp.species_linear_grad_weight(x, dy, sp.group_species(z, g))
    assert not dw[1].any()
    for c in range(0, k, 4096):
        part = x[:, c:c + 4096].double()
        assert_sum(dw[0, c:c + 4096], part.T @ dy.double(), part.abs().T @ dy.double().abs(), n)


def _views(x):
    """x (n, d, k) in other layouts of the same values."""
    n, d, k = x.shape
    wide = torch.zeros(n, (d + 2) * k, dtype=x.dtype, device="cuda")
    slot = wide[:, k:(d + 1) * k].view(n, d, k)  # a slot of a node-feature table
    slot.copy_(x)
    odd = torch.zeros(n * d * k + 3, dtype=x.dtype, device="cuda")[3:].view(n, d, k)  # not 16-byte aligned
    odd.copy_(x)
    turned = torch.zeros(d, n, k, dtype=x.dtype, device="cuda").transpose(0, 1)  # component-major
    turned.copy_(x)
    loose = torch.zeros(n, d, k + 1, dtype=x.dtype, device="cuda")[..., :k]  # an odd row pitch
    loose.copy_(x)
    return {"slot": slot, "odd": odd, "turned": turned, "loose": loose}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,m", [(128, 128), (40, 24), (33, 7)])
def test_linear_layouts_agree(sp, dtype, k, m):
    """Strides and alignment change how rows are fetched, never the result."""
    n, d, g = 301, 3, 4
    z = draw_species(n, g, 30, pad=0.1)
    x, w, dy = randn(n, d, k, seed=31, dtype=dtype), randn(g, k, m, seed=32, dtype=dtype), \
        randn(n, d, m, seed=33, dtype=dtype)
    groups = sp.group_species(z, g)
    y = sp.species_linear(x, w, groups)
    dw = sp.species_linear_grad_weight(x, dy, groups)
    ck = sp.checkpoint_rows(x)
    xs, ys, outs = _views(x), _views(dy), _views(torch.zeros_like(y))
    for name in xs:
        assert torch.equal(sp.species_linear(xs[name], w, groups), y), name
        assert torch.equal(sp.species_linear_grad_weight(xs[name], ys[name], groups), dw), name
        assert torch.equal(sp.species_linear(x, w, groups, out=outs[name]), y), name
        assert torch.equal(outs[name], y), name
        again = sp.checkpoint_rows(xs[name])
        assert torch.equal(again.q, ck.q) and torch.equal(again.scale, ck.scale), name
    # rows shared by every atom (node stride 0)
    shared = x[:1].expand(n, d, k)
    assert torch.equal(sp.species_linear(shared, w, groups), sp.species_linear(shared.contiguous(), w, groups))
    # (n, k) rows are (n, 1, k) rows
    assert torch.equal(sp.species_linear(x[:, 0], w, groups), sp.species_linear(x[:, :1].contiguous(), w, groups)[:, 0])


def test_linear_writes_only_its_slot(sp):
    n, d, k, m, g = 200, 3, 64, 32, 3
    z = draw_species(n, g, 40, pad=0.2)
    x, w = randn(n, d, k, seed=41), randn(g, k, m, seed=42)
    table = torch.full((n, 5 * m), 3.0, device="cuda")
    sp.species_linear(x, w, sp.group_species(z, g), out=table[:, m:4 * m].view(n, d, m))
    assert (table[:, :m] == 3.0).all() and (table[:, 4 * m:] == 3.0).all()
    assert torch.equal(table[~valid(z, g), m:4 * m], torch.zeros(int((~valid(z, g)).sum()), 3 * m, device="cuda"))


def test_rows_with_infinities_and_nan_stay_apart(sp):
    n, k, m, g = 300, 128, 64, 2
    z = draw_species(n, g, 50)
    x, w = randn(n, 1, k, seed=51), randn(g, k, m, seed=52)
    clean = sp.species_linear(x, w, sp.group_species(z, g))
    x[17, 0, 5], x[200, 0, 127] = float("inf"), float("nan")
    got = sp.species_linear(x, w, sp.group_species(z, g))
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[[17, 200]] = False
    assert torch.equal(got[rest], clean[rest])
    assert not got[17].isfinite().any() and got[200].isnan().all()


def assert_ieee(got, want, mass, n, what=""):
    """Infinities and NaN where the 64-bit result has them (rounded to the type), and the other values within bounds."""
    want = torch.where(want.to(got.dtype).isinf(), want.sign() * torch.inf, want)
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN at other places"
    odd = ~want.isfinite()
    assert torch.equal(got[odd & ~want.isnan()].double(), want[odd & ~want.isnan()]), f"{what}: other infinities"
    assert odd.any() and not odd.all()
    assert_sum(got.where(~odd, 0.0), want.where(~odd, 0.0), mass.where(~odd, 0.0), n, what)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d,k,m,g", [(300, 1, 128, 64, 2), (300, 3, 33, 70, 5), (9001, 3, 150, 40, 3)])
def test_infinities_enter_sums_as_in_the_definition(sp, dtype, n, d, k, m, g):
    z = draw_species(n, g, 53, pad=0.1)
    z[:8] = torch.arange(8, device="cuda") % g
    x, w, dy = randn(n, d, k, seed=54, dtype=dtype), randn(g, k, m, seed=55, dtype=dtype), \
        randn(n, d, m, seed=56, dtype=dtype)
    groups = sp.group_species(z, g)

    def both(inf_x, inf_w, inf_dy, what):
        y, mass = linear64(x, w, z, 0.5)
        assert_ieee(sp.species_linear(x, w, groups, alpha=0.5), y, mass, k, what + ": forward")
        dx, mass = linear64(dy, w.transpose(1, 2), z, 0.5)
        dw, wmass = wgrad64(x, dy, z, g, 0.5)
        got_x, got_w = sp.species_linear_grad(x, dy, w, groups, alpha=0.5)
        if inf_w or inf_dy:
            assert_ieee(got_x, dx, mass, m, what + ": input gradient")
        if inf_x or inf_dy:
            assert_ieee(got_w, dw, wmass, n * d, what + ": weight gradient")

    x[3, 0, 5], x[4, 0, 7], x[4, 0, 8] = torch.inf, -torch.inf, -torch.inf
    both(True, False, False, "rows of x")
    x[5, 0, 2] = torch.nan
    both(True, False, False, "a NaN beside them")
    dy[6, 0, 3], dy[2, 0, 4] = -torch.inf, torch.inf
    both(True, False, True, "rows of dy")
    w[1, 2, 6] = torch.inf
    both(True, True, True, "a matrix")
    assert sp.error_flag() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_checkpoint_whose_scale_times_the_gradient_overflows(sp, dtype):
    """q = 0 adds nothing, the others what the restored values give."""
    n, k, m, g = 5000, 130, 48, 3
    z = draw_species(n, g, 93)
    x, dy = randn(n, 1, k, seed=94), randn(n, 1, m, seed=95, dtype=dtype)
    x[7], dy[7] = x[7] * 1e25, 1e20
    x[7, 0, ::3] = 0.0
    ck = sp.checkpoint_rows(x)
    values = sp.restore_rows(ck).double()
    dw, mass = wgrad64(values, dy, z, g, 1.0)
    got = sp.species_linear_grad_weight(ck, dy, sp.group_species(z, g))
    assert_ieee(got, dw, mass, n)
    assert got[z[7], ::3].isfinite().all()


def test_large_and_small_magnitudes(sp):
    """The split operands keep fp32's range: nothing overflows or is lost near its ends."""
    n, k, m = 130, 64, 32
    z = torch.zeros(n, dtype=torch.int32, device="cuda")
    groups = sp.group_species(z, 1)
    for sx, sw in [(1e30, 1e-30), (1e-25, 1e25), (3e38 / 8, 1e-3), (1e-12, 1e-12)]:
        x = (randn(n, 1, k, seed=60).clamp(-4, 4) * sx)
        w = (randn(1, k, m, seed=61).clamp(-4, 4) * sw)
        y, mass = linear64(x, w, z, 1.0)
        assert_sum(sp.species_linear(x, w, groups), y, mass, k, f"{sx} {sw}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sx,sw,alpha", [(1e30, 1e-12, 1e-30), (1e-25, 1e25, 1e20), (1e-12, 1e20, 1e27), (1e4, 1e-30, 1e-9)])
def test_alpha_meets_the_sum(sp, dtype, sx, sw, alpha):
    """alpha x W is in range where alpha W (or alpha x) is not."""
    n, k, m, g = 130, 64, 32, 2
    z = draw_species(n, g, 65)
    groups = sp.group_species(z, g)
    x, dy = (randn(n, 1, k, seed=66) * sx).to(dtype), (randn(n, 1, m, seed=67) * sx).to(dtype)
    w = (randn(g, k, m, seed=68) * sw).to(dtype)
    y, mass = linear64(x, w, z, alpha)
    assert_sum(sp.species_linear(x, w, groups, alpha=alpha), y, mass, k, "forward")
    dx, mass = linear64(dy, w.transpose(1, 2), z, alpha)
    assert_sum(sp.species_linear(dy, w, groups, alpha=alpha, transpose=True), dx, mass, m, "input gradient")


def test_linear_past_32_bit_offsets(sp):
    """Rows whose element offsets pass 2^31."""
    n, k, m, g = 1000, 64, 32, 2
    table = torch.empty(n, 3_000_000, dtype=torch.bfloat16, device="cuda")  # 3e9 elements, 6 GB
    x = table[:, -k:]
    x.copy_(randn(n, k, seed=70, dtype=torch.bfloat16))
    z = draw_species(n, g, 71)
    w = randn(g, k, m, seed=72, dtype=torch.bfloat16)
    groups = sp.group_species(z, g)
    dense = x.contiguous()
    assert torch.equal(sp.species_linear(x, w, groups), sp.species_linear(dense, w, groups))
    dy = randn(n, m, seed=73, dtype=torch.bfloat16)
    assert torch.equal(sp.species_linear_grad_weight(x, dy, groups), sp.species_linear_grad_weight(dense, dy, groups))
    assert torch.equal(sp.species_embedding_grad(x, groups), sp.species_embedding_grad(dense, groups))
    assert torch.equal(sp.checkpoint_rows(x).q, sp.checkpoint_rows(dense).q)
    out = table[:, 2_000_000:2_000_000 + m]
    assert torch.equal(sp.species_linear(dense, w, groups, out=out), sp.species_linear(dense, w, groups))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,m", [(64, 32), (33, 21)])
def test_unaligned_rows_past_32_bit_offsets(sp, dtype, k, m):
    """Rows at any address and results whose element offsets pass 2^32, in every operator."""
    n, g = 500, 3
    pitch = 9_000_000
    table = torch.empty(n, pitch, dtype=dtype, device="cuda")  # 4.5e9 elements, 9 or 18 GB
    z = draw_species(n, g, 74, pad=0.1)
    groups = sp.group_species(z, g)
    x, dy, w = randn(n, k, seed=75, dtype=dtype), randn(n, m, seed=76, dtype=dtype), randn(g, k, m, seed=77, dtype=dtype)
    far_x, far_dy = table[:, -k - 1:-1], table[:, pitch // 2 + 1:pitch // 2 + 1 + m]
    far_x.copy_(x), far_dy.copy_(dy)
    y, mass = linear64(x[:, None], w, z, 1.0)
    far = table[:, pitch - 2000 + 1:pitch - 2000 + 1 + m]
    for source in (x, far_x):
        table[:, pitch - 2000:pitch - 2000 + m + 2] = 7.0
        assert_sum(sp.species_linear(source, w, groups, out=far)[:, None], y, mass, k, "forward")
        assert (table[:, pitch - 2000] == 7.0).all() and (table[:, pitch - 2000 + 1 + m] == 7.0).all()
    dw, mass = wgrad64(x[:, None], dy[:, None], z, g, 1.0)
    assert_sum(sp.species_linear_grad_weight(far_x, far_dy, groups), dw, mass, n, "weight gradient")
    ck = sp.checkpoint_rows(x)
    far_ck = sp.checkpoint_rows(far_x)
    assert torch.equal(far_ck.q, ck.q) and torch.equal(far_ck.scale, ck.scale)
    assert torch.equal(sp.species_linear_grad_weight(ck, far_dy, groups), sp.species_linear_grad_weight(ck, dy, groups))
    ok = valid(z, g)
    want = torch.zeros(g, k, dtype=torch.float64, device="cuda").index_add_(0, z[ok].long(), x[ok].double())
    mass = torch.zeros_like(want).index_add_(0, z[ok].long(), x[ok].double().abs())
    assert_sum(sp.species_embedding_grad(far_x, groups), want, mass, n, "embedding gradient")
    assert torch.equal(sp.species_embedding(w[0], z, out=far), sp.species_embedding(w[0], z))
    assert sp.error_flag() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,m", [(64, 128), (40, 24), (33, 7)])
def test_weights_at_any_address(sp, dtype, k, m):
    n, d, g = 400, 3, 5
    z = draw_species(n, g, 34, pad=0.1)
    x, dy = randn(n, d, k, seed=35, dtype=dtype), randn(n, d, m, seed=36, dtype=dtype)
    groups = sp.group_species(z, g)
    for off in (1, 3):
        w = randn(g * k * m + off, seed=37, dtype=dtype)[off:].view(g, k, m)
        assert w.is_contiguous() and w.data_ptr() % 16
        y, mass = linear64(x, w, z, 0.3)
        assert_sum(sp.species_linear(x, w, groups, alpha=0.3), y, mass, k, "forward")
        dx, mass = linear64(dy, w.transpose(1, 2), z, 0.3)
        assert_sum(sp.species_linear_grad(x, dy, w, groups, alpha=0.3)[0], dx, mass, m, "input gradient")


# ---------------------------------------------------------------- checkpoint
def quantise(x):
    """The checkpoint's definition in fp32 (each operation rounded once)."""
    n, d, c = x.shape
    nb = -(-c // 128)
    xb = torch.nn.functional.pad(x.float(), (0, nb * 128 - c)).view(n, d, nb, 128)
    scale = xb.abs().amax(-1) * torch.tensor(1.0 / 127.0)
    q = torch.round(xb / torch.where(scale > 0, scale, 1.0)[..., None]).clamp(-127, 127)
    return q.to(torch.int8).view(n, d, nb * 128)[..., :c], scale


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d,c", [(0, 1, 8), (1, 1, 1), (3, 5, 7), (100, 3, 128), (77, 1, 129), (65, 4, 96), (10, 1, 300),
                                   (1000, 1, 256), (33, 7, 64)])
def test_checkpoint_is_its_definition(sp, dtype, n, d, c):
    x = randn(n, d, c, seed=80, dtype=dtype)
    if n > 2:
        x[1] = 0.0  # a block of zeros
        x[2] *= 1e-30
    ck = sp.checkpoint_rows(x)
    q, scale = quantise(x)
    assert torch.equal(ck.q, q) and torch.equal(ck.scale, scale)
    values = q.float() * scale.repeat_interleave(128, dim=-1)[..., :c]
    for out in DTYPES:
        assert torch.equal(sp.restore_rows(ck, out), values.to(out))
    off = (sp.restore_rows(ck).double() - x.double()).abs()
    assert (off <= 0.5 * (1 + 2.0**-16) * scale.repeat_interleave(128, dim=-1)[..., :c].double()).all()


def test_checkpoint_of_extreme_rows(sp):
    x = torch.zeros(6, 1, 128, device="cuda")
    x[0, 0, 3] = float("nan")
    x[1, 0, 3] = float("inf")
    x[2, 0, :] = 3.4e38
    x[3, 0, 5] = 1e-44  # the scale underflows to zero
    x[4, 0, 5] = 3e-43  # a subnormal scale: the quotient passes 127
    x[5, 0, 100] = -1.0
    ck = sp.checkpoint_rows(x)
    v = sp.restore_rows(ck)
    assert v[0].isnan().all() and v[1].isnan().all()
    assert torch.equal(ck.q[2], torch.full_like(ck.q[2], 127)) and v[2].isfinite().all()
    assert (v[3] == 0).all() and int(ck.q[4].max()) <= 127 and v[4].isfinite().all()
    assert int(ck.q[5, 0, 100]) == -127 and abs(float(v[5, 0, 100]) + 1.0) <= 2 * U


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d,k,m,g,pad", [c for c in LINEAR if c[0] * c[1] > 1])
def test_weight_gradient_from_a_checkpoint(sp, dtype, n, d, k, m, g, pad):
    z = draw_species(n, g, 90, pad=pad)
    x, dy = randn(n, d, k, seed=91), randn(n, d, m, seed=92, dtype=dtype)
    x[~valid(z, g)] = float("nan")
    dy[~valid(z, g)] = float("nan")
    ck = sp.checkpoint_rows(x)
    values = ck.q.double() * ck.scale.double().repeat_interleave(128, dim=-1)[..., :k]
    dw, mass = wgrad64(values, dy, z, g, 0.7)
    assert_sum(sp.species_linear_grad_weight(ck, dy, sp.group_species(z, g), alpha=0.7), dw, mass, n * d)
    assert sp.error_flag() == 0


# ------------------------------------------------------- gradients as a user has them
@pytest.mark.parametrize("checkpoint", [False, True])
def test_autograd_matches_differences(sp, checkpoint):
    """The maps are linear in each argument, so a difference over any step is the derivative."""
    n, d, k, m, g = 150, 3, 48, 40, 5
    z = draw_species(n, g, 100, pad=0.1)
    groups = sp.group_species(z, g)
    x, w, v = randn(n, d, k, seed=101), randn(g, k, m, seed=102), randn(n, d, m, seed=103)
    x.requires_grad_(), w.requires_grad_()
    y = sp.species_linear(x, w, groups, alpha=0.2, checkpoint=checkpoint)
    (y * v).sum().backward()
    with torch.no_grad():
        for t, step, slack in ((x, randn(n, d, k, seed=104), 0.0), (w, randn(g, k, m, seed=105), 1.0)):
            moved = (x + step, w) if t is x else (x, w + step)
            y1 = sp.species_linear(*moved, groups, alpha=0.2).double()
            diff = float(((y1 - y.double()) * v.double()).sum())
            dot = float((t.grad.double() * step.double()).sum())
            mass = float(((y1.abs() + y.double().abs()) * v.double().abs()).sum())
            # y and y1 carry (k + 16) 2u each; the checkpoint moves x by half a scale (max / 254) at most
            bound = (k + 16) * 2 * U * mass * 4
            if checkpoint and slack:
                top = x.detach().double().abs().amax(-1, keepdim=True).expand_as(x) / 254
                bound += float(linear64(top, step.abs(), z, 0.2)[0].mul(v.double().abs()).sum())
            assert abs(diff - dot) <= bound, (diff, dot, bound)


@pytest.mark.parametrize("dtype", DTYPES)
def test_autograd_through_a_checkpoint_is_that_of_the_restored_rows(sp, dtype):
    """The weight gradient against its formula and against differences of the map on the rows that the checkpoint holds."""
    n, d, k, m, g = 150, 3, 48, 40, 5
    z = draw_species(n, g, 106, pad=0.1)
    groups = sp.group_species(z, g)
    x, w, v = randn(n, d, k, seed=107, dtype=dtype), randn(g, k, m, seed=108, dtype=dtype), randn(n, d, m, seed=109, dtype=dtype)
    x.requires_grad_(), w.requires_grad_()
    sp.species_linear(x, w, groups, alpha=0.2, checkpoint=True).backward(v)
    kept = sp.restore_rows(sp.checkpoint_rows(x.detach())).double()
    dw, mass = wgrad64(kept, v, z, g, 0.2)
    assert_sum(w.grad, dw, mass, n * d, "weight gradient")
    dx, mass = linear64(v, w.detach().transpose(1, 2), z, 0.2)
    assert_sum(x.grad, dx, mass, m, "input gradient")
    if dtype == torch.float32:
        # the map is linear in w: the difference over any step, in 64 bits, is the gradient's product with the step
        step = randn(g, k, m, seed=110)
        diff = float(((linear64(kept, w.detach() + step, z, 0.2)[0] - linear64(kept, w.detach(), z, 0.2)[0]) * v.double()).sum())
        dot = float((w.grad.double() * step.double()).sum())
        # every entry of the gradient within assert_sum's bound, and w + step rounded once
        bound = float(((n * d + 16) * 2 * U * wgrad64(kept, v, z, g, 0.2)[1] * step.abs().double()).sum())
        bound += float((U * (w.detach() + step).abs().double() * wgrad64(kept, v, z, g, 0.2)[1]).sum())
        assert abs(diff - dot) <= bound < 0.05 * abs(diff), (diff, dot, bound)


def test_embedding_autograd_and_expanded_gradients(sp):
    n, g, c = 500, 7, 24
    z = draw_species(n, g, 110, pad=0.1)
    table = randn(g, c, seed=111).requires_grad_()
    sp.species_embedding(table, z, scale=0.5).sum().backward()  # the gradient arrives expanded from one value
    counts = torch.stack([(z == i).sum() for i in range(g)]).float()
    assert torch.equal(table.grad, 0.5 * counts[:, None].expand(g, c))
    table.grad = None
    groups = sp.group_species(z, g)
    sp.species_embedding(table, z, scale=0.5, groups=groups).sum().backward()
    assert torch.equal(table.grad, 0.5 * counts[:, None].expand(g, c))
    # weights shared by several uses add up, and a frozen argument gets none
    x, w = randn(n, 1, c, seed=112), randn(g, c, c, seed=113).requires_grad_()
    (sp.species_linear(x, w, groups) + sp.species_linear(x, w, groups)).sum().backward()
    once = sp.species_linear_grad_weight(x, torch.ones(n, 1, c, device="cuda"), groups)
    assert torch.equal(w.grad, once + once) and x.grad is None


# ------------------------------------------------------------ streams, graphs
def test_other_streams_and_cuda_graphs(sp):
    n, d, k, m, g = 2000, 3, 64, 64, 9
    z = draw_species(n, g, 120, pad=0.05)
    x, w, dy = randn(n, d, k, seed=121), randn(g, k, m, seed=122), randn(n, d, m, seed=123)

    def step():
        groups = sp.group_species(z, g)
        ck = sp.checkpoint_rows(x)
        emb = sp.species_embedding(w[:, 0], z)
        return [groups.order, groups.offsets, sp.species_linear(x, w, groups), *sp.species_linear_grad(x, dy, w, groups),
                sp.species_linear_grad_weight(ck, dy, groups), emb, sp.species_embedding_grad(emb, groups),
                sp.restore_rows(ck)]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    x.mul_(2.0)
    want = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_calls_from_two_host_threads(sp):
    import threading

    n, d, k, g = 3000, 3, 64, 6

    def work(seed):
        z = draw_species(n, g, seed, pad=0.05)
        x, w = randn(n, d, k, seed=seed + 1), randn(g, k, k, seed=seed + 2)
        groups = sp.group_species(z, g)
        y = sp.species_linear(x, w, groups)
        return [*groups, y, *sp.species_linear_grad(x, y, w, groups),
                sp.species_linear_grad_weight(sp.checkpoint_rows(x), y, groups), sp.species_embedding_grad(y[:, 0], groups)]

    want = {seed: work(seed) for seed in (150, 160)}
    torch.cuda.synchronize()
    got, errors = {}, []

    def thread(seed):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[seed] = work(seed)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=thread, args=(seed,)) for seed in want]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for seed, values in want.items():
        assert all(torch.equal(a, b) for a, b in zip(got[seed], values, strict=True))


# ------------------------------------------------------------------ refusals
def test_refusals(sp):
    z = torch.zeros(8, dtype=torch.int32, device="cuda")
    groups = sp.group_species(z, 2)
    x, w = torch.zeros(8, 3, 16, device="cuda"), torch.zeros(2, 16, 4, device="cuda")
    dy = torch.zeros(8, 3, 4, device="cuda")
    ck = sp.checkpoint_rows(x)
    bad = [
        lambda: sp.group_species(z.long(), 2), lambda: sp.group_species(z[::2], 2), lambda: sp.group_species(z, 0),
        lambda: sp.group_species(z, sp.MAX_INDEX + 1), lambda: sp.group_species(z.view(2, 4), 2),
        lambda: sp.species_embedding(w[:, :, 0], z),  # channels not contiguous
        lambda: sp.species_embedding(w, z), lambda: sp.species_embedding(w[:, 0].half(), z),
        lambda: sp.species_embedding(w[:, 0], z.cpu()), lambda: sp.species_embedding(w[:, 0], z, out=x[:, 0]),
        lambda: sp.species_embedding_grad(x, groups), lambda: sp.species_embedding_grad(x[:4, 0], groups),
        lambda: sp.species_linear(x.transpose(1, 2), w, groups), lambda: sp.species_linear(x.bfloat16(), w, groups),
        lambda: sp.species_linear(x.double(), w.double(), groups), lambda: sp.species_linear(x[:7], w, groups),
        lambda: sp.species_linear(x[..., :15], w, groups), lambda: sp.species_linear(x, w[:1], groups),
        lambda: sp.species_linear(x, w.transpose(1, 2), groups), lambda: sp.species_linear(x[0, 0], w, groups),
        lambda: sp.species_linear(x, w, groups, out=dy[:4]), lambda: sp.species_linear(x, w, groups, out=dy.bfloat16()),
        lambda: sp.species_linear(x, w, groups, out=dy[:1].expand(8, 3, 4)),
        lambda: sp.species_linear(x, w, groups, out=torch.zeros(8, 3, 4)),
        lambda: sp.species_linear(x.cpu(), w, groups), lambda: sp.species_linear(x, w.cpu(), groups),
        lambda: sp.species_linear(x, w, sp.SpeciesGroups(groups.order.cpu(), groups.offsets)),
        lambda: sp.species_linear(x, w, sp.SpeciesGroups(groups.order, groups.offsets.long())),
        lambda: sp.species_linear(x, w, sp.SpeciesGroups(groups.order, groups.offsets[:1])),
        lambda: sp.species_linear(x, torch.zeros(513, 16, 4, device="cuda"), sp.group_species(z, 513)),
        lambda: sp.species_linear_grad_weight(x[:4], dy, groups), lambda: sp.species_linear_grad_weight(x, dy[:, :2], groups),
        lambda: sp.species_linear_grad_weight(x.bfloat16(), dy, groups),
        lambda: sp.species_linear_grad_weight(sp.RowCheckpoint(ck.q, ck.scale[:, :2]), dy, groups),
        lambda: sp.species_linear_grad_weight(sp.RowCheckpoint(ck.q.int(), ck.scale), dy, groups),
        lambda: sp.species_linear_grad_weight(x, dy, sp.group_species(z, 513)),
        lambda: sp.checkpoint_rows(x.half()), lambda: sp.checkpoint_rows(x[..., ::2]), lambda: sp.checkpoint_rows(x[0, 0]),
        lambda: sp.checkpoint_rows(torch.zeros(1, 2000, 1, device="cuda")),
        lambda: sp.restore_rows(ck, torch.float16), lambda: sp.restore_rows(sp.RowCheckpoint(ck.q, ck.scale.double())),
        lambda: sp.species_linear(x.requires_grad_(), w, groups, transpose=True),
        lambda: sp.species_embedding(torch.zeros(3, 4, device="cuda", requires_grad=True), z, groups=groups),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")
    with pytest.raises(TypeError):
        sp.group_species([0, 1], 2)
    torch.cuda.synchronize()
    assert sp.error_flag() == 0


def test_a_grouping_of_other_rows_is_refused_in_the_forward(sp):
    z = torch.zeros(8, dtype=torch.int32, device="cuda")
    table = torch.zeros(2, 4, device="cuda", requires_grad=True)
    groups = sp.group_species(z, 2)
    for bad in (sp.group_species(z[:5], 2), sp.group_species(z, 3), sp.SpeciesGroups(groups.order.cpu(), groups.offsets),
                sp.SpeciesGroups(groups.order.long(), groups.offsets)):
        with pytest.raises(ValueError):
            sp.species_embedding(table, z, groups=bad)
    assert sp.species_embedding(table, z, groups=groups).requires_grad


@pytest.mark.parametrize("requires_grad", [False, True])
def test_tangents_are_refused(sp, requires_grad):
    """A forward-mode tangent would be dropped: every entry that takes features refuses it."""
    from torch.autograd import forward_ad

    z = torch.zeros(8, dtype=torch.int32, device="cuda")
    groups = sp.group_species(z, 2)
    plain = {"x": torch.zeros(8, 3, 16), "w": torch.zeros(2, 16, 4), "dy": torch.zeros(8, 3, 4), "t": torch.zeros(2, 16)}
    plain = {k: v.cuda() for k, v in plain.items()}
    ck = sp.checkpoint_rows(plain["x"])
    with forward_ad.dual_level():
        dual = {k: forward_ad.make_dual(v.clone().requires_grad_(requires_grad), torch.ones_like(v))
                for k, v in plain.items()}
        scale = forward_ad.make_dual(ck.scale, torch.ones_like(ck.scale))
        for i, call in enumerate((
            lambda: sp.species_linear(dual["x"], plain["w"], groups), lambda: sp.species_linear(plain["x"], dual["w"], groups),
            lambda: sp.species_linear_grad(dual["x"], plain["dy"], plain["w"], groups),
            lambda: sp.species_linear_grad(plain["x"], dual["dy"], plain["w"], groups),
            lambda: sp.species_linear_grad(plain["x"], plain["dy"], dual["w"], groups),
            lambda: sp.species_linear_grad_weight(dual["x"], plain["dy"], groups),
            lambda: sp.species_linear_grad_weight(plain["x"], dual["dy"], groups),
            lambda: sp.species_embedding(dual["t"], z), lambda: sp.species_embedding_grad(dual["x"][:, 0], groups),
            lambda: sp.checkpoint_rows(dual["x"]), lambda: sp.restore_rows(sp.RowCheckpoint(ck.q, scale)),
        )):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
                pytest.fail(f"call {i} was accepted")
        sp.species_linear(plain["x"], plain["w"], groups)  # without a tangent: as ever


def test_groupings_that_are_not_permutations_stay_in_bounds(sp):
    """order and offsets come from the caller: whatever they hold, no row outside the tensors is touched."""
    n, k, g = 300, 32, 3
    x, w, dy = randn(n, 1, k, seed=130), randn(g, k, k, seed=131), randn(n, 1, k, seed=132)
    order = torch.randint(-5, n + 5, (n,), generator=gen(133), device="cuda", dtype=torch.int32)
    for offsets in ([0, 500, -3, 2000], [200, 100, 50, 0], [-7, -7, -7, -7], [10, 20, 30, 40]):
        bad = sp.SpeciesGroups(order, torch.tensor(offsets, dtype=torch.int32, device="cuda"))
        sp.species_linear(x, w, bad)
        sp.species_linear_grad_weight(x, dy, bad)
        sp.species_linear_grad_weight(sp.checkpoint_rows(x), dy, bad)
        sp.species_embedding_grad(dy[:, 0], bad)
    torch.cuda.synchronize()
    assert sp.error_flag() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_calls_in_a_row_on_buffers_used_again(sp, dtype):
    """Each call reads what the call before it has just written to memory that earlier calls had read."""
    n, g, c = 700, 5, 64
    tables, w = randn(6, g, c, seed=140, dtype=dtype), randn(g, c, c, seed=141, dtype=dtype)
    lists = [draw_species(n, g, 142 + k, pad=0.1) for k in range(6)]

    def chain(k, rows, y):
        groups = sp.group_species(lists[k], g)
        sp.species_embedding(tables[k], lists[k], out=rows)
        sp.species_linear(rows, w, groups, out=y)
        ck = sp.checkpoint_rows(y)
        return [*groups, y.clone(), sp.restore_rows(ck), sp.species_embedding_grad(y, groups),
                sp.species_linear_grad_weight(ck, y, groups)]

    want = []
    for k in range(6):
        rows, y = torch.empty(n, c, dtype=dtype, device="cuda"), torch.empty(n, c, dtype=dtype, device="cuda")
        want.append(chain(k, rows, y))
        torch.cuda.synchronize()
    rows, y = torch.empty(n, c, dtype=dtype, device="cuda"), torch.empty(n, c, dtype=dtype, device="cuda")
    for _ in range(10):
        got = [chain(k, rows, y) for k in range(6)]
        for a, b in zip(sum(got, []), sum(want, []), strict=True):
            assert torch.equal(a, b)


# ------------------------------------------------------------- ends and repeats
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", [1, 8, 33, 61, 64, 128, 129, 250])
def test_embedding_gradient_at_group_ends(sp, dtype, c):
    # groups that end with, before and after the 8, 16 or 32 rows read at a time, empty ones between them, one over many
    # warps' shares, padding last
    sizes = [0, 1, 31, 32, 33, 0, 0, 64, 7, 8, 9, 16, 0, 1, 1, 1, 4096, 32, 128, 0, 5, 27, 0]
    z = torch.cat([torch.full((k,), i, dtype=torch.int32) for i, k in enumerate(sizes)] + [torch.full((40,), -1, dtype=torch.int32)])
    z = z[torch.randperm(len(z), generator=torch.Generator().manual_seed(c))].cuda()
    g = len(sizes)
    dy = randn(len(z), c, seed=c, dtype=dtype)
    dy[z < 0] = float("nan")
    got = sp.species_embedding_grad(dy, sp.group_species(z, g))
    ok = z >= 0
    want = torch.zeros(g, c, device="cuda", dtype=torch.float64).index_add_(0, z[ok].long(), dy[ok].double())
    mass = torch.zeros_like(want).index_add_(0, z[ok].long(), dy[ok].double().abs())
    assert_sum(got, want, mass, max(sizes))


@pytest.mark.parametrize("dtype,k,m", [(torch.float32, 128, 128), (torch.float32, 97, 61), (torch.bfloat16, 96, 96),
                                       (torch.bfloat16, 97, 61)])
def test_equal_calls_give_equal_bits(sp, dtype, k, m):
    n, d, g = 30_011, 3, 7
    z = draw_species(n, g, 4, pad=0.01)
    x, dy, w = randn(n, d, k, seed=1, dtype=dtype), randn(n, d, m, seed=2, dtype=dtype), randn(g, k, m, seed=3, dtype=dtype)

    def everything():
        groups = sp.group_species(z, g)
        ck = sp.checkpoint_rows(x)
        return [*groups, sp.species_linear(x, w, groups), *sp.species_linear_grad(x, dy, w, groups),
                sp.species_linear_grad_weight(ck, dy, groups), sp.species_embedding_grad(x[:, 0], groups), *ck]

    first = everything()
    for _ in range(5):
        for a, b in zip(first, everything(), strict=True):
            assert torch.equal(a, b)


# ------------------------------------------------------------------- together
@pytest.fixture(scope="module")
def head_example():
    import importlib.util
    import pathlib

    path = pathlib.Path(__file__).resolve().parents[1] / "examples" / "species_head.py"
    spec = importlib.util.spec_from_file_location("species_head", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_head_on_model_features_has_the_plain_gradients(sp, head_example):
    n = 6
    h, z, graph = head_example.frozen_features(n, seed=1)
    groups = sp.group_species(z, 4)
    head = head_example.SpeciesHead(4, h.shape[2], 48, gen(5))
    energy = head(h, z, groups, graph, n)
    energy.square().sum().backward()
    # the same in 64 bits; the weight gradient of what the 8-bit rows stand for, by exchanging them behind the forward
    p = {k: v.detach().double().requires_grad_() for k, v in head.named_parameters()}
    kept = sp.restore_rows(sp.checkpoint_rows(h)).double()

    def plain(rows):
        y = torch.einsum("ndk,nkm->ndm", rows, p["weight"][z.long()]) * h.shape[2]**-0.5
        return y

    y = plain(h.double())
    y = y + (plain(kept) - plain(kept).detach()) - (y - y.detach())  # the value of h, the gradient of `kept`
    y0 = y[:, 0] + p["table"][z.long()]
    atom = torch.tanh(y0) @ p["scalar"] + y[:, 1:].square().sum(1) @ p["vector"]
    want = torch.zeros(n, device="cuda", dtype=torch.float64).index_add(0, graph, atom) / graph.bincount(minlength=n)
    want.square().sum().backward()
    # fp32 sums of a few thousand terms each way: 2^-16 of the largest value covers their roundings and torch's
    assert (energy.double() - want).abs().max() <= 2.0**-16 * want.abs().max()
    for name, q in p.items():
        got = getattr(head, name).grad.double()
        assert (got - q.grad).abs().max() <= 2.0**-16 * q.grad.abs().max(), name


def test_head_example_learns(head_example):
    losses = head_example.train(n_structures=8, steps=60)
    assert losses[-1] < 0.2 * losses[0]
