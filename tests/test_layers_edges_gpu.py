"""Borders of ops.group_norm, ops.linear and ops.grouped_linear."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from distributed_machine_learning_amd import ops  # noqa: E402
from test_layers_gpu import ACTS, BF, FP, HF, act64, close, gen, normal, over  # noqa: E402

INF, NAN = float("inf"), float("nan")


def same(got, want):
    """Equal, with NaN equal to NaN."""
    return torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


# ---------------------------------------------------------------- infinities in the activations


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", (BF, HF))
@pytest.mark.parametrize("m, k, n", [(4, 100, 70), (40, 512, 64), (300, 136, 264), (300, 137, 130), (1000, 256, 512)])
def test_products_at_infinity(m, k, n, act, dtype):
    """Sums of +inf, -inf and NaN give what the formula gives for them: +inf stays +inf in every activation."""
    g = gen(m + n)
    x, w = normal(g, m, k).to(dtype), (normal(g, n, k).abs() + 0.1).to(dtype)
    ends = torch.tensor([3, m], device="cuda")
    for out in (dtype, FP):
        want = ops.linear(x, w, act=act, out_dtype=out)
        bad = x.clone()
        bad[1, k - 1], bad[2, 0], bad[3, k // 2] = INF, -INF, NAN
        want[1:4] = act64(torch.tensor([INF, -INF, NAN], device="cuda", dtype=torch.double), act)[:, None].to(out)
        assert same(ops.linear(bad, w, act=act, out_dtype=out), want)
        assert same(ops.grouped_linear(bad, torch.stack([w, w]), ends, act=act, out_dtype=out), want)
        r = torch.full((m, n), INF, device="cuda", dtype=out)  # +inf + -inf is NaN
        want[:] = act64(torch.tensor(INF, device="cuda", dtype=torch.double), act)
        want[2:4] = NAN
        assert same(ops.linear(bad, w, act=act, residual=r, act_last=True, out_dtype=out), want)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", (BF, HF, FP))
@pytest.mark.parametrize("shape, groups", [((2, 50, 64), 8), ((1, 9000, 96), 3), ((2, 20, 35), 5), ((2, 9, 3), 3)])
def test_group_norm_at_infinity(shape, groups, act, dtype):
    """An infinity that the affine map brings."""
    g = gen(5)
    x, b = normal(g, *shape).to(dtype), normal(g, shape[-1])
    want = ops.group_norm(x, groups, None, b, act=act)
    b[1], b[2] = INF, -INF
    want[..., 1:3] = act64(b[1:3].double(), act).to(dtype)
    assert same(ops.group_norm(x, groups, None, b, act=act), want)


# ---------------------------------------------------------------- group norm


@pytest.mark.parametrize("dtype", (BF, FP))
@pytest.mark.parametrize("shape, groups", [((2, 50, 72), 8), ((2, 35, 35, 288), 32), ((2, 20, 100), 10), ((3, 20, 55), 5),
                                           ((2, 40, 40), 8), ((2, 30, 39), 3), ((2, 9000, 99), 9), ((1, 9000, 130), 10),
                                           ((2, 20, 14), 2), ((2, 20, 21), 7)])
@pytest.mark.parametrize("bad", (NAN, INF, -INF))
def test_group_norm_keeps_bad_values_to_groups_that_cut_vectors(shape, groups, bad, dtype):
    """Groups whose width is no multiple of a vector's: each in turn, at its first and last channel."""
    g = gen(13)
    clean = normal(g, *shape).to(dtype)
    want = ops.group_norm(clean, groups, act="gelu")
    assert not want.isnan().any()
    cg = shape[-1] // groups
    n = shape[0] - 1
    for k in range(groups):
        for c in (k * cg, (k + 1) * cg - 1):
            x = clean.clone()
            x[n].reshape(-1, shape[-1])[7, c] = bad
            y = ops.group_norm(x, groups, act="gelu")
            hit = torch.zeros(shape, dtype=torch.bool, device="cuda")
            hit[n, ..., k * cg:(k + 1) * cg] = True
            assert y[hit].isnan().all() and torch.equal(y[~hit], want[~hit]), (k, c)


@pytest.mark.parametrize("positions, c", [(2 ** 23, 256), (2 ** 26, 64), (2 ** 25 + 4097, 80), (2 ** 29, 64)])
def test_group_norm_of_groups_beyond_31_bits(positions, c):
    """One group of 2^31 to 2^35 values, half of them 1 and half 3: mean 2, variance 1, so -1 and 1 in bf16 (0.999995
    rounds to it, and stays there for errors of the statistics up to 2^-10)."""
    row = torch.tensor([1.0, 3.0], device="cuda", dtype=BF).repeat(c // 2)
    y = ops.group_norm(row.expand(1, positions, c), 1)
    for part in y[0].split(2 ** 22):
        assert (part == row - 2).all()
    del y, part
    torch.cuda.empty_cache()


def steps_of_chunks():
    """Additions in a row, at most, on the way from a value to its group's mean or sum of squares where a sample goes
    through chunks: a thread's own (8 rows, as many values each as a vector has where that is one statistic: 64), the
    workgroup's merge (with a statistic per vector NT / 64 = 16 a lane, with one per channel 8 times that, but then a
    thread has 8 values: so 8 + 128), 6 levels over lanes; then, by 8 lanes, fewer than 2048 chunks, or with `join` far
    fewer: 256 + 6; a dozen for the products, the division and the last subtraction."""
    return 8 + 128 + 6 + 256 + 6 + 12


def tight64(x, groups, d, eps=1e-5):
    """(y, err) of the norm without its affine map: fp32 statistics over chains of d operations, centred and merged.

    A mean is off by at most e = d 2^-24 mean|x|. A sum of squared distances from it, merged as M2 + n (mu_i - mu)^2,
    is off by d 2^-24 of itself and, for means that are off by e each, by 2 (2e) sd + (2e)^2 a value."""
    n, c = x.shape[0], x.shape[-1]
    xd = x.double().reshape(n, -1, groups, c // groups)
    count, u = xd.shape[1] * xd.shape[3], 2.0 ** -24
    mu = over(xd, torch.sum) / count
    var = over((xd - mu).square(), torch.sum) / count
    e = d * u * over(xd.abs(), torch.sum) / count
    rel = (d * u * var + 4 * e * var.sqrt() + 4 * e ** 2) / (var + eps) / 2 + 4 * u
    rs = 1 / torch.sqrt(var + eps)
    y = (xd - mu) * rs
    return y.reshape(x.shape), ((e + u * (xd - mu).abs()) * rs * (1 + rel) + y.abs() * (rel + 4 * u)).reshape(x.shape)


def drifting(drift, positions, device):
    """Levels along a sample, [positions, 1]."""
    p = torch.arange(positions, device=device) / positions
    return {"ramp": 16 * p - 8, "steps": 10 * (p * 7).floor().remainder(3) - 10, "level": 50 + 0 * p}[drift][:, None]


@pytest.mark.parametrize("drift", ("ramp", "steps", "level"))
@pytest.mark.parametrize("dtype", (BF, FP))
@pytest.mark.parametrize("shape, groups", [((1, 9000, 96), 3), ((1, 20000, 64), 8), ((2, 70001, 256), 32), ((1, 300000, 64), 8),
                                           ((1, 400000, 35), 5), ((1, 150000, 520), 520), ((1, 30011, 99), 9)])
def test_group_norm_merges_chunks_of_different_levels(shape, groups, dtype, drift):
    """The levels drift along the sample, so that the distances between the chunks' means are most of the variance."""
    g = gen(31)
    x = (normal(g, *shape) + drifting(drift, shape[1], "cuda")).to(dtype)
    y, err = tight64(x, groups, steps_of_chunks())
    assert err.max() < 0.02  # a lost chunk or a missing term between them is far more
    close(ops.group_norm(x, groups), y, err)


@pytest.mark.parametrize("dtype", (BF, HF, FP))
@pytest.mark.parametrize("shape, groups", [((1, 2 ** 24, 3), 1), ((1, 2 ** 25, 3), 1), ((2, 500000, 2), 1), ((1, 300000, 3), 3),
                                           ((1, 2000, 8200), 1)])
def test_group_norm_of_odd_widths_at_a_level(shape, groups, dtype):
    """What no slab fits (fewer channels than a vector, groups of more than 1024 vectors), far from 0: sums in 64 bits, so
    that mean and variance are off by their roundings to fp32 and no more, whatever the number of values."""
    x = (100 + normal(gen(37), *shape)).to(dtype)
    y, err = tight64(x, groups, 4)
    close(ops.group_norm(x, groups), y, err)


# ---------------------------------------------------------------- products


@pytest.mark.parametrize("out_dtype", (BF, FP))
@pytest.mark.parametrize("m, k, n", [(300, 6144, 346), (64, 8192, 1024), (150, 4728, 1730), (256, 4096, 4096), (563, 4584, 2515),
                                     (1024, 512, 2048), (200, 2001, 600), (9, 4096, 264)])
def test_products_into_their_residual(m, k, n, out_dtype):
    """Sums that several sets of waves hold, each finishing its own part: the residual is read where they then write."""
    g = gen(m + n)
    x, w, b = normal(g, m, k).to(BF), (normal(g, n, k) * k ** -0.5).to(BF), normal(g, n)
    ends, pair = torch.tensor([m // 3, m], device="cuda"), torch.stack([w, -w])
    r = normal(g, m, n).to(out_dtype)
    kw = {"act": "gelu", "out_dtype": out_dtype}
    want = ops.linear(x, w, b, residual=r, **kw), ops.grouped_linear(x, pair, ends, residual=r, act_last=True, **kw)
    for _ in range(3):
        y, z = r.clone(), r.clone()
        ops.linear(x, w, b, residual=y, out=y, **kw)
        ops.grouped_linear(x, pair, ends, residual=z, act_last=True, out=z, **kw)
        assert torch.equal(y, want[0]) and torch.equal(z, want[1])


def test_linear_of_more_than_2_30_rows():
    """More rows than 2^32 threads hold in tiles of 64."""
    row = torch.tensor([1.0, -2.0, 3.0, 0.0, 0.5, 0.0, 0.0, 4.0], device="cuda", dtype=BF)
    m = 2 ** 30 + 77
    y = ops.linear(row.expand(m, 8), torch.ones(1, 8, device="cuda", dtype=BF))
    assert y.shape == (m, 1)
    for part in y.split(2 ** 28):
        assert (part == 6.5).all()


def test_out_that_a_backward_pass_saved():
    """Writing into a tensor that some graph saved is seen by autograd, as with any in-place operation."""
    g = gen(41)
    x, w = normal(g, 8, 16).to(BF), normal(g, 16, 16).to(BF)
    ends = torch.tensor([3, 8], device="cuda")
    for call in (lambda t: ops.group_norm(x, 4, out=t), lambda t: ops.linear(x, w, out=t),
                 lambda t: ops.linear(x, w, residual=t, out=t), lambda t: ops.grouped_linear(x, torch.stack([w, w]), ends, out=t)):
        leaf, saved = torch.ones(8, 16, device="cuda", dtype=BF, requires_grad=True), normal(g, 8, 16).to(BF)
        y = (leaf * saved).sum()
        with torch.no_grad():
            call(saved)
        with pytest.raises(RuntimeError, match="inplace"):
            y.backward()
    with torch.inference_mode():
        out = torch.empty(8, 16, device="cuda", dtype=BF)
        assert torch.equal(ops.linear(x, w, out=out), ops.linear(x, w))
