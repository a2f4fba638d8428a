"""The operators on device tensors against their definitions in 64 bits (device_op_forms)."""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import device_op_forms as forms  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0**-24  # half a step of fp32 relative to the value


@pytest.fixture(scope="module")
def ops():
    from distributed_kge_poplar_b200 import device_ops

    return device_ops


def gen(seed):
    return torch.Generator().manual_seed(seed)


def cuda(t):
    return None if t is None else t.cuda()


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ---------------------------------------------------------------------------
# Log probabilities.
#
# A term 2^d has d = (x - reference) s2 with three roundings (s2, difference, product) and an ex2 right to 2^-22: relative error
# (2 |d| + 4) 2^-23 at most.  Each thread adds its columns up one by one, then 9 rounds of joining rescale and add.  So log S is
# off by (2 D + 4 + 4) 2^-23 + (C / 512 + 24) 2^-24 with D the largest |d| that counts (terms below 2^-30 of the sum do not: 30),
# and log p by that, its own three roundings and the result's.


def log_tolerance(cols, value):
    return U * (2 * (2 * 30 + 8) + cols / 512 + 24 + 12 * value.abs() + 8)


def check_log_probs(got, want, cols, entropy_scale=1.0):
    for name in ("log_prob", "log_sum", "best_log_prob"):
        g, w = getattr(got, name).cpu().double(), want[name]
        assert g.shape == w.shape
        infinite = torch.isinf(w)
        assert torch.equal(torch.isnan(g), torch.isnan(w)), name
        assert torch.equal(g[infinite], w[infinite]), name
        fine = torch.isfinite(w)
        # a log sum is a logit more: its own rounding is relative to it, and the logits' products are
        tol = log_tolerance(cols, w[fine])
        assert torch.all((g[fine] - w[fine]).abs() <= tol), (name, ((g[fine] - w[fine]).abs() / tol).max())
    g, w = got.entropy.cpu().double(), want["entropy"]
    assert torch.equal(torch.isnan(g), torch.isnan(w))
    fine = torch.isfinite(w)
    # T / S: terms of |d| up to 30 with the terms' errors, sums of both
    tol = log_tolerance(cols, w[fine]) * (1 + w[fine])
    assert torch.all((g[fine] - w[fine]).abs() <= tol), ((g[fine] - w[fine]).abs() / tol).max()
    assert torch.equal(got.best_index.cpu(), want["best_index"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,n_best", [(1, 1, 1), (3, 1, 4), (2, 7, 10), (5, 63, 5), (1, 1387, 10), (4, 2049, 128), (7, 4097, 100), (2, 40_003, 17), (3, 100_001, 128),
                                              (40, 20_001, 30), (20, 90_003, 100), (200, 9000, 100), (400, 5000, 128),
                                              (600, 4003, 128), (600, 8003, 5), (592, 12_001, 0), (100, 140_001, 0)])
def test_log_probs(ops, rows, cols, n_best, dtype):
    g = gen(rows * 1000 + cols)
    x = (torch.randn(rows, cols, generator=g) * 3).to(dtype)
    target = torch.randint(cols, (rows,), generator=g, dtype=torch.int32)
    got = ops.log_probs(x.cuda(), target.cuda(), scale=0.7, n_best=n_best)
    check_log_probs(got, forms.log_probs(x, target, scale=0.7, n_best=n_best), cols)


@pytest.mark.parametrize("dtype", TYPES)
def test_log_probs_of_strided_rows_with_masks_and_counts(ops, dtype):
    rows, cols = 37, 1003
    g = gen(3)
    wide = (torch.randn(rows, cols + 22, generator=g) * 4).to(dtype)
    allowed = torch.rand(rows, cols + 9, generator=g) > 0.3
    allowed[5] = False
    count = torch.randint(1, cols + 1, (rows,), generator=g, dtype=torch.int32)
    count[7], count[8], count[9] = 0, cols, cols + 50  # more than there are: all
    target = torch.randint(cols, (rows,), generator=g, dtype=torch.int32)
    target[:5] = torch.tensor([-1, cols, cols + 5, -(2**31), 2**31 - 1])  # none of these is a column
    for lead in (0, 1, 3):
        x, mask = wide[:, lead : lead + cols], allowed[:, lead : lead + cols]
        hidden = torch.where(mask, x, torch.tensor([math.nan, math.inf, -math.inf, 1e30])[torch.arange(cols) % 4].to(dtype))
        device = torch.empty_like(wide).cuda()
        device[:, lead : lead + cols] = hidden.cuda()
        got = ops.log_probs(device[:, lead : lead + cols], target.cuda(), mask=allowed.cuda()[:, lead : lead + cols], count=count.cuda(), n_best=33)
        check_log_probs(got, forms.log_probs(x, target, mask, count, n_best=33), cols)
    for r in (5, 7):  # nothing is left of these rows
        assert got.log_sum[r] == -math.inf and got.entropy[r] == 0 and torch.all(got.best_index[r] == -1) and torch.all(got.best_log_prob[r] == -math.inf)
    one = allowed[11:12, :cols]
    x = wide[:, :cols].contiguous()
    got = ops.log_probs(x.cuda(), target.cuda(), mask=one.cuda().expand(rows, cols), n_best=3)
    check_log_probs(got, forms.log_probs(x, target, one.expand(rows, cols), n_best=3), cols)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,n_best", [(1, 300_007, 128), (3, 150_000, 0), (5, 600_001, 20)])
def test_log_probs_of_rows_in_parts(ops, rows, cols, n_best, dtype):
    """Few long rows: each is cut into parts.  Counts end inside a part, at one's start and before all but the first."""
    g = gen(cols)
    x = (torch.randn(rows, cols, generator=g) * 3).to(dtype)
    x[rows - 1, ::2] = 2.0  # equal scores in every part
    target = torch.randint(cols, (rows,), generator=g, dtype=torch.int32)
    count = torch.tensor([cols, 70_000, 5, cols // 2, cols - 1][:rows], dtype=torch.int32)
    for c in (None, count):
        got = ops.log_probs(x.cuda(), target.cuda(), count=cuda(c), n_best=n_best)
        check_log_probs(got, forms.log_probs(x, target, count=c, n_best=n_best), cols)
        again = ops.log_probs(x.cuda(), target.cuda(), count=cuda(c), n_best=n_best)
        assert torch.equal(got.log_sum, again.log_sum) and torch.equal(got.entropy, again.entropy)


@pytest.mark.parametrize("rows,cols", [(3, 200), (400, 5000), (200, 9000), (20, 60_000)])
def test_log_probs_of_rows_of_equal_scores(ops, rows, cols):
    """Every size of block: all columns reach any threshold, and the lowest are listed."""
    x = torch.zeros(rows, cols)
    x[1, cols // 2 :] = 2.0
    got = ops.log_probs(x.cuda(), n_best=100)
    want = torch.arange(100, dtype=torch.int32).repeat(rows, 1)
    want[1] += cols // 2
    assert torch.equal(got.best_index.cpu(), want)
    check_log_probs(got, forms.log_probs(x, None, n_best=100), cols)


def test_log_probs_of_equal_scores_in_many_parts(ops):
    """More columns than any list of candidates holds share the best score: the lowest columns are listed."""
    x = torch.zeros(2, 400_000)
    x[1, 100::7] = 1.0
    got = ops.log_probs(x.cuda(), n_best=128)
    assert torch.equal(got.best_index[0].cpu(), torch.arange(128, dtype=torch.int32))
    assert torch.equal(got.best_index[1].cpu(), torch.arange(128, dtype=torch.int32) * 7 + 100)


@pytest.mark.parametrize("scale", [1e-6, 1e-3, 30.0])
@pytest.mark.parametrize("dtype", TYPES)
def test_log_probs_of_small_and_large_scales(ops, dtype, scale):
    """-inf stays out of the sums where a step of the scale reaches from any score to any other."""
    g = gen(2)
    x = (torch.randn(4, 3000, generator=g) * 2).to(dtype)
    x[1, ::2] = -math.inf
    x[2] = torch.finfo(dtype).min
    x[2, 5:50] = -math.inf
    x[3, 7] = torch.finfo(dtype).min
    want = forms.log_probs(x, torch.full((4,), 2, dtype=torch.int32), scale=scale, n_best=5)
    got = ops.log_probs(x.cuda(), torch.full((4,), 2, dtype=torch.int32).cuda(), scale=scale, n_best=5)
    assert torch.equal(got.best_index.cpu(), want["best_index"])
    for name in ("log_prob", "best_log_prob"):
        g, w = getattr(got, name).cpu().double(), want[name]
        tol = log_tolerance(3000, w)
        assert torch.all((g == w) | ((g - w).abs() <= tol)), name
    g, w = got.entropy.cpu().double(), want["entropy"]
    assert torch.all((g - w).abs() <= log_tolerance(3000, w) * (1 + w))


def test_log_probs_of_special_rows(ops):
    lowest = torch.finfo(torch.float32).min
    cols = 5000
    x = torch.zeros(12, cols)
    x[0] = lowest                               # all equal, however low
    x[1] = lowest
    x[1, 17] = 3.0                              # one column has it all
    x[2] = -math.inf                            # none live
    x[3] = -math.inf
    x[3, 4999] = -80.0                          # one live
    x[4] = 1000.0 + torch.arange(cols) / 5000   # high and near each other
    x[5] = torch.arange(cols) * 0.01            # ever higher
    x[6] = torch.arange(cols).flip(0) * 0.01
    x[7, ::2] = -0.0                            # equal to the zeros between
    x[8, 100] = math.nan
    x[9, 100] = math.inf
    x[10] = lowest
    x[10, ::3] = -math.inf
    x[11, 1000:3000] = 5.0                      # two thousand equal ones
    target = torch.full((12,), 17, dtype=torch.int32)
    want = forms.log_probs(x, target, n_best=100)
    got = ops.log_probs(x.cuda(), target.cuda(), n_best=100)
    assert torch.all(torch.isnan(got.log_prob[8:10])) and torch.all(torch.isnan(got.log_sum[8:10])) and torch.all(torch.isnan(got.entropy[8:10]))
    assert got.best_index[9, 0] == 100
    assert torch.equal(got.best_index.cpu(), want["best_index"])
    rest = [r for r in range(12) if r not in (8, 9)]
    for name in ("log_prob", "best_log_prob"):
        g, w = getattr(got, name).cpu().double()[rest], want[name][rest]
        # row 5: |d| is up to 72, and log p of the target as large
        assert torch.equal(torch.isinf(g), torch.isinf(w))
        near = torch.isfinite(w) & (w.abs() < 1e30)
        assert torch.all((g[near] - w[near]).abs() <= log_tolerance(cols, w[near])), name
        far = torch.isfinite(w) & (w.abs() >= 1e30)  # row 1's alternatives: the lowest value, give or take roundings
        assert torch.allclose(g[far], w[far], rtol=8 * U, atol=0)
    g, w = got.entropy.cpu().double()[rest], want["entropy"][rest]
    assert torch.all((g - w).abs() <= log_tolerance(cols, w) * (1 + w))


def grad_tolerance(form, dtype, total, g_entropy, scale, cols, want):
    """A probability is off by the error of its logarithm; both are multiplied by what comes from above."""
    p, log_p, entropy = form["p"], torch.where(form["p"] > 0, form["log_p"], 0.0), form["entropy"][:, None]
    off = log_tolerance(cols, log_p)
    size = total[:, None].abs() + g_entropy[:, None].abs() * (log_p.abs() + entropy)
    tol = scale * p * (off * (size + g_entropy[:, None].abs() * (1 + entropy)) + 8 * U * size)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # steps of subnormal numbers
    return tol + (half_step(dtype) + 4 * U) * (want.abs() + tol) + tiny


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 5), (9, 768), (4, 2049), (3, 20_001)])
def test_log_probs_grad(ops, rows, cols, dtype):
    g = gen(cols)
    scale, k = 1.7, 6
    x = (torch.randn(rows, cols + 3, generator=g) * 2).to(dtype)[:, 1 : cols + 1]
    mask = torch.rand(rows, cols, generator=g) > 0.1
    mask[rows // 2] = rows == 1
    target = torch.randint(-1, cols, (rows,), generator=g, dtype=torch.int32)
    g_prob, g_entropy, g_best = (torch.randn(s, generator=g) for s in ((rows,), (rows,), (rows, k)))
    form = forms.log_probs(x, target, mask, scale=scale, n_best=k)
    device = torch.empty(rows, cols + 3, dtype=dtype).cuda()
    for prob, entropy, best in ((g_prob, None, None), (None, g_entropy, None), (g_prob, g_entropy, None), (g_prob, g_entropy, g_best), (None, None, None)):
        zero = torch.zeros(rows).double()
        want = forms.log_probs_grad(x, form, target, scale, prob, entropy, best)
        total = (zero if prob is None else prob.double().abs()) + (zero if best is None else best.double().abs().sum(1))
        tol = grad_tolerance(form, dtype, total, zero if entropy is None else entropy.double(), scale, cols, want)
        for place in ("new", "scores", "other"):
            device[:, 1 : cols + 1] = x.cuda()
            scores = device[:, 1 : cols + 1]
            result = ops.log_probs(scores, target.cuda(), mask=mask.cuda(), scale=scale, n_best=k)
            out = None if place == "new" else scores if place == "scores" else torch.full((rows, cols + 5), 9.0, dtype=dtype).cuda()[:, 2 : cols + 2]
            got = ops.log_probs_grad(scores, result, grad_log_prob=cuda(prob), grad_entropy=cuda(entropy), grad_best=cuda(best), out=out)
            assert out is None or got is out
            got = got.cpu().double()
            assert torch.all(got[~form["live"]] == 0)
            assert torch.all((got - want).abs() <= tol), (place, ((got - want).abs() / tol).max())


def test_log_probs_grad_against_differences(ops):
    """Central differences of the operator's own outputs, summed in 64 bits: off by h^2 / 6 of the third derivative (below 1 here)
    and by twice the outputs' error over 2 h."""
    rows, cols, k, h = 2, 9, 3, 2.0**-6
    g = gen(1)
    x = torch.randn(rows, cols, generator=g)
    target = torch.tensor([4, 0], dtype=torch.int32).cuda()
    weights = [torch.randn(s, generator=g).double() for s in ((rows,), (rows,), (rows, k))]

    def outputs(x):
        r = ops.log_probs(x.cuda(), target, n_best=k)
        return sum((w * t.cpu().double()).sum() for w, t in zip(weights, (r.log_prob, r.entropy, r.best_log_prob)))

    result = ops.log_probs(x.cuda(), target, n_best=k)
    got = ops.log_probs_grad(x.cuda(), result, grad_log_prob=weights[0].float().cuda(), grad_entropy=weights[1].float().cuda(), grad_best=weights[2].float().cuda())
    for r in range(rows):
        for c in range(cols):
            a, b = x.clone(), x.clone()
            a[r, c] += h
            b[r, c] -= h
            slope = float((outputs(a) - outputs(b)) / (a[r, c].double() - b[r, c].double()))
            assert abs(float(got[r, c]) - slope) <= 4 * h * h + 10 * float(log_tolerance(cols, torch.tensor(8.0))) / h


def test_log_probs_of_a_row_that_is_not_finite_has_no_finite_gradient(ops):
    x = torch.randn(2, 50)
    x[0, 3] = math.nan
    r = ops.log_probs(x.cuda(), torch.tensor([1, 2], dtype=torch.int32).cuda())
    got = ops.log_probs_grad(x.cuda(), r, grad_log_prob=torch.ones(2).cuda())
    assert torch.all(torch.isnan(got[0])) and torch.all(torch.isfinite(got[1]))


def test_log_probs_of_empty_matrices(ops):
    r = ops.log_probs(torch.empty(0, 5).cuda(), n_best=2)
    assert r.log_prob.shape == (0,) and r.best_index.shape == (0, 2)
    assert ops.log_probs_grad(torch.empty(0, 5).cuda(), r).shape == (0, 5)
    r = ops.log_probs(torch.empty(3, 0).cuda(), torch.zeros(3, dtype=torch.int32).cuda(), n_best=2)
    assert torch.all(r.log_sum == -math.inf) and torch.all(r.entropy == 0) and torch.all(r.log_prob == 0) and torch.all(r.best_index == -1)
    assert ops.log_probs_grad(torch.empty(3, 0).cuda(), r, grad_log_prob=torch.ones(3).cuda()).shape == (3, 0)


# ---------------------------------------------------------------------------
# Products of 8-bit rows


def rows_of_lengths(rows, cols, seed):
    g = gen(seed)
    return torch.randn(rows, cols, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g)) * torch.exp(torch.randn(1, cols, generator=g))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 16), (3, 127), (130, 128), (5, 129), (257, 700), (64, 1024), (2, 5000)])
def test_quantised_rows_are_the_definition_s(ops, rows, cols, dtype):
    wide = rows_of_lengths(rows, cols + 5, rows + cols).to(dtype)
    device = wide.cuda()
    for lead in (0, 3):
        x = wide[:, lead : lead + cols]
        want, exponent = forms.rows8(x)
        got = ops.quantise_rows(device[:, lead : lead + cols])
        assert torch.equal(got.dequantise().cpu().double(), want)
        layout = got.exponents.cpu().view(-(-rows // 128), -1, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-(-rows // 128) * 128, -1).int() - 127
        assert torch.equal(layout[:rows, : exponent.shape[1]], exponent)
        assert torch.all(layout[rows:] == 0) and torch.all(layout[:, exponent.shape[1] :] == 0)
        assert torch.all(got.values[:, cols:] == 0)
        turned = ops.quantise_rows(device[:, lead : lead + cols], transposed=True)
        want_t, exponent_t = forms.rows8(x.T)
        assert (turned.rows, turned.cols) == (cols, rows)
        assert torch.equal(turned.dequantise().cpu().double(), want_t)
        assert torch.all(turned.values[:, rows:] == 0)
        layout = turned.exponents.cpu().view(-(-cols // 128), -1, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-(-cols // 128) * 128, -1).int() - 127
        assert torch.all(layout[cols:] == 0) and torch.all(layout[:, exponent_t.shape[1] :] == 0)


def test_quantised_rows_at_the_ends_of_the_range(ops):
    x = torch.zeros(8, 256)
    x[0, :4] = torch.tensor([448.0, 449.0, -1.0, 2.0**-9])
    x[1, :3] = torch.tensor([math.inf, 3.0, math.nan])
    x[2, 0] = 2.0**-149
    x[2, 130] = 2.0**-126
    x[3, 0] = torch.finfo(torch.float32).max
    x[3, 1] = -1.0
    x[4, :5] = torch.tensor([448.0, 0.5 * 2.0**-9, 1.5 * 2.0**-9, -0.5 * 2.0**-9, 0.51 * 2.0**-9])  # halves of the smallest step
    x[5, 128:132] = torch.tensor([1.0, 1.0625, 1.1875, -0.0])  # ties between codes
    x[6] = -math.inf
    x[7, 7] = 1.75 * 2.0**-119
    got = ops.quantise_rows(x.cuda())
    want, exponent = forms.rows8(x)
    assert torch.equal(torch.isnan(want), ~torch.isfinite(x))
    assert want[3, 0] == 2.0**128  # the largest fp32 is rounded up past itself: as an fp32 that is infinite
    assert torch.allclose(got.dequantise().cpu(), want.float(), rtol=0, atol=0, equal_nan=True)


def product_tolerance(a, b, cols, out):
    """Products of two e4m3 numbers are exact in fp32.  An instruction adds 32 of them to the accumulator: each of its terms and the
    sum may lose what is below 2^-22 of the largest."""
    size = a.abs() @ b.abs().T
    want = a @ b.T
    tol = (cols / 32 + 4) * 2.0**-22 * size
    return want, tol + (half_step(out) + U) * (want.abs() + tol) + torch.finfo(out).smallest_normal * torch.finfo(out).eps


PRODUCT_SIZES = [(1, 1, 1), (1, 300, 256), (2, 129, 130), (16, 128, 128), (17, 500, 100), (33, 257, 640), (64, 64, 2000), (65, 130, 48),
                 (128, 384, 513), (200, 1000, 512), (300, 150, 1153), (513, 77, 300)]


@pytest.mark.parametrize("m,n,k", PRODUCT_SIZES)
def test_product8(ops, m, n, k):
    x, y = rows_of_lengths(m, k, m).clamp(-1e3, 1e3), rows_of_lengths(n, k, n + 1).clamp(-1e3, 1e3)
    a, b = ops.quantise_rows(x.cuda()), ops.quantise_rows(y.cuda())
    for out in TYPES:
        want, tol = product_tolerance(forms.rows8(x)[0], forms.rows8(y)[0], k, out)
        want = want.clamp(-torch.finfo(out).max, torch.finfo(out).max) if out == torch.float16 else want
        got = ops.product8(a, b, dtype=out).cpu().double()
        fine = want.abs() < 60000 if out == torch.float16 else torch.ones_like(want, dtype=torch.bool)
        assert torch.all(((got - want).abs() <= tol)[fine]), (out, ((got - want).abs() / tol)[fine].max())
    for out in TYPES:  # into a part of a larger matrix, at every alignment
        want, tol = product_tolerance(forms.rows8(x)[0], forms.rows8(y)[0], k, out)
        fine = want.abs() < 60000 if out == torch.float16 else torch.ones_like(want, dtype=torch.bool)
        for lead in (0, 3, 4):
            frame = torch.full((m, n + 9 - lead % 2), 5.0, dtype=out).cuda()
            ops.product8(x.cuda(), b, out=frame[:, lead : n + lead])
            assert torch.all(((frame[:, lead : n + lead].cpu().double() - want).abs() <= tol)[fine])
            assert torch.all(frame[:, :lead] == 5) and torch.all(frame[:, n + lead :] == 5)
    from distributed_kge_poplar_b200 import capi

    assert capi.load_library().kge_op_product8_status() == capi.OK


def test_product8_of_long_sums_and_few_tiles(ops):
    """The sum is split over the GPU's blocks and joined in order: the same bits each time."""
    m, n, k = 40, 70, 30_001
    x, y = rows_of_lengths(m, k, 1).clamp(-1e3, 1e3), rows_of_lengths(n, k, 2).clamp(-1e3, 1e3)
    a, b = ops.quantise_rows(x.cuda()), ops.quantise_rows(y.cuda())
    got = ops.product8(a, b)
    want, tol = product_tolerance(forms.rows8(x)[0], forms.rows8(y)[0], k, torch.float32)
    assert torch.all((got.cpu().double() - want).abs() <= tol)
    for _ in range(3):
        assert torch.equal(ops.product8(a, b), got)


@pytest.mark.parametrize("m,n,k", [(130, 300, 70_000), (600, 2000, 17_000), (20, 140, 9000)])
def test_product8_of_sums_that_only_grow(ops, m, n, k):
    """2048 products are summed in tensor memory, whose additions round toward zero: with all of one sign that takes at most their
    number of instructions, 64, times half of 2^-23 on average off the sum; those sums are joined in fp32, rounded to nearest.  One sum
    over all of k was 6e-5 off at 65 536."""
    g = gen(k)
    a, b = (ops.quantise_rows(torch.rand(rows, k, generator=g).cuda()) for rows in (m, n))
    got = ops.product8(a, b).double()
    want = a.dequantise().double() @ b.dequantise().double().T
    assert float(((got - want) / want).abs().max()) <= 64 * 2.0**-24 + math.sqrt(k / 2048) * 2.0**-22


def test_product8_with_values_that_are_not_finite(ops):
    x, y = torch.randn(20, 200), torch.randn(150, 200)
    x[3, 5], y[140, 199] = math.inf, math.nan
    got = ops.product8(x.cuda(), ops.quantise_rows(y.cuda())).cpu()
    bad = torch.zeros(20, 150, dtype=torch.bool)
    bad[3], bad[:, 140] = True, True
    assert torch.equal(torch.isnan(got), bad)


def test_product8_of_nothing(ops):
    a, b = ops.quantise_rows(torch.empty(0, 8).cuda()), ops.quantise_rows(torch.randn(3, 8).cuda())
    assert ops.product8(a, b).shape == (0, 3) and ops.product8(b, a).shape == (3, 0)
    empty = ops.quantise_rows(torch.empty(3, 0).cuda())
    assert torch.equal(ops.product8(empty, empty), torch.zeros(3, 3).cuda())


def test_products_are_each_other_s_gradients(ops):
    """d(a b^T): grad b and grad^T a, on operands quantised along the summed dimension."""
    m, n, k = 30, 200, 72
    x, y, g = (rows_of_lengths(r, c, s).clamp(-100, 100) for r, c, s in ((m, k, 1), (n, k, 2), (m, n, 3)))
    quantise = ops.quantise_rows
    for got, left, right in ((ops.product8(g.cuda(), quantise(y.cuda(), transposed=True)), g, y.T),
                             (ops.product8(quantise(g.cuda(), transposed=True), quantise(x.cuda(), transposed=True)), g.T, x.T)):
        want, tol = product_tolerance(forms.rows8(left)[0], forms.rows8(right)[0], left.shape[1], torch.float32)
        assert torch.all((got.cpu().double() - want).abs() <= tol)


# ---------------------------------------------------------------------------
# AdamW


def arena(sizes):
    first, total = [], 0
    for n in sizes:
        first.append(total)
        total += -(-n // 128) * 128
    return first, total


def adamw_step(p, g, m, v, step, rate, decay, beta_m=0.9, beta_v=0.99, epsilon=1e-6):
    m = beta_m * m + (1 - beta_m) * g
    v = beta_v * v + (1 - beta_v) * g * g
    update = rate / (1 - beta_m**step) * m / (v.sqrt() / math.sqrt(1 - beta_v**step) + epsilon)
    return p * (1 - rate * decay) - update, m, v, update


SIZES = [1, 127, 128, 129, 1000, 3, 4096, 77]


@pytest.mark.parametrize("grad_type", TYPES)
@pytest.mark.parametrize("param_type", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw(ops, bits, param_type, grad_type):
    """Each new value has one to four roundings of fp32; division and square root are counted as right to 2^-22.  What is rounded
    stochastically is off by less than a step, and differs from the same draws' choice in 64 bits only where a rounding of fp32 (2^-21
    of a value) decides: 2^-18 of a step, so of 16 000 choices at most one is expected in a run of ten of these tests."""
    g = gen(7)
    first, total = arena(SIZES)
    seed, rate, decay = 1234, 0.01, 0.1
    params = [torch.randn(n, generator=g).to(param_type) for n in SIZES]
    device = [p.cuda() for p in params]
    optimiser = ops.AdamW(device, state_bits=bits, beta_m=0.9, beta_v=0.99, epsilon=1e-6, weight_decay=decay, seed=seed)
    assert optimiser.first == first and optimiser.adam_m.numel() == total
    flips = 0
    for step in range(1, 4):
        grads = [(torch.randn(n, generator=g) * torch.exp(torch.randn(n, generator=g) * 2)).to(grad_type) for n in SIZES]
        grads[4][::5] = 0
        m0, v0 = (t.cpu().double() for t in optimiser.moments())
        before = [p.cpu().double() for p in device]
        optimiser.step([t.cuda() for t in grads], rate, grad_scale=0.5)
        m1, v1 = (t.cpu().double() for t in optimiser.moments())
        where = torch.zeros(total, dtype=torch.bool)
        for i, n in enumerate(SIZES):
            at = slice(first[i], first[i] + n)
            where[at] = True
            p, m, v, update = adamw_step(before[i], grads[i].double() * 0.5, m0[at], v0[at], step, rate, decay)
            position = torch.arange(first[i], first[i] + n)
            draw = forms.draws(position, seed, step)
            got = device[i].cpu().double()
            tol = 4 * U * (before[i].abs() + p.abs()) + 16 * U * update.abs()
            if param_type == torch.float32:
                assert torch.all((got - p).abs() <= tol)
            else:
                step_of = torch.exp2(torch.frexp(p)[1] - 8.0)
                down = torch.floor(p.abs() / step_of)
                want = torch.sign(p) * (down + ((p.abs() / step_of - down) + (draw >> 8 & 0xFFFF) / 65536 >= 1)) * step_of
                assert torch.all((got - want).abs() <= step_of * 1.001)
                flips += int((got != want).sum())
            if bits == 32:
                assert torch.all((m1[at] - m).abs() <= 4 * U * (m0[at].abs() + grads[i].double().abs()))
                assert torch.all((v1[at] - v).abs() <= 6 * U * v)
        if bits == 8:
            full_m, full_v = torch.zeros(total).double(), torch.zeros(total).double()
            for i, n in enumerate(SIZES):
                at = slice(first[i], first[i] + n)
                _, full_m[at], full_v[at], _ = adamw_step(before[i], grads[i].double() * 0.5, m0[at], v0[at], step, rate, decay)
            draw = forms.draws(torch.arange(total), seed, step)
            for full, got, code, exponent, random16, top in ((full_m, m1, optimiser.adam_m, optimiser.m_exponent, draw & 0xFFFF, 127),
                                                             (full_v, v1, optimiser.adam_v, optimiser.v_exponent, draw >> 16, 255)):
                want_code, want_exponent = forms.adamw_codes(full, random16, top)
                assert torch.equal(exponent.cpu().long(), want_exponent.view(-1))
                assert torch.equal(forms.adamw_values(code.cpu(), exponent.cpu(), top), got)
                held = torch.where(code.cpu() == 128, 0, code.cpu().long()) if top == 127 else code.cpu().long()  # zero of either sign
                other = held != want_code
                assert torch.all(((held & top) - (want_code & top)).abs()[other] <= 1)
                flips += int(other.sum())
        assert torch.all(m1[~where] == 0) and torch.all(v1[~where] == 0)
    assert optimiser.step_count == 3
    assert flips <= 2


def test_adamw_of_many_tensors_with_gaps(ops):
    """More tensors than one launch takes, some empty, some without a gradient, one that starts off a vector's boundary."""
    count = 600
    base = torch.randn(count * 3 + 1).cuda()
    params = [base[1 + 3 * i : 1 + 3 * i + (i % 4)] for i in range(count)]
    optimiser = ops.AdamW(params, beta_v=0.99, epsilon=1e-6)
    before = base.clone()
    grads = [torch.full((i % 4,), 2.0).cuda() if i % 5 else None for i in range(count)]
    optimiser.step(grads, 0.01)
    want = before.clone()
    for i, g in enumerate(grads):
        if g is not None:
            want[1 + 3 * i : 1 + 3 * i + (i % 4)] -= 0.01  # the first step is the sign's
    assert torch.allclose(base, want, rtol=0, atol=1e-7 + 1e-6 * 0.01 + 4 * U * float(before.abs().max()))
    optimiser.step([None] * count, 0.01)
    assert optimiser.step_count == 2


def test_adamw_moments_in_8_bits_are_right_on_average(ops):
    """v moves by a hundredth of itself a step, a twelfth of what separates two codes: it follows only if rounding is unbiased.  After
    400 steps of g = 1 it stands at 1 - 0.99^400 = 0.982; each value is a walk of steps of 1/8 with variance 1/8 * (1 - beta_v) a
    step against a pull of 1 - beta_v: variance 1/16, a deviation of 0.25 / sqrt(n) of the mean of n."""
    n = 1 << 16
    p = torch.zeros(n).cuda()
    optimiser = ops.AdamW([p], state_bits=8, beta_m=0.9, beta_v=0.99, seed=5)
    g = torch.ones(n).cuda()
    for _ in range(400):
        optimiser.step([g], 1e-3)
    m, v = optimiser.moments()
    assert abs(float(v.float().mean()) - (1 - 0.99**400)) <= 6 * 0.25 / math.sqrt(n)
    assert abs(float(m.float().mean()) - 1) <= 6 * 0.125 / math.sqrt(n)
    assert float(v.float().min()) > 0


def test_adamw_of_gradients_that_are_not_finite(ops):
    for bits in (8, 32):
        p = torch.ones(300).cuda()
        optimiser = ops.AdamW([p], state_bits=bits)
        g = torch.ones(300).cuda()
        g[5] = math.nan
        g[200] = math.inf
        optimiser.step([g], 0.1)
        m, _ = optimiser.moments()
        bad = torch.zeros(300, dtype=torch.bool)
        bad[[5, 200]] = True
        assert torch.equal(torch.isnan(p.cpu()), bad)
        lost = torch.zeros(384, dtype=torch.bool)
        if bits == 8:
            lost[:128], lost[128:256] = True, True  # their blocks' codes say nothing any more
        else:
            lost[[5, 200]] = True
        assert torch.equal(~torch.isfinite(m.cpu().float()), lost)


def test_adamw_state_goes_on_where_it_was(ops):
    for bits in (8, 32):
        g = gen(bits)
        start = torch.randn(1000, generator=g)
        grads = [torch.randn(1000, generator=g).cuda() for _ in range(6)]
        p, q = start.cuda(), start.cuda()
        whole, part = ops.AdamW([p], state_bits=bits, seed=3), ops.AdamW([q], state_bits=bits, seed=3)
        for t in grads:
            whole.step([t], 0.01)
        for t in grads[:3]:
            part.step([t], 0.01)
        later = ops.AdamW([q], state_bits=bits)
        later.load_state(part.state())
        for t in grads[3:]:
            later.step([t], 0.01)
        assert torch.equal(p, q) and torch.equal(whole.adam_m, later.adam_m) and torch.equal(whole.adam_v, later.adam_v)


# ---------------------------------------------------------------------------
# Together, captured, and side by side


def train_step(ops, queries, table, target, optimiser, **how):
    """A step of a softmax over all rows of a table: scores, loss, gradients, update."""
    table8, queries8 = ops.quantise_rows(table), ops.quantise_rows(queries)
    scores = ops.product8(queries8, table8, dtype=torch.bfloat16)
    result = ops.log_probs(scores, target)
    grad = ops.log_probs_grad(scores, result, grad_log_prob=torch.full_like(result.log_prob, -1.0 / queries.shape[0]))
    grad_queries = ops.product8(grad, ops.quantise_rows(table, transposed=True))
    grad_table = ops.product8(ops.quantise_rows(grad, transposed=True), ops.quantise_rows(queries, transposed=True))
    optimiser.step([grad_queries, grad_table], **how)
    return result.log_prob, grad_queries, grad_table


def test_a_training_step_of_all_of_them(ops):
    """Loss and gradients against the same step in 64 bits on the same rounded operands: scores are rounded to bf16 in both, so only
    choices at a border of bf16 or e4m3 differ."""
    m, n, k = 48, 700, 200
    g = gen(11)
    queries, table = torch.randn(m, k, generator=g), torch.randn(n, k, generator=g) * 0.2
    target = torch.randint(n, (m,), generator=g, dtype=torch.int32)
    a, b = queries.cuda(), table.cuda()
    optimiser = ops.AdamW([a, b])
    log_prob, grad_queries, grad_table = train_step(ops, a, b, target.cuda(), optimiser, learning_rate=0.01)
    scores = (forms.rows8(queries)[0] @ forms.rows8(table)[0].T).float().bfloat16()
    form = forms.log_probs(scores, target)
    assert torch.allclose(log_prob.cpu().double(), form["log_prob"], rtol=0, atol=0.05)  # a border of bf16 scores of 10: 2^-5
    grad = forms.log_probs_grad(scores, form, target, 1.0, torch.full((m,), -1.0 / m)).float().bfloat16()
    for got, want in ((grad_queries, forms.rows8(grad)[0] @ forms.rows8(table.T)[0].T), (grad_table, forms.rows8(grad.T)[0] @ forms.rows8(queries.T)[0].T)):
        off = (got.cpu().double() - want).norm() / want.norm()
        assert off <= 2.0**-4  # were every choice of e4m3 the other one
    assert torch.all((a.cpu() - queries).abs() <= 0.01001) and float((a.cpu() - queries).abs().max()) > 0.009


def test_a_captured_step_replays_as_it_ran(ops):
    m, n, k = 20, 300, 64
    g = gen(12)
    queries, table = torch.randn(m, k, generator=g), torch.randn(n, k, generator=g)
    target = torch.randint(n, (m,), generator=g, dtype=torch.int32).cuda()
    eager = [queries.cuda(), table.cuda()]
    by_graph = [t.clone() for t in eager]
    one, other = (ops.AdamW(p, state_bits=8, seed=9) for p in (eager, by_graph))
    schedule = other.new_schedule()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # once outside a capture
        scratch = ops.AdamW([t.clone() for t in by_graph], state_bits=8)
        train_step(ops, *scratch.params, target, scratch, learning_rate=0.01)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = train_step(ops, *by_graph, target, other, schedule=schedule)
    for rate in (0.01, 0.005, 0.02):
        want = train_step(ops, *eager, target, one, learning_rate=rate)
        other.advance(schedule, rate)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(want, result):
            assert torch.equal(x, y)
        for x, y in zip(eager, by_graph):
            assert torch.equal(x, y)
        assert torch.equal(one.adam_v, other.adam_v) and one.step_count == other.step_count
    with pytest.raises(RuntimeError, match="schedule"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            one.step([torch.zeros_like(t) for t in eager], 0.01)


def test_calls_on_two_streams_at_once(ops):
    g = gen(13)
    x = [torch.randn(200, 30_000, generator=g).bfloat16().cuda() for _ in range(2)]
    t = torch.zeros(200, dtype=torch.int32).cuda()
    long_a, long_b = torch.randn(40, 20_000, generator=g).cuda(), torch.randn(60, 20_000, generator=g).cuda()
    want = [(ops.log_probs(v, t, n_best=20), ops.product8(long_a, long_b)) for v in x]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in x]
    got = []
    for _ in range(3):
        for s, v in zip(streams, x):
            with torch.cuda.stream(s):
                got.append((v, ops.log_probs(v, t, n_best=20), ops.product8(long_a, long_b)))
    torch.cuda.synchronize()
    for v, r, p in got:
        w, q = want[0 if v is x[0] else 1]
        assert torch.equal(r.log_prob, w.log_prob) and torch.equal(r.entropy, w.entropy) and torch.equal(r.best_index, w.best_index) and torch.equal(p, q)


def test_calls_that_are_refused(ops):
    x = torch.randn(6, 8).cuda()
    r = ops.log_probs(x, n_best=2)
    column = torch.zeros(8, 6).cuda().T
    for call, text in [(lambda: ops.log_probs(column), "contiguous along its rows"), (lambda: ops.log_probs(x[0]), "two dimensions"),
                       (lambda: ops.log_probs(x.double()), "not torch.float64"), (lambda: ops.log_probs(x[:1].expand(6, 8)), "apart"),
                       (lambda: ops.log_probs(x, torch.zeros(6).cuda()), "torch.int32"), (lambda: ops.log_probs(x, torch.zeros(5, dtype=torch.int32).cuda()), "shape"),
                       (lambda: ops.log_probs(x, torch.zeros(6, dtype=torch.int32)), "on a GPU"), (lambda: ops.log_probs(x, torch.zeros(12, dtype=torch.int32).cuda()[::2]), "contiguous"),
                       (lambda: ops.log_probs(x, mask=torch.ones(6, 7, dtype=torch.bool).cuda()), "shape"), (lambda: ops.log_probs(x, mask=x), "torch.bool"),
                       (lambda: ops.log_probs(x, scale=0.0), "scale"), (lambda: ops.log_probs(x, scale=3e38), "scale"), (lambda: ops.log_probs(x, n_best=-1), "n_best"),
                       (lambda: ops.log_probs_grad(x[:5], r), "shape"), (lambda: ops.log_probs_grad(x, r, grad_log_prob=torch.ones(6).cuda().half()), "torch.float32"),
                       (lambda: ops.log_probs_grad(x, r, grad_best=torch.ones(6, 3).cuda()), "shape"), (lambda: ops.log_probs_grad(x, r, out=x.half()), "out must be"),
                       (lambda: ops.log_probs_grad(x[:, :7], ops.log_probs(x[:, :7]), out=x[:, 1:]), "overlap"),
                       (lambda: ops.quantise_rows(column), "contiguous along its rows"), (lambda: ops.product8(x, x[:, :4]), "rows of 8 and of 4"),
                       (lambda: ops.product8(x, x, dtype=torch.float64), "dtype"), (lambda: ops.product8(x, x, out=torch.zeros(6, 5).cuda()), "shape"),
                       (lambda: ops.AdamW([x, x[2:4]]), "overlap"), (lambda: ops.AdamW([x, x.bfloat16()]), "an optimiser for each type"), (lambda: ops.AdamW([x.half()]), "parameter 0 must be"),
                       (lambda: ops.AdamW([column]), "contiguous"), (lambda: ops.AdamW([x], beta_v=1.0), "beta"), (lambda: ops.AdamW([x], epsilon=0.0), "epsilon")]:
        with pytest.raises(ValueError, match=text):
            call()
    optimiser = ops.AdamW([x, torch.zeros(3).cuda()])
    for grads, how, text in [([x], dict(learning_rate=0.1), "1 gradients for 2"), ([x, x], dict(learning_rate=0.1), "shape"), ([x.half(), torch.zeros(3).cuda()], dict(learning_rate=0.1), "others"),
                             ([column, None], dict(learning_rate=0.1), "contiguous"), ([x, None], {}, "learning_rate or a schedule"),
                             ([x, None], dict(schedule=torch.zeros(3).cuda()), "schedule has shape")]:
        with pytest.raises(ValueError, match=text):
            optimiser.step(grads, **how)
    assert optimiser.step_count == 0
    with pytest.raises(ValueError, match="does not fit"):
        optimiser.load_state(ops.AdamW([x], state_bits=8).state())


def test_gradients_that_are_broadcast_and_leaves_that_require_them(ops):
    x = torch.randn(5, 300).cuda()
    r = ops.log_probs(x, torch.zeros(5, dtype=torch.int32).cuda())
    one = torch.tensor([0.25]).cuda()
    assert torch.equal(ops.log_probs_grad(x, r, grad_log_prob=one.expand(5)), ops.log_probs_grad(x, r, grad_log_prob=torch.full((5,), 0.25).cuda()))
    leaf = torch.randn(40, 3).cuda().requires_grad_()
    optimiser = ops.AdamW([leaf])
    before, version = leaf.detach().clone(), leaf._version
    optimiser.step([torch.ones_like(leaf)], 0.1)
    assert leaf._version > version and float((before - leaf.detach() - 0.1).abs().max()) < 1e-5


def test_adamw_of_tensors_whose_memory_was_replaced(ops):
    for change, text in [(lambda t: t.cpu(), "parameter 1 is no longer"), (lambda t: t.bfloat16(), "parameter 1 is no longer"), (lambda t: t.new_zeros(4, 300), "parameter 1 is no longer"),
                         (lambda t: t.T.contiguous().T, "parameter 1 is no longer")]:
        params = [torch.zeros(5).cuda(), torch.zeros(4, 3).cuda()]
        optimiser = ops.AdamW(params)
        params[1].data = change(params[1].data)
        with pytest.raises(ValueError, match=text):
            optimiser.step([torch.ones(5).cuda(), torch.ones_like(params[1])], 0.1)
        assert torch.all(params[0] == 0)
    optimiser = ops.AdamW([torch.zeros(400).cuda()], state_bits=8)
    optimiser.adam_v = optimiser.adam_v[:128]
    with pytest.raises(ValueError, match="adam_v has shape"):
        optimiser.step([torch.ones(400).cuda()], 0.1)
    params = [torch.zeros(4, 3).cuda()]
    optimiser = ops.AdamW(params)
    params[0].data = torch.ones(4, 3).cuda()
    optimiser.step([torch.ones(4, 3).cuda()], 0.1)  # new memory of the same kind is updated
    assert float((params[0] - 0.9).abs().max()) < 1e-5
