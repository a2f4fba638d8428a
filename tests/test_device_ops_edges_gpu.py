"""The operators on device tensors where their definitions are easily missed: values that are not finite or far from the others, lists
that are thinned out, larger blocks, tiles and parts."""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import device_op_forms as forms  # noqa: E402
from test_device_ops_gpu import TYPES, U, check_log_probs, cuda, gen, grad_tolerance, log_tolerance, ops, product_tolerance, rows_of_lengths  # noqa: E402, F401

pytestmark = pytest.mark.gpu

# Rows and columns of fp32 scores for which a row is one block of 128, 256, 512 or 1024 threads, or is cut into parts.
SHAPES = {128: (6, 1500), 256: (330, 9001), 512: (200, 9001), 1024: (100, 20_001), "few parts": (1, 100_001), "parts": (3, 150_001)}


@pytest.mark.parametrize("size", SHAPES)
def test_lists_of_many_candidates(ops, size):  # noqa: F811
    """600 columns share the best score: more pass the first threshold than are ranked, so a second one is looked for among them."""
    rows, cols = SHAPES[size]
    g = gen(cols)
    x = torch.randn(rows, cols, generator=g).clamp(max=2.0)
    at = torch.stack([torch.randperm(cols, generator=g)[:600] for _ in range(rows)])
    x.scatter_(1, at, 3.0)
    want = at.sort(1).values[:, :100].int()
    device = x.cuda()
    for _ in range(20):
        got = ops.log_probs(device, n_best=100)
        assert torch.equal(got.best_index.cpu(), want)
    few = min(rows, 12)
    check_log_probs(ops.log_probs(device[:few], n_best=100), forms.log_probs(x[:few], None, n_best=100), cols)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_live_nan_wherever_it_is(ops, dtype):  # noqa: F811
    """Short rows at every alignment, the NaN in each of their columns: it may be all that a thread sees."""
    for cols in range(1, 20):
        for lead in range(8):
            wide = torch.randn(cols, cols + 9, generator=gen(cols * 10 + lead)).to(dtype)
            x = wide[:, lead : lead + cols]
            x.diagonal().fill_(math.nan)
            device = wide.cuda()[:, lead : lead + cols]
            target = torch.zeros(cols, dtype=torch.int32)
            got = ops.log_probs(device, target.cuda(), n_best=4)
            check_log_probs(got, forms.log_probs(x, target, n_best=4), cols)
            assert torch.all(torch.isnan(got.log_sum)) and torch.all(torch.isnan(got.entropy)) and torch.all(torch.isnan(got.log_prob))
            assert torch.all(torch.isnan(ops.log_probs_grad(device, got, grad_log_prob=torch.ones(cols).cuda())))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hidden", ["mask", "-inf"])
@pytest.mark.parametrize("size", SHAPES)
def test_a_live_nan_among_hidden_columns(ops, size, hidden, dtype):  # noqa: F811
    """One NaN and twenty other live columns a row, far apart; in every third row the NaN is hidden too."""
    rows, cols = SHAPES[size]
    g = gen(cols + 1)
    x = torch.randn(rows, cols, generator=g).to(dtype)
    at = torch.stack([torch.randperm(cols, generator=g)[:21] for _ in range(rows)])
    live = torch.zeros(rows, cols, dtype=torch.bool).scatter_(1, at, True)
    live[torch.arange(0, rows, 3), at[::3, 0]] = False
    x[torch.arange(rows), at[:, 0]] = math.nan
    target = at[:, 1].int().contiguous()
    mask = live if hidden == "mask" else None
    if hidden == "-inf":
        x = torch.where(live, x, -math.inf)
    got = ops.log_probs(x.cuda(), target.cuda(), mask=cuda(mask), n_best=25)
    check_log_probs(got, forms.log_probs(x, target, mask, n_best=25), cols)
    lost = torch.ones(rows, dtype=torch.bool)
    lost[::3] = False
    assert torch.equal(torch.isnan(got.log_sum).cpu(), lost)
    grad = ops.log_probs_grad(x.cuda(), got, grad_log_prob=torch.ones(rows).cuda()).cpu()
    assert torch.equal(torch.isnan(grad), live & lost[:, None]) and torch.all(grad[~live] == 0)


@pytest.mark.parametrize("far", [-1e9, -3e9, -1e10, -1e20, 1e10, 1e20])
@pytest.mark.parametrize("dtype,scale", [(torch.float32, 1.0), (torch.bfloat16, 0.5), (torch.float16, 1e6)])
@pytest.mark.parametrize("cols", [5000, 70_001])
def test_scores_far_from_the_others(ops, cols, dtype, scale, far):  # noqa: F811
    """Finite numbers that stand for hidden columns, or for the one answer: logits whose rounding in fp32 is more than a power of two's
    whole range.  A row's own differences are what counts; equal scores share the row however far out they are."""
    far = max(-65504.0, min(65504.0, far / scale)) if dtype == torch.float16 else far
    g = gen(cols)
    x = (torch.randn(8, cols, generator=g) * (3 / max(scale, 1.0))).to(dtype)
    x[0] = far
    x[1, : cols // 2] = far
    x[2, -40:] = far
    x[3, : cols - cols // 10] = far
    x[4] = far
    x[4, cols - 1] = 1.0
    x[5].view(-1, 8 if cols % 8 == 0 else 1)[::2] = far
    x[6] = far
    x[6, ::3] = -math.inf
    x[7, 4] = far
    target = torch.tensor([3, 5, cols - 1, cols - 2, cols - 1, 2, 1, 4], dtype=torch.int32)
    weights = [torch.randn(shape, generator=g) / max(scale, 1.0) for shape in ((8,), (8,), (8, 5))]
    want = forms.log_probs(x, target, scale=scale, n_best=5)
    got = ops.log_probs(x.cuda(), target.cuda(), scale=scale, n_best=5)
    for name in ("log_prob", "log_sum", "best_log_prob"):
        a, b = getattr(got, name).cpu().double(), want[name]
        assert torch.all((a - b).abs() <= log_tolerance(cols, b)), (name, a, b)
    a, b = got.entropy.cpu().double(), want["entropy"]
    assert torch.all((a - b).abs() <= log_tolerance(cols, b) * (1 + b))
    assert torch.equal(got.best_index.cpu(), want["best_index"])
    grad = ops.log_probs_grad(x.cuda(), got, grad_log_prob=weights[0].cuda(), grad_entropy=weights[1].cuda(), grad_best=weights[2].cuda()).cpu().double()
    right = forms.log_probs_grad(x, want, target, scale, *weights)
    total = weights[0].double().abs() + weights[2].double().abs().sum(1)
    tol = grad_tolerance(want, dtype, total, weights[1].double(), scale, cols, right)
    assert torch.all((grad - right).abs() <= tol), ((grad - right).abs() / tol).max()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_of_tiny_gradients(ops, bits):  # noqa: F811
    """Second moments that are subnormal in fp32 count: (1 - beta_v) g^2 and its sum are off by a step of subnormal numbers, 2^-149, which
    moves the root by that over 2 v of itself.  A step in 8 bits divides by the sum before it is encoded."""
    g = torch.exp(torch.linspace(math.log(2e-20), math.log(3e-16), 4096).double()).float() * torch.tensor([1.0, -1.0]).repeat(2048)
    p = torch.zeros(4096).cuda()
    optimiser = ops.AdamW([p], state_bits=bits, beta_m=0.9, beta_v=0.999, epsilon=1e-20)
    optimiser.step([g.cuda()], 0.01)
    m, v = 0.1 * g.double(), 0.001 * g.double() ** 2
    want = -0.01 * (m / 0.1) / ((v / 0.001).sqrt() + 1e-20)
    off = 2.0**-149 / (2 * v) + 32 * U
    assert torch.all((p.cpu().double() - want).abs() <= off * want.abs())


def test_a_step_of_32_bits_is_rounded_as_its_formula_is(ops):  # noqa: F811
    """The first step in numpy's fp32 arithmetic, its two fused operations in 64 bits and rounded once more: that differs from a fused one
    only where 53 bits end in a half of 24, once in 2^28."""
    n = 1 << 16
    g = (torch.randn(n, generator=gen(5)) * torch.exp(2 * torch.randn(n, generator=gen(6)))).numpy()
    p0 = torch.randn(n, generator=gen(7)).numpy()
    p = torch.from_numpy(p0).cuda()
    optimiser = ops.AdamW([p], beta_m=0.9, beta_v=0.999, epsilon=1e-8, weight_decay=0.1)
    optimiser.step([torch.from_numpy(g).cuda()], 0.01)
    f = np.float32
    m, v = f(1 - 0.9) * g, f(1 - 0.999) * g * g
    assert np.array_equal(optimiser.adam_m[:n].cpu().numpy(), m) and np.array_equal(optimiser.adam_v[:n].cpu().numpy(), v)
    under = (np.sqrt(v).astype(np.float64) * f((1 - 0.999) ** -0.5) + np.float64(f(1e-8))).astype(f)
    step = -f(0.01 / (1 - 0.9)) * m / under
    want = (p0.astype(np.float64) * f(1 - 0.01 * 0.1) + step).astype(f)
    assert np.array_equal(p.cpu().numpy(), want)


def test_the_product_s_status_waits_for_every_stream(ops):  # noqa: F811
    x = torch.randn(200, 300).cuda()
    ops.product8(x, x)  # the first call of a kernel loads it and waits
    ops.check_product8()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # a tenth of a second
        ops.product8(x, x)
    ops.check_product8()
    assert side.query()


def test_outputs_that_overlap_what_is_read_are_refused(ops):  # noqa: F811
    x = torch.randn(6, 8).cuda()
    r = ops.log_probs(x, torch.zeros(6, dtype=torch.int32).cuda(), n_best=8)
    ones = torch.ones(6, 8).cuda()
    a, b = ops.quantise_rows(torch.randn(64, 128).cuda()), ops.quantise_rows(torch.randn(16, 128).cuda())
    for call, text in [(lambda: ops.log_probs_grad(x, r, out=r.best_log_prob), "out and the result"),
                       (lambda: ops.log_probs_grad(x, r, grad_best=ones, out=ones), "out and grad_best"),
                       (lambda: ops.log_probs_grad(x, r, grad_log_prob=ones.view(-1)[:6], out=ones), "out and grad_log_prob"),
                       (lambda: ops.log_probs_grad(x, ops.log_probs(x, ones.view(torch.int32)[0, :6]), out=ones), "out and target"),
                       (lambda: ops.log_probs_grad(x, ops.log_probs(x, count=ones.view(torch.int32)[0, :6]), out=ones), "out and count"),
                       (lambda: ops.log_probs_grad(x, ops.log_probs(x, mask=ones.view(torch.uint8)[:6, 4:12]), out=ones), "out and mask"),
                       (lambda: ops.product8(a, b, out=a.values.view(torch.bfloat16).view(-1)[: 64 * 16].view(64, 16)), "out and a overlap"),
                       (lambda: ops.product8(b, a, out=a.values.view(torch.bfloat16).view(-1)[: 64 * 16].view(16, 64)), "out and b overlap"),
                       (lambda: ops.product8(b, b, out=a.exponents.view(torch.bfloat16).view(16, 16)), None)]:
        if text is None:
            call()
            continue
        with pytest.raises(ValueError, match=text):
            call()
    assert torch.equal(ops.log_probs_grad(x.clone(), r, grad_best=ones), ops.log_probs_grad(x, r, grad_best=ones, out=x))  # in place is no overlap


def test_parameters_that_overlap_a_gradient_or_one_another_are_refused(ops):  # noqa: F811
    base = torch.zeros(400).cuda()
    params = [base[200:300], base[:100], torch.zeros(0).cuda(), torch.zeros(50).cuda()]
    optimiser = ops.AdamW(params)
    apart = [torch.ones(100).cuda(), torch.ones(100).cuda(), torch.zeros(0).cuda(), torch.ones(50).cuda()]
    for i, grad, text in [(0, base[200:300], "gradient 0 and parameter 0"), (0, base[1:101], "gradient 0 and parameter 1"),
                          (1, base[299:399], "gradient 1 and parameter 0"), (3, base[170:220], "gradient 3 and parameter 0")]:
        with pytest.raises(ValueError, match=text + " overlap"):
            optimiser.step([grad if j == i else g for j, g in enumerate(apart)], 0.1)
    params[3].data = base[80:130]
    with pytest.raises(ValueError, match="parameters 1 and 3 overlap"):
        optimiser.step(apart, 0.1)
    assert optimiser.step_count == 0 and torch.all(base == 0)
    optimiser.step([base[300:400], base[100:200], None, None], 0.1)  # side by side
    params[3].data = base[130:180]
    optimiser.step([torch.ones(100).cuda()] * 2 + [None, torch.ones(50).cuda()], 0.1)  # moved, and one gradient for two
    assert torch.all(base[130:180] < 0) and torch.all(base[180:200] == 0)


def test_a_schedule_is_written_without_waiting(ops):  # noqa: F811
    """Replays are queued behind a stream that is busy; each reads its own step's words all the same."""
    g = gen(4)
    start, grad = torch.randn(1000, generator=g), torch.randn(1000, generator=g).cuda()
    p, q = start.cuda(), start.cuda()
    one, other = ops.AdamW([p], state_bits=8, seed=3), ops.AdamW([q], state_bits=8, seed=3)
    one.step([grad], 0.01)
    schedule = other.new_schedule()
    other.advance(schedule, 0.01)
    other.step([grad], schedule=schedule)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        other.step([grad], schedule=schedule)
    torch.cuda.synchronize()
    torch.cuda._sleep(400_000_000)  # a fifth of a second
    for i in range(20):
        other.advance(schedule, 0.01 / (i + 1))
        graph.replay()
    assert not torch.cuda.current_stream().query()
    for i in range(20):
        one.step([grad], 0.01 / (i + 1))
    assert torch.equal(p, q) and torch.equal(one.adam_m, other.adam_m) and torch.equal(one.adam_v, other.adam_v)
    with pytest.raises(RuntimeError, match="not under its capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            other.advance(schedule, 0.01)
    assert other.step_count == 21


def test_moments_whose_memory_was_replaced(ops):  # noqa: F811
    for name, text in [("m_exponent", "m_exponent has shape"), ("v_exponent", "v_exponent has shape"), ("adam_v", "adam_v has shape"), ("adam_m", "exponent has shape")]:
        optimiser = ops.AdamW([torch.zeros(400).cuda()], state_bits=8)
        kept = getattr(optimiser, name)
        setattr(optimiser, name, kept[: kept.numel() // 2])
        with pytest.raises(ValueError, match=text):
            optimiser.moments()
        setattr(optimiser, name, kept.cpu())
        with pytest.raises(ValueError, match="on a GPU|is on"):
            optimiser.moments()


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_schedule_that_was_not_advanced_leaves_the_parameters(ops, dtype, bits):  # noqa: F811
    start = torch.randn(1000, generator=gen(8)).to(dtype)
    p = start.cuda()
    optimiser = ops.AdamW([p], state_bits=bits)
    optimiser.step([torch.randn(1000, generator=gen(9)).to(dtype).cuda()], schedule=optimiser.new_schedule())  # as a step before a capture may be
    assert torch.equal(p.cpu(), start)


@pytest.mark.parametrize("n", [1, 7, 77, 127, 129, 264, 300, 385, 1001])
@pytest.mark.parametrize("m", [20, 40, 100, 300])
def test_product8_into_a_part_of_rows_on_16_bytes(ops, m, n):  # noqa: F811
    """Results of any width in rows that begin on 16 bytes: what lies beside and below them stays."""
    k = 130
    a, b = (ops.quantise_rows(rows_of_lengths(rows, k, rows).clamp(-1e3, 1e3).cuda()) for rows in (m, n))
    for out in TYPES:
        want, tol = product_tolerance(a.dequantise().double(), b.dequantise().double(), k, out)
        fine = want.abs() < 60000 if out == torch.float16 else torch.ones_like(want, dtype=torch.bool)
        for lead in (0, 8):
            frame = torch.full((m + 3, n + 16 + -n % 8), 5.0, dtype=out, device="cuda")
            got = ops.product8(a, b, out=frame[:m, lead : lead + n])
            assert torch.all(((got.double() - want).abs() <= tol) | ~fine)
            frame[:m, lead : lead + n] = 5
            assert torch.all(frame == 5)


# (queries, rows of the table, values of a row): a block's tile of 16, 32, 64, 128 or 256 queries, which it keeps or fetches with each part
# of the table; more tiles than blocks; tiles in a row or four side by side; sums of one to four times 2048 values.
MANY_TILES = [(100, 25_001, 256), (512, 10_003, 300), (1500, 7000, 200), (4700, 9001, 100), (600, 7700, 900), (513, 3205, 2100), (300, 9600, 6200), (100, 20_001, 900),
              (64, 20_000, 1700), (20, 20_001, 3300), (9, 20_003, 6500), (19_001, 300, 100)]


@pytest.mark.parametrize("m,n,k", MANY_TILES)
def test_product8_of_many_tiles(ops, m, n, k):  # noqa: F811
    g = torch.Generator(device="cuda").manual_seed(m + n + k)

    def rows(count):
        length = torch.exp(2 * torch.randn(count, 1, generator=g, device="cuda"))
        return (torch.randn(count, k, generator=g, device="cuda") * length).clamp(-1e3, 1e3)

    a, b = ops.quantise_rows(rows(m)), ops.quantise_rows(rows(n))
    for out in TYPES:
        want, tol = product_tolerance(a.dequantise().double(), b.dequantise().double(), k, out)
        fine = want.abs() < 60000 if out == torch.float16 else torch.ones_like(want, dtype=torch.bool)
        for pad, lead in ((0, 0), (9, 3), (8 - n % 8, 0)):  # as it comes, at no boundary, in rows on 16 bytes
            frame = torch.full((m + 2, n + pad), 5.0, dtype=out, device="cuda")
            got = ops.product8(a, b, out=frame[:m, lead : lead + n])
            off = (got.double() - want).abs()
            assert torch.all((off <= tol) | ~fine), (out, pad, (off / tol)[fine].max())
            assert torch.all(frame[:m, :lead] == 5) and torch.all(frame[:m, lead + n :] == 5) and torch.all(frame[m:] == 5)
    ops.check_product8()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SHAPES)
def test_masks_and_counts_in_every_size_of_block(ops, size, dtype):  # noqa: F811
    """What is hidden holds NaN, infinities and numbers above all others; some rows are hidden whole, some columns in all rows."""
    rows, cols = SHAPES[size]
    g, scale = gen(cols + 2), 0.7
    x = (torch.randn(rows, cols, generator=g) * 3).to(dtype)
    mask = torch.rand(rows, cols, generator=g) > 0.4
    mask[:, cols // 3 : cols // 2] = False
    mask[2::7] = False
    count = torch.randint(1, cols + 9, (rows,), generator=g, dtype=torch.int32)
    target = torch.randint(-1, cols, (rows,), generator=g, dtype=torch.int32)
    live = forms.live_columns(x, mask, count)
    hidden = torch.where(live, x, torch.tensor([math.nan, math.inf, -math.inf, 6e4])[torch.arange(cols) % 4].to(dtype)).cuda()
    weights = [torch.randn(shape, generator=g) for shape in ((rows,), (rows,), (rows, 40))]
    want = forms.log_probs(x, target, mask, count, scale=scale, n_best=40)
    right = forms.log_probs_grad(x, want, target, scale, *weights)
    tol = grad_tolerance(want, dtype, weights[0].double().abs() + weights[2].double().abs().sum(1), weights[1].double(), scale, cols, right)
    wide = torch.zeros(rows, cols + 5, dtype=torch.bool).cuda()  # a mask at no boundary
    wide[:, 3 : cols + 3] = mask.cuda()
    for m in (mask.cuda(), wide[:, 3 : cols + 3], mask.to(torch.uint8).cuda() * 130):
        got = ops.log_probs(hidden, target.cuda(), mask=m, count=count.cuda(), scale=scale, n_best=40)
        check_log_probs(got, want, cols)
        grad = ops.log_probs_grad(hidden, got, grad_log_prob=weights[0].cuda(), grad_entropy=weights[1].cuda(), grad_best=weights[2].cuda()).cpu().double()
        assert torch.all(grad[~live] == 0) and torch.all((grad - right).abs() <= tol), ((grad - right).abs() / tol).nan_to_num(0).max()


@pytest.mark.parametrize("grad_type", TYPES)
@pytest.mark.parametrize("param_type", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_of_tensors_at_no_boundary(ops, bits, param_type, grad_type):  # noqa: F811
    """Draws depend on a value's place in the moments alone: tensors that lie elsewhere get the same bits."""
    sizes, g = [1, 5, 127, 128, 513, 2000, 16, 700], gen(21)
    start = [torch.randn(n, generator=g).to(param_type) for n in sizes]

    def lying(values, lead):
        held = [torch.full((len(v) + lead + 3,), 7.0, dtype=v.dtype).cuda() for v in values]
        for h, v in zip(held, values):
            h[lead : lead + len(v)] = v.cuda()
        return held, [h[lead : lead + len(v)] for h, v in zip(held, values)]

    kept = [lying(start, lead) for lead in (0, 1, 2, 4)]
    optimisers = [ops.AdamW(views, state_bits=bits, seed=11, weight_decay=0.1) for _, views in kept]
    for _ in range(3):
        grads = [(torch.randn(n, generator=g) * torch.exp(torch.randn(n, generator=g))).to(grad_type) for n in sizes]
        for i, optimiser in enumerate(optimisers):
            optimiser.step(lying(grads, (0, 1, 2, 4)[i])[1], 0.01)
    for (held, views), optimiser, lead in zip(kept[1:], optimisers[1:], (1, 2, 4)):
        for h, v, w in zip(held, views, kept[0][1]):
            assert torch.equal(v, w) and not torch.equal(v, start[0].cuda())
            assert torch.all(h[:lead] == 7) and torch.all(h[lead + len(v) :] == 7)
        for name in optimiser._state_names():
            assert torch.equal(getattr(optimiser, name), getattr(optimisers[0], name))


def test_parameters_of_inference_mode(ops):  # noqa: F811
    """Stepped there; outside they may not be written, by torch's operators neither, and are not."""
    with torch.inference_mode():
        p = torch.zeros(300).cuda()
        optimiser = ops.AdamW([p])
        optimiser.step([torch.ones(300).cuda()], 0.1)
    after = p.cpu().clone()
    with pytest.raises(RuntimeError, match="inference"):
        optimiser.step([torch.ones(300).cuda()], 0.1)
    assert torch.all(after < 0) and torch.equal(p.cpu(), after) and optimiser.step_count == 1


def test_sizes_past_32_bits(ops):  # noqa: F811
    """More than 2^31 scores, table values, results and parameters: the last rows are the same as by themselves."""
    rows, cols, k = 21_600, 100_003, 16
    g = torch.Generator(device="cuda").manual_seed(3)
    queries, table = (torch.randn(n, k, generator=g, device="cuda") for n in (rows, cols))
    table8 = ops.quantise_rows(table)
    scores = ops.product8(queries, table8, dtype=torch.bfloat16)
    assert scores.numel() > 2**31
    last = slice(rows - 130, rows)
    assert torch.equal(scores[last], ops.product8(queries[last].contiguous(), table8, dtype=torch.bfloat16))
    target = torch.randint(cols, (rows,), generator=g, device="cuda", dtype=torch.int32)
    mask = torch.ones(rows, cols, dtype=torch.bool, device="cuda")
    mask[:, ::3] = False
    result = ops.log_probs(scores, target, mask=mask, n_best=5)
    few = ops.log_probs(scores[last], target[last].contiguous(), mask=mask[last], n_best=5)
    tol = log_tolerance(cols, few.best_log_prob.double())
    assert torch.equal(result.best_index[last], few.best_index) and torch.all((result.best_log_prob[last] - few.best_log_prob).abs() <= tol)
    turned = ops.quantise_rows(scores, transposed=True)
    part = ops.quantise_rows(scores[rows // 128 * 128 :], transposed=True)  # the blocks from there on
    assert torch.equal(turned.values[:, rows // 128 * 128 : rows // 128 * 128 + part.values.shape[1]], part.values)
    straight = ops.quantise_rows(scores)
    assert torch.equal(straight.values[last], ops.quantise_rows(scores[last]).values)
    weight = torch.full((rows,), -1.0, device="cuda")
    grad = ops.log_probs_grad(scores[last].clone(), few, grad_log_prob=weight[last].contiguous())
    ops.log_probs_grad(scores, result, grad_log_prob=weight, out=scores)
    assert torch.all((scores[last].float() - grad.float()).abs() <= 2.0**-7 * grad.float().abs() + 1e-30)  # a neighbouring bf16 number at most
    assert torch.all(scores[last][~mask[last]] == 0)
    del turned, straight, mask, grad
    p = torch.zeros(2**31 + 1000, dtype=torch.bfloat16, device="cuda")
    optimiser = ops.AdamW([p[: 2**31 - 128], p[2**31 - 128 :]], state_bits=8)
    optimiser.step([torch.ones_like(v) for v in optimiser.params], 0.25)
    m, v = optimiser.moments()
    for at in (slice(0, 1000), slice(2**31 - 1000, 2**31 + 1000)):
        assert torch.all((p[at].float() + 0.25).abs() <= 2.0**-8) and torch.all((m[at].float() - 0.1).abs() <= 0.1 / 8) and torch.all((v[at].float() - 0.001).abs() <= 0.001 / 8)
