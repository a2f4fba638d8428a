"""The operators of a softmax over all candidates: log probabilities with entropy and alternatives and their gradient, scores as a
product of 8-bit floating-point rows, and AdamW over many tensors with moments in 8 or 32 bits.

``run`` computes them in elementary torch operations, or, where ``own`` is true, through
``distributed_kge_poplar_b200.device_ops``.  Sizes are those of the repository's presets, benchmark and tests (1387 relations,
768 tails of a batch, tables of 2 500 001 rows and cuts of them, 256-wide rows, 128 or 512 queries, lists of 100) or generic.
"""

import math
import random

import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BLOCK = 128


def _log_probs(**options):
    return dict(dict(do="log_probs", rows=1, cols=1, dtype="float32", scale=1.0, n_best=0, mask=False, count=False, train=False), **options)


def _product(**options):
    return dict(dict(do="product", m=1, n=1, k=1, dtype="bfloat16", out="float32", grad=False), **options)


def _adamw(**options):
    return dict(dict(do="adamw", total=1, tensors=1, bits=32, param="float32", grad="float32", step=10), **options)


def listed():
    return [
        # One query's relation type: the latency of a single small answer.
        _log_probs(name="lp_one_answer", cols=1387, n_best=10),
        # A training batch against its shared tails, known positives masked out, some rows with nothing left.
        _log_probs(name="lp_batch_train", rows=512, cols=768, scale=0.5, mask=True, train=True),
        # A prediction batch against a cut of the table in 16 bits, lists of 100, shards of different sizes.
        _log_probs(name="lp_rank_bf16", rows=128, cols=100_003, dtype="bfloat16", n_best=100, count=True),
        # A few queries against a whole shard: the work of a row is spread over the GPU.
        _log_probs(name="lp_whole_shard", rows=4, cols=2_500_001, n_best=100),
        # The training step of a softmax over all candidates: the largest matrix of scores, read for the loss and for its gradient.
        _log_probs(name="lp_full_train", rows=2048, cols=100_001, dtype="bfloat16", train=True),
        # One query's scores against a cut of the table: as fast as the table can be read.
        _product(name="pr_one_query", m=1, n=250_001, k=256),
        # A prediction batch against the table: as fast as scores can be written.
        _product(name="pr_batch", m=512, n=500_000, k=256, out="bfloat16"),
        # Wide rows on both sides, as in a projection of long features: bound by the tensor cores.
        _product(name="pr_wide", m=4096, n=8192, k=8192, out="bfloat16"),
        # Both gradients of the scores of a training batch: short and long sums, operands laid out anew in each call.
        _product(name="pr_both_grads", m=512, n=100_001, k=256, grad=True),
        # The dense parameters of a model: a few small tensors, where launches are everything.
        _adamw(name="aw_dense", total=700_000, tensors=6),
        # A candidate table and its networks with 8-bit moments and bf16 parameters.
        _adamw(name="aw_table_8bit", total=120_000_000, tensors=12, bits=8, param="bfloat16", grad="bfloat16"),
        # The same in 32 bits.
        _adamw(name="aw_table_32bit", total=60_000_000, tensors=12, grad="bfloat16"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    do = rng.choice(["log_probs", "log_probs", "product", "product", "adamw"])
    if do == "log_probs":
        cols = _log_int(rng, 2, 2_500_001)
        rows = _log_int(rng, 1, max(1, min(4096, 200_000_000 // cols)))
        train = rng.random() < 0.5
        return _log_probs(rows=rows, cols=cols, dtype=rng.choice(list(TYPES)), scale=rng.choice([1.0, 0.25, 1.7]), train=train,
                          n_best=0 if train else rng.choice([0, 1, 10, rng.randint(1, 128)]), mask=rng.random() < 0.4, count=rng.random() < 0.3)
    if do == "product":
        grad = rng.random() < 0.3
        m, n, k = _log_int(rng, 1, 4096), _log_int(rng, 1, 500_000), _log_int(rng, 1, 1024 if grad else 8192)
        while m * n > 250_000_000 or m * n * k > 2.7e11 or n * k > 128_000_000:
            m, n, k = max(1, m // 2), max(1, n - n // 3), max(1, k - k // 3)
        return _product(m=m, n=n, k=k, dtype=rng.choice(list(TYPES)), out=rng.choice(list(TYPES)), grad=grad)
    bits = rng.choice([8, 32])
    return _adamw(total=_log_int(rng, 100, 100_000_000 if bits == 8 else 50_000_000), tensors=rng.randint(1, 20), bits=bits,
                  param=rng.choice(["float32", "bfloat16"]), grad=rng.choice(list(TYPES)), step=_log_int(rng, 1, 100_000))


def work(case):
    size = {"float32": 4, "float16": 2, "bfloat16": 2}
    if case["do"] == "log_probs":
        scores = case["rows"] * case["cols"]
        x = size[case["dtype"]]
        masks = scores if case["mask"] else 0
        bytes_ = scores * x + masks + case["rows"] * (4 + 8 + 8 * case["n_best"] + (4 if case["count"] else 0))
        if case["train"]:
            bytes_ += scores * x + 8 * case["rows"]
        return {"bytes": bytes_, "flops": scores * (16 if case["train"] else 8)}
    if case["do"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        x, out = size[case["dtype"]], size[case["out"]]
        if case["grad"]:
            return {"bytes": (m * n + m * k + n * k) * x + (m + n) * k * out, "flops": 4 * m * n * k}
        return {"bytes": m * k * x + n * k + n * -(-k // BLOCK) + m * n * out, "flops": 2 * m * n * k}
    n, p, g = case["total"], size[case["param"]], size[case["grad"]]
    moments = 16 if case["bits"] == 32 else 4 + 4 / BLOCK + 4  # in 8 bits the moments also come back as the values they stand for
    return {"bytes": n * (2 * p + g + moments), "flops": 12 * n}


# ---------------------------------------------------------------------------
# Inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _sizes(case):
    """The tensors' sizes: one table with most of the values, networks and vectors of all lengths beside it."""
    rng = random.Random(case["total"])
    left, sizes = case["total"], []
    for i in range(case["tensors"] - 1):
        size = max(1, min(left - (case["tensors"] - 1 - i), _log_int(rng, 1, max(1, case["total"] // 8))))
        sizes.append(size)
        left -= size
    return sizes + [left]


def _rows_of_lengths(n, k, generator):
    """Rows of different lengths, as those of frequent and of rare entities."""
    length = torch.exp(torch.randn(n, 1, generator=generator, device="cuda"))
    return torch.randn(n, k, generator=generator, device="cuda") * length


def _product_inputs(case, generator):
    t = TYPES[case["dtype"]]
    queries, table = (_rows_of_lengths(n, case["k"], generator).to(t) for n in (case["m"], case["n"]))
    return queries, table


def prepare(case, seed):
    g = _generator(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    s = dict(case)
    if case["do"] == "log_probs":
        rows, cols = case["rows"], case["cols"]
        s["scores"] = (normal(rows, cols) * 3).to(TYPES[case["dtype"]])
        s["target"] = torch.randint(cols, (rows,), generator=g, device="cuda", dtype=torch.int32)
        s["target"][7::16] = -1  # rows of a padded batch have no target
        s["mask"] = s["count"] = None
        if case["mask"]:
            s["mask"] = torch.rand(rows, cols, generator=g, device="cuda") > 0.05
            s["mask"][3::16] = False  # nothing is left of these rows
        if case["count"]:
            s["count"] = torch.randint(max(1, cols * 2 // 3), cols + 1, (rows,), generator=g, device="cuda", dtype=torch.int32)
        if case["train"]:
            s["grad_log_prob"] = -torch.rand(rows, generator=g, device="cuda") / rows
            s["grad_entropy"] = 0.01 * normal(rows) / rows
        return s
    if case["do"] == "product":
        m, n = case["m"], case["n"]
        s["queries"], table = _product_inputs(case, g)
        if case["grad"]:
            s["table"] = table
            s["grad_scores"] = (normal(m, n) * torch.exp(2 * normal(m, 1)) * 1e-3).to(TYPES[case["dtype"]])
        elif own:
            from distributed_kge_poplar_b200 import device_ops

            s["table8"] = device_ops.quantise_rows(table)
        else:
            s["table8"] = _quantise(table)
        return s
    sizes = _sizes(case)
    first = [0]
    for size in sizes:
        first.append(first[-1] + -(-size // BLOCK) * BLOCK)
    total = first[-1]
    live = torch.zeros(total, dtype=torch.bool, device="cuda")
    for start, size in zip(first, sizes):
        live[start : start + size] = True
    s["step_count"], s["seed"] = case["step"], seed & 0xFFFF
    # the tensors lie in one arena, each from a multiple of 128 values on, as they do where one allocation holds a model
    s["param"] = (normal(total) * 0.05 * live).to(TYPES[case["param"]])
    s["grad"] = (normal(total) * torch.exp(2 * normal(total // BLOCK, 1)).expand(-1, BLOCK).reshape(-1) * 1e-4 * live).to(TYPES[case["grad"]])
    m = s["grad"].float() * torch.rand(total, generator=g, device="cuda")
    v = s["grad"].float().square() * torch.rand(total, generator=g, device="cuda") + 1e-12 * live
    if case["bits"] == 8:
        half = torch.full((total,), 0x8000, dtype=torch.int32, device="cuda")
        m, m_exp = _encode(m, half, 127)
        v, v_exp = _encode(v, half, 255)
        moments = dict(adam_m=m, adam_v=v, m_exponent=m_exp, v_exponent=v_exp)
    else:
        moments = dict(adam_m=m, adam_v=v)
    if own:
        from distributed_kge_poplar_b200 import device_ops

        params, grads = ([s[x][a : a + size] for a, size in zip(first, sizes)] for x in ("param", "grad"))
        optimiser = device_ops.AdamW(params, state_bits=case["bits"], beta_m=0.9, beta_v=0.999, epsilon=1e-8, weight_decay=0.01, seed=s["seed"])
        optimiser.step_count = case["step"]
        for name, value in moments.items():
            getattr(optimiser, name).copy_(value)
        s["optimiser"], s["grads"] = optimiser, grads
    else:
        s.update(moments)
    return s


# ---------------------------------------------------------------------------
# Plain forms


def _quantise(x):
    """Rows as 8-bit floating point (4 exponent bits, 3 of the significand) with a power of two for each 128 values along a row: the
    smallest, from 2^-127 on, that brings the block's largest finite value down to 448."""
    rows, cols = x.shape
    blocks = torch.nn.functional.pad(x.float(), (0, -cols % BLOCK)).view(rows, -1, BLOCK)
    finite = torch.isfinite(blocks)
    largest = torch.where(finite, blocks.abs(), 0.0).amax(2, keepdim=True)
    fraction, exponent = torch.frexp(largest)
    e = (exponent - 8 - (fraction <= 0.875).int()).clamp(min=-127)
    e = torch.where(largest == 0, 0, e)
    codes = (blocks * ((127 - e) << 23).view(torch.float32)).to(torch.float8_e4m3fn)
    codes = torch.where(finite, codes.view(torch.uint8), 0x7F).view(torch.float8_e4m3fn)
    return codes, e, cols


def _values(rows8):
    codes, e, cols = rows8
    power = ((e.to(torch.int64) + 1023) << 52).view(torch.float64).float()
    return (codes.float() * power).flatten(1)[:, :cols]


def _scores(a, b):
    return _values(a) @ _values(b).T


def _live(s):
    x = s["scores"]
    live = ~torch.isneginf(x)
    if s["mask"] is not None:
        live &= s["mask"]
    if s["count"] is not None:
        live &= torch.arange(x.shape[1], device=x.device) < s["count"][:, None]
    return live


def _run_log_probs(s):
    live = _live(s)
    z = torch.where(live, s["scores"].float() * s["scale"], -math.inf)
    largest = z.amax(1, keepdim=True)
    d = z - torch.where(torch.isneginf(largest), 0.0, largest)
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    log_sum = torch.where(torch.isneginf(largest), -math.inf, largest + log_total)
    entropy = torch.where(total > 0, log_total - torch.where(live, e * d, 0.0).sum(1, keepdim=True) / total, 0.0)
    target = s["target"].long()[:, None]
    has = (target >= 0) & (target < z.shape[1])
    at = torch.where(has, target, 0)
    z_target = z.gather(1, at)
    log_prob = torch.where(has, torch.where(torch.isneginf(z_target), -math.inf, z_target - log_sum), 0.0)
    out = {"log_prob": log_prob[:, 0], "entropy": entropy[:, 0]}
    if s["n_best"]:
        raw = torch.where(live & ~torch.isnan(s["scores"]), s["scores"], -math.inf)
        best, index = torch.sort(raw, dim=1, descending=True, stable=True)
        n = min(s["n_best"], z.shape[1])
        none = torch.isneginf(best[:, :n])
        best_log_prob = torch.where(none, -math.inf, best[:, :n].float() * s["scale"] - log_sum)
        rest = (0, s["n_best"] - n)
        out["best_log_prob"] = torch.nn.functional.pad(best_log_prob, rest, value=-math.inf)
        out["best_index"] = torch.nn.functional.pad(torch.where(none, -1, index[:, :n]).int(), rest, value=-1)
    if s["train"]:
        counts = has & ~torch.isneginf(z_target)
        grad_target = torch.where(counts, s["grad_log_prob"][:, None], 0.0)
        log_p = z - torch.where(torch.isneginf(log_sum), 0.0, log_sum)
        p = torch.exp(log_p)
        grad = -grad_target * p - torch.where(live, s["grad_entropy"][:, None] * p * (log_p + entropy), 0.0)
        grad.scatter_add_(1, at, grad_target)
        out["grad"] = (grad * s["scale"]).to(s["scores"].dtype)
    return out


def _encode(x, random16, top):
    """8-bit codes of blocks of 128 values.  A block's exponent is its largest value's, that value rounded up to 3 significand bits;
    code c > 0 stands for the value of that exponent that is top - c steps below the largest (8 steps an octave), 0 for zero; a
    sign where top is 127.  Values are rounded up with the probability of what rounding down would leave; where top is 255 none is
    rounded to zero."""
    bits = x.view(torch.int32) & 0x7FFFFFFF
    exponent = ((bits.view(-1, BLOCK).amax(1, keepdim=True) + 0xFFFFF) >> 23).clamp(min=33 if top == 255 else 16)
    step = ((bits + (random16 << 4)) >> 20).view(-1, BLOCK) - (8 * exponent + 7 - top)
    bits = bits.view(-1, BLOCK)
    lowest = torch.where(bits > 0, 1, 0) if top == 255 else torch.zeros_like(step)
    code = torch.where(step < 1, lowest, step.clamp(max=top))
    if top == 127:
        code = code | torch.where((x.view(-1, BLOCK) < 0) & (code > 0), 128, 0)
    return code.to(torch.uint8).view(-1), exponent.to(torch.uint8).view(-1)


def _decode(code, exponent, top):
    code = code.int().view(-1, BLOCK)
    magnitude = code & top
    value = torch.where(magnitude > 0, (magnitude + (8 * exponent.int()[:, None] + 7 - top)) << 20, 0).view(torch.float32)
    return torch.where(code > top, -value, value).view(-1)


def _mix(x):
    """Mixes the bits of 32-bit numbers held in 64."""
    x = ((x ^ (x >> 16)) * 0x85A308D3) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x6A09E667) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _random32(total, seed, step):
    position = torch.arange(total, device="cuda")
    key = _mix(torch.tensor((seed * 0x9E3779B9 + step * 0xBB67AE85) & 0xFFFFFFFF, device="cuda"))
    return _mix((position * 0x9E3779B9 + (position >> 32) * 0x6A09E667 + key) & 0xFFFFFFFF)


def _run_adamw(s):
    s["step_count"] += 1
    t, rate, beta_m, beta_v = s["step_count"], 1e-3, 0.9, 0.999
    grad, param, eight = s["grad"].float(), s["param"].float(), s["bits"] == 8
    m = _decode(s["adam_m"], s["m_exponent"], 127) if eight else s["adam_m"]
    v = _decode(s["adam_v"], s["v_exponent"], 255) if eight else s["adam_v"]
    m = beta_m * m + (1 - beta_m) * grad
    v = beta_v * v + (1 - beta_v) * grad * grad
    step = rate / (1 - beta_m**t) * m / (torch.sqrt(v) * (1 - beta_v**t) ** -0.5 + 1e-8)
    param = param * (1 - rate * 0.01) - step
    draws = _random32(param.numel(), s["seed"], t) if eight or s["param"].dtype == torch.bfloat16 else None
    if s["param"].dtype == torch.bfloat16:  # rounded up with the probability of what rounding down would leave
        param = ((param.view(torch.int32) + ((draws >> 8) & 0xFFFF).int()) & -0x10000).view(torch.float32)
    s["param"].copy_(param)
    if not eight:
        s["adam_m"].copy_(m)
        s["adam_v"].copy_(v)
        return s["param"], s["adam_m"], s["adam_v"]
    s["adam_m"], s["m_exponent"] = _encode(m, (draws & 0xFFFF).int(), 127)
    s["adam_v"], s["v_exponent"] = _encode(v, (draws >> 16).int(), 255)
    return s["param"], _decode(s["adam_m"], s["m_exponent"], 127).bfloat16(), _decode(s["adam_v"], s["v_exponent"], 255).bfloat16()


def _run_product(s):
    out = TYPES[s["out"]]
    if not s["grad"]:
        return _scores(_quantise(s["queries"]), s["table8"]).to(out)
    grad_queries = _scores(_quantise(s["grad_scores"]), _quantise(s["table"].T))
    grad_table = _scores(_quantise(s["grad_scores"].T), _quantise(s["queries"].T))
    return grad_queries.to(out), grad_table.to(out)


def _run_own(s):
    from distributed_kge_poplar_b200 import device_ops

    if s["do"] == "log_probs":
        r = device_ops.log_probs(s["scores"], s["target"], mask=s["mask"], count=s["count"], scale=s["scale"], n_best=s["n_best"])
        out = {"log_prob": r.log_prob, "entropy": r.entropy}
        if s["n_best"]:
            out["best_log_prob"], out["best_index"] = r.best_log_prob, r.best_index
        if s["train"]:
            out["grad"] = device_ops.log_probs_grad(s["scores"], r, grad_log_prob=s["grad_log_prob"], grad_entropy=s["grad_entropy"])
        return out
    if s["do"] == "product":
        out = TYPES[s["out"]]
        if not s["grad"]:
            return device_ops.product8(s["queries"], s["table8"], dtype=out)
        quantise, grad_scores = device_ops.quantise_rows, s["grad_scores"]
        grad_queries = device_ops.product8(grad_scores, quantise(s["table"], transposed=True), dtype=out)
        grad_table = device_ops.product8(quantise(grad_scores, transposed=True), quantise(s["queries"], transposed=True), dtype=out)
        return grad_queries, grad_table
    optimiser = s["optimiser"]
    optimiser.step(s["grads"], 1e-3)
    if s["bits"] == 8:
        return (s["param"], *optimiser.moments())
    return s["param"], optimiser.adam_m, optimiser.adam_v


def run(state):
    if own:
        return _run_own(state)
    return {"log_probs": _run_log_probs, "product": _run_product, "adamw": _run_adamw}[state["do"]](state)


# ---------------------------------------------------------------------------
# The definitions in 64 bits


def _exact_rows(x):
    """The values that the 8-bit rows of `x` stand for."""
    rows, cols = x.shape
    x = x.double()
    out = torch.empty_like(x)
    for c in range(0, cols, BLOCK):
        part = x[:, c : c + BLOCK]
        largest = part.abs().amax(1, keepdim=True)
        e = torch.ceil(torch.log2(largest / 448))
        e = torch.where(largest > 448 * torch.exp2(e), e + 1, e)  # log2 rounds
        e = torch.where(largest <= 448 * torch.exp2(e - 1), e - 1, e)
        unit = torch.exp2(torch.where(largest == 0, 0.0, e).clamp(min=-127))
        y = part / unit
        octave = torch.floor(torch.log2(y.abs().clamp(min=2.0**-6)))
        octave = torch.where(torch.exp2(octave) > y.abs().clamp(min=2.0**-6), octave - 1, octave)
        grid = torch.exp2(octave - 3)
        out[:, c : c + BLOCK] = torch.round(y / grid) * grid * unit
    return out


def _exact_log_probs(case, s):
    x = s["scores"].double()
    rows, cols = x.shape
    allowed = torch.ones_like(x, dtype=torch.bool) if s["mask"] is None else s["mask"].clone()
    if s["count"] is not None:
        for r, n in enumerate(s["count"].tolist()):
            allowed[r, n:] = False
    z = (x * case["scale"]).masked_fill_(~allowed, -math.inf)
    empty = ~allowed.any(1)
    log_p = torch.log_softmax(z.masked_fill(empty[:, None], 0.0), 1).masked_fill_(~allowed, -math.inf)
    p = log_p.exp()
    plogp = torch.special.xlogy(p, p)
    entropy = -plogp.sum(1)
    target = s["target"].long()
    asked = target >= 0
    picked = log_p.gather(1, target.clamp(min=0)[:, None])[:, 0]
    out = {"log_prob": picked.masked_fill(~asked, 0.0), "entropy": entropy}
    if case["n_best"]:
        take = min(case["n_best"], cols)
        values, index = torch.sort(z, dim=1, descending=True, stable=True)
        values, index = values[:, :take], index[:, :take]
        best = log_p.gather(1, index)
        index = index.int().masked_fill(torch.isneginf(values), -1)
        full = torch.full((rows, case["n_best"]), -math.inf, dtype=torch.float64, device="cuda")
        which = torch.full((rows, case["n_best"]), -1, dtype=torch.int32, device="cuda")
        full[:, :take], which[:, :take] = best, index
        out["best_log_prob"], out["best_index"] = full, which
    if case["train"]:
        counted = asked & ~torch.isneginf(picked)
        g = s["grad_log_prob"].double() * counted
        grad = -(g + s["grad_entropy"].double() * entropy)[:, None] * p - s["grad_entropy"].double()[:, None] * plogp
        where = torch.arange(rows, device="cuda")[counted]
        grad[where, target[counted]] += g[counted]
        out["grad"] = grad * case["scale"]
    return out


def _exact_codes(x, draws16, top):
    """The values that the 8-bit codes of non-negative blocks `x` stand for."""
    x = x.view(-1, BLOCK)
    largest = x.amax(1, keepdim=True)

    def octave(y):
        return torch.frexp(y)[1] - 1.0

    ceiled = torch.ceil(largest / torch.exp2(octave(largest) - 3)) * torch.exp2(octave(largest) - 3)
    highest = torch.where(largest > 0, octave(ceiled), -1000.0).clamp(min=(33 if top == 255 else 16) - 127)
    unit = torch.exp2(octave(x) - 3)
    down = torch.floor(x / unit)
    value = (down + ((x / unit - down) + draws16.view(-1, BLOCK) / 65536 >= 1)) * unit
    steps = 8 * octave(value) + (value / torch.exp2(octave(value)) - 1) * 8  # on the grid, 8 an octave
    lowest = 8 * highest + 7 - top + 1
    floor_value = torch.exp2(torch.floor(lowest / 8)) * (1 + (lowest - 8 * torch.floor(lowest / 8)) / 8)
    kept = torch.where(steps < lowest, floor_value if top == 255 else 0.0, value)
    return torch.where(x > 0, kept, 0.0).view(-1)


def _exact_adamw(case, s):
    t = case["step"] + 1
    seed = s["seed"]
    if case["bits"] == 8:
        signed, unsigned = s["adam_m"].double(), s["adam_v"].double()
        m_top, v_top = (8.0 * (s[x].double() - 127).repeat_interleave(BLOCK) + 7 for x in ("m_exponent", "v_exponent"))

        def value(code, highest, top):
            at = highest - top + code
            return torch.where(code > 0, torch.exp2(torch.floor(at / 8)) * (1 + (at - 8 * torch.floor(at / 8)) / 8), 0.0)

        m = value(signed % 128, m_top, 127) * torch.where(signed >= 128, -1.0, 1.0)
        v = value(unsigned, v_top, 255)
    else:
        m, v = s["adam_m"].double(), s["adam_v"].double()
    g = s["grad"].double()
    m = 0.9 * m + 0.1 * g
    v = 0.999 * v + 0.001 * g**2
    p = s["param"].double()
    p = p - 1e-3 * (0.01 * p + (m / (1 - 0.9**t)) / ((v / (1 - 0.999**t)).sqrt() + 1e-8))
    if case["bits"] == 32 and case["param"] == "float32":
        return p, m, v
    word = 1 << 32
    place = torch.arange(p.numel(), device="cuda")

    def stir(x):
        x = (x ^ (x // (1 << 16))) * 0x85A308D3 % word
        x = (x ^ (x // (1 << 15))) * 0x6A09E667 % word
        return x ^ (x // (1 << 16))

    key = stir(torch.tensor([(seed * 0x9E3779B9 + t * 0xBB67AE85) % word], device="cuda"))
    h = stir((place % word * 0x9E3779B9 + place // word * 0x6A09E667 + key) % word)
    if case["param"] == "bfloat16":
        unit = torch.exp2(torch.frexp(p)[1] - 8.0)
        down = torch.floor(p.abs() / unit)
        p = torch.sign(p) * (down + ((p.abs() / unit - down) + (h // 256 % 65536) / 65536 >= 1)) * unit
    if case["bits"] == 8:
        m = _exact_codes(m.abs(), h % 65536, 127) * torch.sign(m)
        v = _exact_codes(v, h // 65536, 255)
    return p, m, v


def exact(case, seed):
    global own
    mine, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = mine
    if case["do"] == "log_probs":
        return _exact_log_probs(case, s)
    if case["do"] == "adamw":
        return _exact_adamw(case, s)
    if case["grad"]:
        grad_scores = s["grad_scores"]
        return (_exact_rows(grad_scores) @ _exact_rows(s["table"].T).T, _exact_rows(grad_scores.T) @ _exact_rows(s["queries"].T).T)
    queries, table = _product_inputs(case, _generator(seed))
    return _exact_rows(queries) @ _exact_rows(table).T
