"""The operators of ``device_ops`` from their definitions, in 64 bits on the CPU."""

import math

import torch

BLOCK = 128


def live_columns(x, mask=None, count=None):
    live = ~torch.isneginf(x)
    if mask is not None:
        live = live & mask.bool()
    if count is not None:
        live = live & (torch.arange(x.shape[1])[None] < count[:, None].long())
    return live


def log_probs(x, target=None, mask=None, count=None, scale=1.0, n_best=0):
    """Everything that device_ops.log_probs returns, with p and log p."""
    rows, cols = x.shape
    live = live_columns(x, mask, count)
    z = torch.where(live, x.double() * scale, -math.inf)
    some = live.any(1)
    top = torch.where(some, z.amax(1) if cols else torch.zeros(rows).double(), 0.0)
    e = torch.where(live, torch.exp(z - top[:, None]), 0.0)
    total = e.sum(1)
    log_sum = torch.where(some, top + torch.log(total), -math.inf)
    # not z - log_sum: next to the type's lowest value that sum is the value itself
    log_p = torch.where(live, (z - top[:, None]) - torch.where(some, torch.log(total), 0.0)[:, None], -math.inf)
    p = torch.where(live, torch.exp(log_p), 0.0)
    entropy = -torch.where(p > 0, p * log_p, torch.where(torch.isnan(p), p, 0.0)).sum(1)
    log_prob = torch.zeros(rows).double()
    if target is not None:
        for r in range(rows):
            t = int(target[r])
            if 0 <= t < cols:
                log_prob[r] = log_p[r, t]
    best = torch.full((rows, n_best), -math.inf).double()
    index = torch.full((rows, n_best), -1, dtype=torch.int32)
    for r in range(rows if n_best else 0):
        at = torch.nonzero(live[r] & ~torch.isnan(x[r]))[:, 0]
        order = at[torch.sort(x[r, at].double(), descending=True, stable=True)[1]][:n_best]
        index[r, : len(order)] = order.int()
        best[r, : len(order)] = log_p[r, order]
    return dict(log_prob=log_prob, entropy=entropy, log_sum=log_sum, best_log_prob=best, best_index=index, p=p, log_p=log_p, live=live)


def log_probs_grad(x, form, target, scale, grad_log_prob=None, grad_entropy=None, grad_best=None):
    rows, cols = x.shape
    p, log_p, live = form["p"], form["log_p"], form["live"]
    given = torch.zeros(rows, cols).double()
    if grad_log_prob is not None:
        for r in range(rows):
            t = -1 if target is None else int(target[r])
            if 0 <= t < cols and live[r, t]:
                given[r, t] += float(grad_log_prob[r])
    if grad_best is not None:
        for r in range(rows):
            for i, c in enumerate(form["best_index"][r].tolist()):
                if c >= 0:
                    given[r, c] += float(grad_best[r, i])
    grad = given - given.sum(1, keepdim=True) * p
    if grad_entropy is not None:
        grad -= grad_entropy.double()[:, None] * torch.where(p > 0, p * (log_p + form["entropy"][:, None]), torch.where(torch.isnan(p), p, 0.0))
    return scale * torch.where(live, grad, 0.0)


def e4m3(y):
    """To 3 bits after the leading one, exponents from -6 on, ties to even."""
    octave = torch.floor(torch.log2(y.abs().clamp(min=2.0**-6)))
    octave = torch.where(torch.exp2(octave) > y.abs().clamp(min=2.0**-6), octave - 1, octave)
    octave = torch.where(torch.exp2(octave + 1) <= y.abs(), octave + 1, octave)
    step = torch.exp2(octave - 3)
    return torch.round(y / step) * step


def rows8(x):
    """(values, exponents [rows, blocks]) of the rows of x."""
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    padded = torch.zeros(rows, blocks * BLOCK).double()
    padded[:, :cols] = x.double()
    padded = padded.view(rows, blocks, BLOCK)
    finite = torch.isfinite(padded)
    largest = torch.where(finite, padded.abs(), 0.0).amax(2)
    exponent = torch.zeros_like(largest)
    for i in torch.nonzero(largest):
        value = float(largest[tuple(i)])
        e = math.frexp(value)[1] - 10
        while value > 448 * 2.0**e:
            e += 1
        exponent[tuple(i)] = max(e, -127)
    power = torch.exp2(exponent)[:, :, None]
    values = torch.where(finite, e4m3(torch.where(finite, padded / power, 0.0)) * power, math.nan)
    return values.view(rows, -1)[:, :cols], exponent.int()


def mix(x):
    x = ((x ^ (x >> 16)) * 0x85A308D3) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x6A09E667) & 0xFFFFFFFF
    return x ^ (x >> 16)


def draws(position, seed, step):
    key = mix((seed * 0x9E3779B9 + step * 0xBB67AE85) & 0xFFFFFFFF)
    return mix((position * 0x9E3779B9 + (position >> 32) * 0x6A09E667 + key) & 0xFFFFFFFF)


def adamw_values(code, exponent, top):
    """The values of codes whose blocks have the given exponents."""
    code = code.long().view(-1, BLOCK)
    magnitude, e = code & top, exponent.long()[:, None]
    at = magnitude + 8 * e + 7 - top  # octaves of 8 steps
    value = torch.where(magnitude > 0, torch.exp2((at // 8 - 127).double()) * (1 + (at % 8).double() / 8), 0.0)
    value = torch.where(code > top, -value, value)
    return torch.where(e == 255, math.nan, value).view(-1)


def adamw_codes(x, random16, top):
    """(codes, exponents) of blocks of 128 values, rounded up with the probability random16 / 2^16 decides on."""
    x = x.double().view(-1, BLOCK)
    random16 = random16.view(-1, BLOCK)
    fraction, octave = torch.frexp(x.abs())  # fraction in [1/2, 1)
    steps = 8 * (octave.double() - 1 + 127) + (2 * fraction - 1) * 8  # position on the grid, in eighths of an octave
    steps = torch.where(x == 0, -1e9, steps)
    rounded = torch.floor(steps + random16.double() / 65536)
    exponent = torch.floor(torch.ceil(steps.amax(1)) / 8).clamp(min=33 if top == 255 else 16, max=255)
    code = rounded - (8 * exponent[:, None] + 7 - top)
    least = torch.where(x > 0, 1.0, 0.0) if top == 255 else torch.zeros_like(code)
    code = torch.minimum(torch.maximum(code, least), torch.tensor(float(top)).double())
    code = code.long() | torch.where((x < 0) & (code > 0) & (top == 127), 128, 0)
    return code.view(-1), exponent.long()
