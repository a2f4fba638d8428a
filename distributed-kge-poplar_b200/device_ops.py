"""Operators on device tensors: what training and answering with a softmax over all candidates takes.

  log_probs, log_probs_grad   log probability of a given candidate per row of scores, entropy and the n_best alternatives
  quantise_rows, product8     scores as a product of rows in 8-bit floating point with a power of two for each 128 values
  AdamW                       one step over many tensors, moments in 32 or in 8 bits

They are the ``kge_op_*`` entry points for device arrays of ``include/kge_b200.h``, which states their arithmetic, with torch
tensors for the arrays.  Work is queued on torch's current stream of the tensors' device, results and workspaces come from torch's
allocator, and nothing is kept between calls: calls may be captured into CUDA graphs and may run on several streams at once.  A
tensor used on another stream than the one it was made on has to be kept until that stream is done with it, as with torch's own
operators.  Wrong arguments raise ``ValueError`` before anything is launched; indices, counts and masks live on the device and are
not read back: a target outside the columns counts as none.  The reference has no counterpart; its softmax is over the tails of a
batch (src/poplar_kge.cpp:575-600), its lists come without probabilities (:812-855), and it updates one parameter after another
(src/fructose/frnn.cpp:61-90).
"""

from __future__ import annotations

import contextlib
import ctypes as C

from typing import Any, Dict, List, Optional, Sequence, Tuple, Union

import torch

from . import capi

FLOAT_TYPES = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16}
BLOCK = 128

_NO_GUARD = contextlib.nullcontext()


def _guard(device: torch.device):
    """Makes the tensors' device the current one for a launch."""
    return _NO_GUARD if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _tensor(what: str, t: Any, types, shape: Optional[Tuple[int, ...]] = None, device: Optional[torch.device] = None) -> None:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{what} must be a tensor, not {type(t).__name__}")
    if t.dtype not in types:
        raise ValueError(f"{what} must be {' or '.join(str(x) for x in types)}, not {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{what} must be on a GPU, not on {t.device}")
    if device is not None and t.device != device:
        raise ValueError(f"{what} is on {t.device}, the other tensors on {device}")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{what} has shape {tuple(t.shape)}, expected {shape}")


def _matrix(what: str, t: Any, types, shape: Optional[Tuple[int, int]] = None, device: Optional[torch.device] = None) -> None:
    _tensor(what, t, types, shape, device)
    if t.dim() != 2:
        raise ValueError(f"{what} must have two dimensions, not {t.dim()}")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{what} must be contiguous along its rows, not {t.stride(1)} apart")


def _rows_apart(t: torch.Tensor) -> int:
    """A matrix's row stride; that of a single row or an empty matrix says nothing."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _span(t: torch.Tensor) -> Tuple[int, int]:
    first = t.data_ptr()
    return first, first + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _refuse_overlap(what: str, out: torch.Tensor, other: torch.Tensor) -> None:
    if out.numel() and other.numel():
        (a, b), (c, d) = _span(out), _span(other)
        if a < d and c < b:
            raise ValueError(f"{what} overlap in memory")


# ---------------------------------------------------------------------------
# Log probabilities


class LogProbs:
    """What :func:`log_probs` found, and what :func:`log_probs_grad` needs of it.

    log_prob       [rows]          of the target: 0 where there is none, -inf where it is not live
    entropy        [rows]          of the distribution over the live columns, 0 where there are none
    log_sum        [rows]          log of the sum of exp(scale * score), -inf where no column is live
    best_log_prob  [rows, n_best]  highest score first, equal scores by the lower column, -inf past the live columns
    best_index     [rows, n_best]  int32, -1 past the live columns
    """

    __slots__ = ("log_prob", "entropy", "log_sum", "best_log_prob", "best_index", "row_state", "target", "mask", "count", "scale")


def _scores(scores, target, mask, count, scale) -> capi.Scores:
    _matrix("scores", scores, FLOAT_TYPES)
    rows, cols = scores.shape
    device = scores.device
    s = capi.Scores()
    s.x, s.float_type, s.rows, s.cols, s.row_stride = scores.data_ptr(), FLOAT_TYPES[scores.dtype], rows, cols, _rows_apart(scores)
    s.scale = scale
    for name, index in (("target", target), ("count", count)):
        if index is not None:
            _tensor(name, index, (torch.int32,), (rows,), device)
            if rows > 1 and index.stride(0) != 1:
                raise ValueError(f"{name} must be contiguous")
            setattr(s, name, index.data_ptr())
    if mask is not None:
        _matrix("mask", mask, (torch.bool, torch.uint8), (rows, cols), device)
        s.mask, s.mask_stride = mask.data_ptr(), mask.stride(0) if rows > 1 else cols
    return s


def log_probs(scores: torch.Tensor, target: Optional[torch.Tensor] = None, *, mask: Optional[torch.Tensor] = None,
              count: Optional[torch.Tensor] = None, scale: float = 1.0, n_best: int = 0) -> LogProbs:
    """Log probability of ``target``, entropy and the ``n_best`` (at most 128) most probable columns under
    softmax(scale * scores) over each row's live columns, in one pass over the scores.

    scores  [rows, cols] float32, float16 or bfloat16, contiguous along a row
    target  [rows] int32; negative (or past the columns): none
    mask    [rows, cols] bool or uint8, false: not live; may be one row expanded
    count   [rows] int32: columns from count[r] on are not live
    A score of -inf is not live.  Masked places may hold anything; a live NaN or +inf makes a row's results NaN.
    """
    if not 0 <= n_best <= 128:
        raise ValueError(f"n_best must be between 0 and 128, not {n_best}")
    s = _scores(scores, target, mask, count, scale)
    rows = scores.shape[0]
    device = scores.device
    r = LogProbs()
    r.target, r.mask, r.count, r.scale = target, mask, count, scale
    lib = capi.load_library()
    with _guard(device):
        r.log_prob, r.entropy, r.log_sum = torch.empty((3, rows), dtype=torch.float32, device=device).unbind(0)
        r.row_state = torch.empty((rows, 4), dtype=torch.float32, device=device)
        r.best_log_prob = torch.empty((rows, n_best), dtype=torch.float32, device=device)
        r.best_index = torch.empty((rows, n_best), dtype=torch.int32, device=device)
        out = capi.LogProbsOut(r.log_prob.data_ptr(), r.entropy.data_ptr(), r.log_sum.data_ptr(), r.row_state.data_ptr(), n_best,
                               r.best_log_prob.data_ptr(), r.best_index.data_ptr())
        wanted = lib.kge_op_log_probs_workspace(rows, scores.shape[1], n_best)
        workspace = torch.empty(wanted, dtype=torch.uint8, device=device) if wanted else None
        capi._op_check(lib.kge_op_log_probs(C.byref(s), C.byref(out), workspace.data_ptr() if wanted else None, wanted, _stream(device)))
    return r


def log_probs_grad(scores: torch.Tensor, result: LogProbs, *, grad_log_prob: Optional[torch.Tensor] = None,
                   grad_entropy: Optional[torch.Tensor] = None, grad_best: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient with respect to ``scores`` of the outputs of ``result = log_probs(scores, ...)``, given those of
    ``result.log_prob`` [rows], ``result.entropy`` [rows] and ``result.best_log_prob`` [rows, n_best] (float32; None: zero).

    ``out`` (the scores' type and shape) may be ``scores`` itself.  Columns that are not live, rows without live columns, and
    targets and alternatives that are not live have no gradient."""
    s = _scores(scores, result.target, result.mask, result.count, result.scale)
    rows, n_best = result.best_index.shape
    if tuple(scores.shape)[0] != rows:
        raise ValueError(f"scores have {scores.shape[0]} rows, the result {rows}")
    device = scores.device
    shapes = {"grad_log_prob": (grad_log_prob, (rows,)), "grad_entropy": (grad_entropy, (rows,)), "grad_best": (grad_best, (rows, n_best))}
    with _guard(device):
        keep: List[Optional[torch.Tensor]] = []
        for name, (g, shape) in shapes.items():
            if g is not None:
                _tensor(name, g, (torch.float32,), shape, device)
                g = g.contiguous()
            keep.append(g)
        if out is None:
            out = torch.empty(scores.shape, dtype=scores.dtype, device=device)
        else:
            _matrix("out", out, (scores.dtype,), tuple(scores.shape), device)
            if out.data_ptr() != scores.data_ptr() or _rows_apart(out) != _rows_apart(scores):
                _refuse_overlap("out and scores", out, scores)
        pointers = [g.data_ptr() if g is not None else None for g in keep]
        capi._op_check(capi.load_library().kge_op_log_probs_grad(
            C.byref(s), result.row_state.data_ptr(), pointers[0], pointers[1], n_best, result.best_index.data_ptr(), pointers[2],
            out.data_ptr(), _rows_apart(out), _stream(device)))
    return out


# ---------------------------------------------------------------------------
# Products of 8-bit rows


class Rows8:
    """``rows`` x ``cols`` values in 8-bit floating point with a power of two for each 128 values along a row, laid out as
    ``kge_op_quantise_rows`` states.  One byte and 1/128 a value."""

    __slots__ = ("values", "exponents", "rows", "cols")

    def __init__(self, values: torch.Tensor, exponents: torch.Tensor, rows: int, cols: int):
        self.values, self.exponents, self.rows, self.cols = values, exponents, rows, cols

    def dequantise(self) -> torch.Tensor:
        """The float32 values that the rows stand for."""
        blocks = -(-self.cols // BLOCK)
        # [row tile, group, row % 32, row / 32, block % 4] -> [row, block]
        e = self.exponents.view(-(-self.rows // 128), -1, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-(-self.rows // 128) * 128, -1)
        e = e[: self.rows, :blocks].int()
        power = torch.where(e > 0, e << 23, 1 << 22).view(torch.float32)  # 2^-127 is a subnormal fp32
        return self.values.view(torch.float8_e4m3fn)[:, : self.cols].float() * power.repeat_interleave(BLOCK, 1)[:, : self.cols]


def quantise_rows(x: torch.Tensor, *, transposed: bool = False) -> Rows8:
    """The rows of ``x`` [rows, cols] (float32, float16, bfloat16; contiguous along a row) in 8-bit floating point; with
    ``transposed`` its columns, in one pass over ``x`` as it lies.  A block's power of two is the smallest, from 2^-127 on, that
    brings its largest finite value down to 448; NaN and infinities become NaN."""
    _matrix("x", x, FLOAT_TYPES)
    rows, cols = reversed(x.shape) if transposed else x.shape
    n_values, n_exponents = C.c_size_t(), C.c_size_t()
    lib = capi.load_library()
    capi._op_check(lib.kge_op_rows8_bytes(rows, cols, C.byref(n_values), C.byref(n_exponents)))
    device = x.device
    with _guard(device):
        values = torch.empty((rows, n_values.value // rows if rows else 0), dtype=torch.uint8, device=device)
        exponents = torch.empty(n_exponents.value, dtype=torch.uint8, device=device)
        capi._op_check(lib.kge_op_quantise_rows(x.data_ptr(), FLOAT_TYPES[x.dtype], x.shape[0], x.shape[1], _rows_apart(x), int(transposed),
                                                values.data_ptr(), exponents.data_ptr(), _stream(device)))
    return Rows8(values, exponents, rows, cols)


def product8(a: Union[torch.Tensor, Rows8], b: Union[torch.Tensor, Rows8], *, dtype: torch.dtype = torch.float32,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[i, j] = sum_c a[i, c] * b[j, c]`` [a.rows, b.rows] of rows in 8-bit floating point, summed in 32 bits; a tensor is
    quantised by the call.  Scores of queries ``a`` against a table ``b``; their gradients are the products
    ``product8(grad, quantise_rows(b, transposed=True))`` and
    ``product8(quantise_rows(grad, transposed=True), quantise_rows(a, transposed=True))``."""
    a = a if isinstance(a, Rows8) else quantise_rows(a)
    b = b if isinstance(b, Rows8) else quantise_rows(b)
    if a.cols != b.cols:
        raise ValueError(f"rows of {a.cols} and of {b.cols} values")
    device = a.values.device
    if b.values.device != device:
        raise ValueError(f"a is on {device}, b on {b.values.device}")
    if out is not None:
        _matrix("out", out, FLOAT_TYPES, (a.rows, b.rows), device)
        dtype = out.dtype
    elif dtype not in FLOAT_TYPES:
        raise ValueError(f"dtype must be {' or '.join(str(x) for x in FLOAT_TYPES)}, not {dtype}")
    lib = capi.load_library()
    with _guard(device):
        if out is None:
            out = torch.empty((a.rows, b.rows), dtype=dtype, device=device)
        wanted = lib.kge_op_product8_workspace(a.rows, b.rows, a.cols)
        workspace = torch.empty(wanted, dtype=torch.uint8, device=device) if wanted else None
        capi._op_check(lib.kge_op_product8(a.values.data_ptr(), a.exponents.data_ptr(), a.rows, b.values.data_ptr(), b.exponents.data_ptr(),
                                           b.rows, a.cols, out.data_ptr(), FLOAT_TYPES[dtype], _rows_apart(out),
                                           workspace.data_ptr() if wanted else None, wanted, _stream(device)))
    return out


# ---------------------------------------------------------------------------
# AdamW


class AdamW:
    """Adam with decoupled weight decay over many tensors in one launch (256 tensors at a time).

    params          contiguous tensors, all float32 or all bfloat16 (then rounded stochastically), updated in place
    state_bits      32: float32 moments; 8: a byte each with one exponent for each 128 values, rounded stochastically
    seed            of the stochastic rounding; the draws depend on it, the step's number and a value's place alone

    The moments of all tensors lie in ``adam_m`` and ``adam_v`` (8 bits: with ``m_exponent``, ``v_exponent``), tensor i's from
    ``first[i]`` on, a multiple of 128; :meth:`state` and :meth:`load_state` read and set them with the step count.
    """

    def __init__(self, params: Sequence[torch.Tensor], *, state_bits: int = 32, beta_m: float = 0.9, beta_v: float = 0.999,
                 epsilon: float = 1e-8, weight_decay: float = 0.0, seed: int = 0):
        self.params = list(params)
        if not self.params:
            raise ValueError("AdamW needs at least one tensor")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, not {state_bits}")
        if not (0 <= beta_m < 1 and 0 <= beta_v < 1):
            raise ValueError(f"beta_m and beta_v must be at least 0 and below 1, not {beta_m} and {beta_v}")
        if not epsilon > 0:
            raise ValueError(f"epsilon must be positive, not {epsilon}")
        first = self.params[0]
        for i, p in enumerate(self.params):
            _tensor(f"parameter {i}", p, (torch.float32, torch.bfloat16), device=self.params[0].device if i else None)
            if p.dtype != first.dtype:
                raise ValueError(f"parameter {i} is {p.dtype}, parameter 0 {first.dtype}: an optimiser for each type")
            if not p.is_contiguous():
                raise ValueError(f"parameter {i} must be contiguous")
        spans = sorted((*_span(p), i) for i, p in enumerate(self.params) if p.numel())
        for (_, end, i), (begin, _, j) in zip(spans, spans[1:]):
            if begin < end:
                raise ValueError(f"parameters {i} and {j} overlap in memory")
        self.device, self.state_bits = first.device, state_bits
        self.beta_m, self.beta_v, self.epsilon, self.weight_decay, self.seed = beta_m, beta_v, epsilon, weight_decay, seed & 0xFFFFFFFF
        self.step_count = 0
        self.first: List[int] = []
        total = 0
        for p in self.params:
            self.first.append(total)
            total += -(-p.numel() // BLOCK) * BLOCK
        kind = torch.float32 if state_bits == 32 else torch.uint8
        self.adam_m, self.adam_v = (torch.zeros(total, dtype=kind, device=self.device) for _ in range(2))
        if state_bits == 8:
            self.m_exponent, self.v_exponent = (torch.full((total // BLOCK,), least, dtype=torch.uint8, device=self.device) for least in (16, 33))
        else:
            self.m_exponent = self.v_exponent = None
        self._tensors = (capi.AdamWTensor * len(self.params))()
        for t, p, start in zip(self._tensors, self.params, self.first):
            t.size, t.first = p.numel(), start
        self._versions = [p for p in self.params if p.requires_grad]

    def _scalars(self, learning_rate: float, step: int) -> Tuple[float, float, float, int]:
        return (1.0 - learning_rate * self.weight_decay, learning_rate / (1.0 - self.beta_m**step), (1.0 - self.beta_v**step) ** -0.5,
                capi.load_library().kge_op_adamw_key(self.seed, step & 0xFFFFFFFF))

    def new_schedule(self) -> torch.Tensor:
        """Device memory for :meth:`advance`, read by steps that are captured into a graph."""
        return torch.zeros(4, dtype=torch.float32, device=self.device)

    def advance(self, schedule: torch.Tensor, learning_rate: float) -> None:
        """Counts a step and writes what it needs into ``schedule``: before each replay of a graph that holds
        ``step(grads, schedule=schedule)``."""
        _tensor("schedule", schedule, (torch.float32,), (4,), self.device)
        if not schedule.is_contiguous():
            raise ValueError("schedule must be contiguous")
        decay, step_size, correction, key = self._scalars(learning_rate, self.step_count + 1)
        words = torch.tensor([decay, step_size, correction, 0.0], dtype=torch.float32)
        words.view(torch.int32)[3] = key - (1 << 32) if key >> 31 else key
        schedule.copy_(words)
        self.step_count += 1

    def step(self, grads: Sequence[Optional[torch.Tensor]], learning_rate: Optional[float] = None, *,
             schedule: Optional[torch.Tensor] = None, grad_scale: float = 1.0) -> None:
        """One step with ``grads`` (one per parameter, all of one type, contiguous; None: the parameter and its moments stay as they
        are), each multiplied by ``grad_scale``.  Either ``learning_rate`` is given and the step is counted, or ``schedule``, which
        :meth:`advance` has written.  A step under stream capture needs a schedule: its replays would repeat one step's number."""
        if (learning_rate is None) == (schedule is None):
            raise ValueError("step() takes a learning_rate or a schedule")
        if len(grads) != len(self.params):
            raise ValueError(f"{len(grads)} gradients for {len(self.params)} parameters")
        kind = None
        for i, (t, p, g) in enumerate(zip(self._tensors, self.params, grads)):
            if g is None:
                t.size = 0
                continue
            if kind is None:
                kind = g.dtype
                if kind not in FLOAT_TYPES:
                    raise ValueError(f"gradient {i} must be {' or '.join(str(x) for x in FLOAT_TYPES)}, not {kind}")
            if g.dtype != kind or g.device != self.device or g.shape != p.shape or not g.is_contiguous():
                _tensor(f"gradient {i}", g, (kind,), tuple(p.shape), self.device)
                raise ValueError(f"gradient {i} must be contiguous")
            t.size, t.param, t.grad = p.numel(), p.data_ptr(), g.data_ptr()
        if kind is None:
            kind = torch.float32
        args = capi.AdamWArgs()
        if schedule is not None:
            _tensor("schedule", schedule, (torch.float32,), (4,), self.device)
            args.schedule = schedule.data_ptr()
        else:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a step under stream capture takes a schedule instead of a learning_rate")
            args.decay, args.step_size, args.inv_sqrt_correction, args.key = self._scalars(learning_rate, self.step_count + 1)
        args.param_type, args.grad_type, args.state_bits = FLOAT_TYPES[self.params[0].dtype], FLOAT_TYPES[kind], self.state_bits
        args.adam_m, args.adam_v = self.adam_m.data_ptr(), self.adam_v.data_ptr()
        if self.state_bits == 8:
            args.m_exponent, args.v_exponent = self.m_exponent.data_ptr(), self.v_exponent.data_ptr()
        args.beta_m, args.beta_v, args.epsilon, args.grad_scale = self.beta_m, self.beta_v, self.epsilon, grad_scale
        with _guard(self.device):
            capi._op_check(capi.load_library().kge_op_adamw(C.byref(args), self._tensors, len(self.params), _stream(self.device)))
        for p in self._versions:  # as any operator that writes in place tells autograd
            torch.autograd.graph.increment_version(p)
        if schedule is None:
            self.step_count += 1

    def moments(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """Both moments as values: float32 ones as they are, 8-bit ones as bfloat16, which holds them exactly."""
        if self.state_bits == 32:
            return self.adam_m, self.adam_v
        with _guard(self.device):
            m, v = (torch.empty(self.adam_m.shape, dtype=torch.bfloat16, device=self.device) for _ in range(2))
            capi._op_check(capi.load_library().kge_op_adamw_moments(
                self.adam_m.data_ptr(), self.m_exponent.data_ptr(), self.adam_v.data_ptr(), self.v_exponent.data_ptr(),
                self.adam_m.numel(), m.data_ptr(), v.data_ptr(), _stream(self.device)))
        return m, v

    def state(self) -> Dict[str, Any]:
        """The moments as they are held and the step count, for a checkpoint."""
        names = ("adam_m", "adam_v") + (("m_exponent", "v_exponent") if self.state_bits == 8 else ())
        return dict(step_count=self.step_count, seed=self.seed, **{name: getattr(self, name).clone() for name in names})

    def load_state(self, state: Dict[str, Any]) -> None:
        """Sets what :meth:`state` gave for an optimiser of the same tensors and state_bits."""
        names = ("adam_m", "adam_v") + (("m_exponent", "v_exponent") if self.state_bits == 8 else ())
        for name in names:
            mine, given = getattr(self, name), state.get(name)
            if given is None or given.shape != mine.shape or given.dtype != mine.dtype:
                raise ValueError(f"'{name}' of the state does not fit this optimiser")
        for name in names:
            getattr(self, name).copy_(state[name])
        self.step_count, self.seed = int(state["step_count"]), int(state["seed"])
