"""Operators on device tensors: what training and answering with a softmax over all candidates takes.

  log_probs, log_probs_grad   log probability of a given candidate per row of scores, entropy and the n_best alternatives
  quantise_rows, product8     scores as a product of rows in 8-bit floating point with a power of two for each 128 values
  check_product8              whether the product's bounded waits have all ended well
  AdamW                       one step over many tensors, moments in 32 or in 8 bits

They are the ``kge_op_*`` entry points for device arrays of ``include/kge_b200.h``, which states their arithmetic, with torch
tensors for the arrays (``libkge_torch``, built beside this file).  Work is queued on torch's current stream of the tensors' device,
results and workspaces come from torch's allocator, and nothing is kept between calls: calls may be captured into CUDA graphs and may
run on several streams at once.  A tensor used on another stream than the one it was made on has to be kept until that stream is done
with it, as with torch's own operators.  Wrong arguments raise ``ValueError`` before anything is launched; indices, counts and masks
live on the device and are not read back: a target outside the columns counts as none.  The reference has no counterpart; its softmax
is over the tails of a batch (src/poplar_kge.cpp:575-600), its lists come without probabilities (:812-855), and it updates one
parameter after another (src/fructose/frnn.cpp:61-90).
"""

from __future__ import annotations

import contextlib
import importlib.util
import operator
from pathlib import Path
from typing import Any, Dict, Optional, Sequence, Tuple, Union

import torch

from . import capi


def _load_module():
    """Import the compiled ``libkge_torch`` that sits beside this file (no fallback)."""
    capi.load_library()
    candidates = sorted(Path(__file__).resolve().parent.glob("libkge_torch*.so"))
    if not candidates:
        raise ImportError("libkge_torch is missing: build it with `python distributed-kge-poplar_b200/build.py`")
    spec = importlib.util.spec_from_file_location("libkge_torch", candidates[0])
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


_module = _load_module()
LogProbs, Rows8 = _module.LogProbs, _module.Rows8
BLOCK = 128


def _must_be_tensor(what: str, t: Any) -> None:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{what} must be a tensor, not {type(t).__name__}")


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
    _must_be_tensor("scores", scores)
    return _module.log_probs(scores, target, mask, count, scale, n_best)


def log_probs_grad(scores: torch.Tensor, result: LogProbs, *, grad_log_prob: Optional[torch.Tensor] = None,
                   grad_entropy: Optional[torch.Tensor] = None, grad_best: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient with respect to ``scores`` of the outputs of ``result = log_probs(scores, ...)``, given those of
    ``result.log_prob`` [rows], ``result.entropy`` [rows] and ``result.best_log_prob`` [rows, n_best] (float32; None: zero).

    ``out`` (the scores' type and shape) may be ``scores`` itself.  Columns that are not live, rows without live columns, and
    targets and alternatives that are not live have no gradient."""
    _must_be_tensor("scores", scores)
    return _module.log_probs_grad(scores, result, grad_log_prob, grad_entropy, grad_best, out)


def _dequantise(self: Rows8) -> torch.Tensor:
    """The float32 values that the rows stand for."""
    blocks = -(-self.cols // BLOCK)
    # [row tile, group, row % 32, row / 32, block % 4] -> [row, block]
    e = self.exponents.view(-(-self.rows // 128), -(-blocks // 4), 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-(-self.rows // 128) * 128, -(-blocks // 4) * 4)
    e = e[: self.rows, :blocks].int()
    power = torch.where(e > 0, e << 23, 1 << 22).view(torch.float32)  # 2^-127 is a subnormal fp32
    return self.values.view(torch.float8_e4m3fn)[:, : self.cols].float() * power.repeat_interleave(BLOCK, 1)[:, : self.cols]


Rows8.dequantise = _dequantise


def quantise_rows(x: torch.Tensor, *, transposed: bool = False) -> Rows8:
    """The rows of ``x`` [rows, cols] (float32, float16, bfloat16; contiguous along a row) in 8-bit floating point; with
    ``transposed`` its columns, in one pass over ``x`` as it lies.  A block's power of two is the smallest, from 2^-127 on, that
    brings its largest finite value down to 448; NaN and infinities become NaN."""
    _must_be_tensor("x", x)
    return _module.quantise_rows(x, transposed)


def product8(a: Union[torch.Tensor, Rows8], b: Union[torch.Tensor, Rows8], *, dtype: torch.dtype = torch.float32,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[i, j] = sum_c a[i, c] * b[j, c]`` [a.rows, b.rows] of rows in 8-bit floating point, summed in 32 bits; a tensor is
    quantised by the call.  Scores of queries ``a`` against a table ``b``; their gradients are the products
    ``product8(grad, quantise_rows(b, transposed=True))`` and
    ``product8(quantise_rows(grad, transposed=True), quantise_rows(a, transposed=True))``.  :func:`check_product8` tells whether the
    device has kept to it."""
    a = a if isinstance(a, Rows8) else quantise_rows(a)
    b = b if isinstance(b, Rows8) else quantise_rows(b)
    return _module.product8(a, b, dtype, out)


def check_product8(device: Union[torch.device, int, None] = None) -> None:
    """Waits for the device (None: the current one) and raises ``RuntimeError`` if a wait inside a :func:`product8` on it has given up
    since the last question: the product's waits are bounded, and one that ran out leaves results that are not to be used."""
    lib = capi.load_library()
    with contextlib.nullcontext() if device is None else torch.cuda.device(device):
        status = lib.kge_op_product8_status()
    if status != capi.OK:
        raise RuntimeError(lib.kge_last_error(None).decode())


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
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, not {state_bits}")
        if not (0 <= beta_m < 1 and 0 <= beta_v < 1):
            raise ValueError(f"beta_m and beta_v must be at least 0 and below 1, not {beta_m} and {beta_v}")
        if not torch.finfo(torch.float32).tiny <= epsilon <= torch.finfo(torch.float32).max:
            raise ValueError(f"epsilon must be positive and a normal number in float32, not {epsilon}")
        for i, p in enumerate(self.params):
            _must_be_tensor(f"parameter {i}", p)
        self._tensors = _module.AdamWTensors(self.params)
        self.device, self.state_bits = self.params[0].device, state_bits
        self.beta_m, self.beta_v, self.epsilon, self.weight_decay, self.seed = beta_m, beta_v, epsilon, weight_decay, seed & 0xFFFFFFFF
        self.step_count = 0
        self.first, total = self._tensors.first, self._tensors.total
        kind = torch.float32 if state_bits == 32 else torch.uint8
        self.adam_m, self.adam_v = (torch.zeros(total, dtype=kind, device=self.device) for _ in range(2))
        self.m_exponent = self.v_exponent = None
        if state_bits == 8:
            self.m_exponent, self.v_exponent = (torch.full((total // BLOCK,), least, dtype=torch.uint8, device=self.device) for least in (16, 33))

    def _scalars(self, learning_rate: float, step: int) -> Tuple[float, float, float, int]:
        return (1.0 - learning_rate * self.weight_decay, learning_rate / (1.0 - self.beta_m**step), (1.0 - self.beta_v**step) ** -0.5,
                _module.adamw_key(self.seed, step & 0xFFFFFFFF))

    def new_schedule(self) -> torch.Tensor:
        """Device memory for :meth:`advance`, read by steps that are captured into a graph.  Until it is advanced it is that of a step of
        length 0: moments are updated, parameters stay."""
        schedule = torch.zeros(4, dtype=torch.float32, device=self.device)
        schedule[:1] = schedule[2:3] = 1.0  # decay and the second moments' correction
        return schedule

    def advance(self, schedule: torch.Tensor, learning_rate: float) -> None:
        """Counts a step and writes what it needs into ``schedule``, on the current stream: before each replay of a graph that holds
        ``step(grads, schedule=schedule)``.  The host does not wait: steps may be queued ahead."""
        if schedule.shape != (4,) or schedule.dtype != torch.float32:
            raise ValueError("schedule must be what new_schedule() gave")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("advance() is called before a graph's replay, not under its capture")
        decay, step_size, correction, key = self._scalars(learning_rate, self.step_count + 1)
        # page-locked: of other memory the copy would wait for the stream; torch lends it anew once the copy is done
        words = torch.empty(4, dtype=torch.float32, pin_memory=True)
        words.copy_(torch.tensor([decay, step_size, correction, 0.0], dtype=torch.float32))
        words.view(torch.int32)[3] = key - (1 << 32) if key >> 31 else key
        schedule.copy_(words, non_blocking=True)
        self.step_count += 1

    def step(self, grads: Sequence[Optional[torch.Tensor]], learning_rate: Optional[float] = None, *,
             schedule: Optional[torch.Tensor] = None, grad_scale: float = 1.0) -> None:
        """One step with ``grads`` (one per parameter, all of one type, contiguous; None: the parameter and its moments stay as they
        are), each multiplied by ``grad_scale`` (from about 1e-17 to 1e20, since its square goes into the second moments; or 0).  Either
        ``learning_rate`` is given and the step is counted, or ``schedule``, which :meth:`advance` has written.  A step under stream
        capture needs a schedule: its replays would repeat one step's number."""
        if (learning_rate is None) == (schedule is None):
            raise ValueError("step() takes a learning_rate or a schedule")
        if schedule is not None:
            scalars = (0.0, 0.0, 0.0, 0)
        else:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a step under stream capture takes a schedule instead of a learning_rate")
            scalars = self._scalars(learning_rate, self.step_count + 1)
        self._tensors.step(grads, self.state_bits, self.adam_m, self.adam_v, self.m_exponent, self.v_exponent, self.beta_m, self.beta_v,
                           self.epsilon, grad_scale, *scalars, schedule)
        if schedule is None:
            self.step_count += 1

    def moments(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """Both moments as values: float32 ones as they are, 8-bit ones as bfloat16, which holds them exactly."""
        if self.state_bits == 32:
            return self.adam_m, self.adam_v
        return _module.adamw_moments(self.adam_m, self.m_exponent, self.adam_v, self.v_exponent)

    def _state_names(self) -> Tuple[str, ...]:
        return ("adam_m", "adam_v") + (("m_exponent", "v_exponent") if self.state_bits == 8 else ())

    def state(self) -> Dict[str, Any]:
        """The moments as they are held, the seed and the step count, for a checkpoint."""
        return dict(step_count=self.step_count, seed=self.seed, **{name: getattr(self, name).clone() for name in self._state_names()})

    def load_state(self, state: Dict[str, Any]) -> None:
        """Sets what :meth:`state` gave for an optimiser of the same tensors and state_bits.  One that does not fit changes nothing."""
        for name in self._state_names():
            mine, given = getattr(self, name), state.get(name)
            if not isinstance(given, torch.Tensor) or given.shape != mine.shape or given.dtype != mine.dtype:
                raise ValueError(f"'{name}' of the state does not fit this optimiser")
        numbers = {}
        for name in ("step_count", "seed"):
            try:
                numbers[name] = operator.index(state.get(name))
            except TypeError:
                raise ValueError(f"'{name}' of the state does not fit: {state.get(name)!r}") from None
        if numbers["step_count"] < 0:
            raise ValueError(f"'step_count' of the state does not fit: {numbers['step_count']}")
        for name in self._state_names():
            getattr(self, name).copy_(state[name])
        self.step_count, self.seed = numbers["step_count"], numbers["seed"] & 0xFFFFFFFF
