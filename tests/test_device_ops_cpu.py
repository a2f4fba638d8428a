"""Refusals of the operators on device tensors: arguments are checked before anything is launched, so no GPU is needed."""

import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import device_op_forms as forms  # noqa: E402
from distributed_kge_poplar_b200 import capi, device_ops  # noqa: E402

lib = capi.load_library()
SOME = 1 << 20  # stands for a device address: nothing reads it


def scores(**changes):
    s = capi.Scores(x=SOME, float_type=capi.F32, rows=4, cols=10, row_stride=10, scale=1.0)
    for name, value in changes.items():
        setattr(s, name, value)
    return s


def out(**changes):
    o = capi.LogProbsOut(SOME, SOME, SOME, SOME, 0, None, None)
    for name, value in changes.items():
        setattr(o, name, value)
    return o


def refused(status, text):
    assert status == capi.INVALID_ARGUMENT
    assert text in lib.kge_last_error(None).decode()


@pytest.mark.parametrize("changes,text", [
    (dict(float_type=capi.U32), "element type"), (dict(float_type=9), "element type"), (dict(row_stride=9), "apart"), (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(x=None), "null scores"),
    (dict(x=SOME + 2), "not aligned"), (dict(cols=2**31, row_stride=2**31), "columns"), (dict(mask=SOME, mask_stride=9), "mask rows")])
def test_scores_that_are_refused(changes, text):
    s = scores(**changes)
    refused(lib.kge_op_log_probs(C.byref(s), C.byref(out()), None, 0, None), text)
    refused(lib.kge_op_log_probs_grad(C.byref(s), SOME, SOME, None, 0, None, None, SOME, 10, None), text)


def test_outputs_that_are_refused():
    s = scores()
    refused(lib.kge_op_log_probs(None, C.byref(out()), None, 0, None), "null argument")
    refused(lib.kge_op_log_probs(C.byref(s), None, None, 0, None), "null argument")
    refused(lib.kge_op_log_probs(C.byref(s), C.byref(out(n_best=129, best_log_prob=SOME, best_index=SOME)), None, 0, None), "n_best")
    refused(lib.kge_op_log_probs(C.byref(s), C.byref(out(n_best=5)), None, 0, None), "null output")
    refused(lib.kge_op_log_probs(C.byref(s), C.byref(out(log_sum=None)), None, 0, None), "null output")
    refused(lib.kge_op_log_probs(C.byref(s), C.byref(out(row_state=SOME + 4)), None, 0, None), "row_state")
    grad = lib.kge_op_log_probs_grad
    refused(grad(None, SOME, None, None, 0, None, None, SOME, 10, None), "null argument")
    refused(grad(C.byref(s), None, None, None, 0, None, None, SOME, 10, None), "null argument")
    refused(grad(C.byref(s), SOME, None, None, 0, None, None, None, 10, None), "null argument")
    refused(grad(C.byref(s), SOME, None, None, 0, None, None, SOME + 2048, 9, None), "apart")
    refused(grad(C.byref(s), SOME, None, None, 0, None, None, SOME + 2, 10, None), "not aligned")
    refused(grad(C.byref(s), SOME + 8, None, None, 0, None, None, SOME, 10, None), "row_state")
    refused(grad(C.byref(s), SOME, None, None, 3, None, SOME, SOME, 10, None), "no indices")
    refused(grad(C.byref(s), SOME, None, None, 129, SOME, SOME, SOME, 10, None), "n_best")
    refused(grad(C.byref(s), SOME, None, None, 0, None, None, SOME, 12, None), "row stride")


def test_rows8_that_are_refused():
    values, exponents = C.c_size_t(), C.c_size_t()
    assert lib.kge_op_rows8_bytes(129, 513, C.byref(values), C.byref(exponents)) == capi.OK
    assert (values.value, exponents.value) == (129 * 640, 2 * 2 * 512)
    assert lib.kge_op_rows8_bytes(3, 17, C.byref(values), C.byref(exponents)) == capi.OK and values.value == 3 * 32
    refused(lib.kge_op_rows8_bytes(1, 1, None, C.byref(exponents)), "null argument")
    quantise = lib.kge_op_quantise_rows
    refused(quantise(SOME, capi.U32, 4, 10, 10, 0, SOME, SOME, None), "element type")
    refused(quantise(SOME, capi.F32, 4, 10, 9, 0, SOME, SOME, None), "apart")
    refused(quantise(None, capi.F32, 4, 10, 10, 0, SOME, SOME, None), "null argument")
    refused(quantise(SOME, capi.F32, 4, 10, 10, 0, SOME + 8, SOME, None), "aligned")
    refused(quantise(SOME + 1, capi.F16, 4, 10, 10, 0, SOME, SOME, None), "aligned")
    assert quantise(None, capi.F32, 0, 10, 10, 0, None, None, None) == capi.OK


def test_products_that_are_refused():
    product = lib.kge_op_product8
    refused(product(SOME, SOME, 4, SOME, SOME, 8, 10, SOME, capi.U32, 8, None, 0, None), "element type")
    refused(product(SOME, SOME, 4, SOME, SOME, 8, 10, SOME, capi.F32, 7, None, 0, None), "apart")
    refused(product(SOME, SOME, 4, SOME, SOME, 8, 10, None, capi.F32, 8, None, 0, None), "null output")
    refused(product(SOME, None, 4, SOME, SOME, 8, 10, SOME, capi.F32, 8, None, 0, None), "null operand")
    refused(product(SOME + 8, SOME, 4, SOME, SOME, 8, 10, SOME, capi.F32, 8, None, 0, None), "aligned")
    refused(product(SOME, SOME, 2**31, SOME, SOME, 8, 10, SOME, capi.F32, 8, None, 0, None), "too large")
    wanted = lib.kge_op_product8_workspace(4, 8, 100_000)
    assert wanted > 0
    refused(product(SOME, SOME, 4, SOME, SOME, 8, 100_000, SOME, capi.F32, 8, SOME, wanted - 1, None), "workspace")
    refused(product(SOME, SOME, 4, SOME, SOME, 8, 100_000, SOME, capi.F32, 8, None, 0, None), "workspace")
    refused(product(SOME, SOME, 4, SOME, SOME, 8, 100_000, SOME, capi.F32, 8, SOME + 16, wanted, None), "256 bytes")
    assert product(None, None, 0, None, None, 8, 10, None, capi.F32, 8, None, 0, None) == capi.OK


def adamw(tensor=(), **changes):
    args = capi.AdamWArgs(param_type=capi.F32, grad_type=capi.F32, state_bits=32, adam_m=SOME, adam_v=SOME, m_exponent=SOME, v_exponent=SOME,
                          beta_m=0.9, beta_v=0.99, epsilon=1e-8, grad_scale=1.0, decay=1.0, step_size=0.1, inv_sqrt_correction=1.0)
    for name, value in changes.items():
        setattr(args, name, value)
    t = capi.AdamWTensor(SOME, SOME, 100, 128)
    for name, value in dict(tensor).items():
        setattr(t, name, value)
    return lib.kge_op_adamw(C.byref(args), (capi.AdamWTensor * 1)(t), 1, None)


@pytest.mark.parametrize("tensor,changes,text", [
    ({}, dict(param_type=capi.F16), "parameters must be"), ({}, dict(grad_type=capi.U32), "element type"), ({}, dict(state_bits=16), "state_bits"),
    ({}, dict(adam_m=None), "null moments"), ({}, dict(state_bits=8, v_exponent=None), "null moments"), ({}, dict(adam_v=SOME + 4), "aligned"),
    (dict(param=None), {}, "no parameter or no gradient"), (dict(grad=None), {}, "no parameter or no gradient"), (dict(first=64), {}, "multiple of 128"),
    (dict(param=SOME + 2), {}, "not aligned"), (dict(size=2**40), {}, "too many"), ({}, dict(schedule=SOME + 1), "schedule")])
def test_adamw_steps_that_are_refused(tensor, changes, text):
    refused(adamw(tensor, **changes), text)


def test_adamw_steps_of_nothing():
    assert adamw(dict(size=0, param=None, grad=None)) == capi.OK
    assert lib.kge_op_adamw(None, None, 0, None) == capi.INVALID_ARGUMENT
    refused(lib.kge_op_adamw_moments(SOME, SOME, SOME, SOME, 100, SOME, SOME, None), "multiple of 128")
    refused(lib.kge_op_adamw_moments(SOME, None, SOME, SOME, 128, SOME, SOME, None), "null argument")
    assert lib.kge_op_adamw_moments(None, None, None, None, 0, None, None, None) == capi.OK


def test_adamw_keys_are_the_definition_s():
    for seed, step in ((0, 0), (1, 1), (12345, 678), (2**32 - 1, 2**32 - 1)):
        assert lib.kge_op_adamw_key(seed, step) == forms.mix((seed * 0x9E3779B9 + step * 0xBB67AE85) & 0xFFFFFFFF)


def test_tensors_that_are_no_device_tensors():
    x = torch.zeros(2, 3)
    for call in (lambda: device_ops.log_probs(x), lambda: device_ops.quantise_rows(x), lambda: device_ops.product8(x, x), lambda: device_ops.AdamW([x])):
        with pytest.raises(ValueError, match="on a GPU"):
            call()
    with pytest.raises(ValueError, match="must be a tensor"):
        device_ops.log_probs(np.zeros((2, 3), np.float32))
    with pytest.raises(ValueError, match="not torch.float64"):
        device_ops.quantise_rows(x.double())
    with pytest.raises(ValueError, match="n_best"):
        device_ops.log_probs(x, n_best=129)
    with pytest.raises(ValueError, match="at least one"):
        device_ops.AdamW([])
    with pytest.raises(ValueError, match="state_bits"):
        device_ops.AdamW([x], state_bits=4)


def test_the_forms_agree_with_torch():
    """The tests' own definitions against torch's where it has one."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(5, 40, generator=g)
    form = forms.log_probs(x, torch.arange(5, dtype=torch.int32), scale=0.5, n_best=3)
    want = torch.log_softmax(x.double() * 0.5, 1)
    assert torch.allclose(form["log_p"], want, rtol=0, atol=1e-12)
    assert torch.allclose(form["entropy"], torch.distributions.Categorical(logits=x.double() * 0.5).entropy(), atol=1e-12)
    y = torch.randn(1000, generator=g) * 100
    assert torch.equal(forms.e4m3(y.double()).float(), y.to(torch.float8_e4m3fn).float())
    v = x.double().requires_grad_()
    p = torch.log_softmax(v * 0.5, 1)
    loss = (p[torch.arange(5), torch.arange(5)]).sum() - 0.3 * (p.exp() * p).sum() + 0.1 * p.topk(3).values.sum()
    loss.backward()
    got = forms.log_probs_grad(x, form, torch.arange(5), 0.5, torch.ones(5), torch.full((5,), 0.3), torch.full((5, 3), 0.1))
    assert torch.allclose(got, v.grad, atol=1e-8)  # the weights are fp32
