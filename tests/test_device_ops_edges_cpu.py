"""What the operators on device tensors refuse or do on the host, beside test_device_ops_cpu: no GPU is needed."""

import pytest

torch = pytest.importorskip("torch")

from distributed_kge_poplar_b200 import capi, device_ops  # noqa: E402
from test_device_ops_cpu import SOME, adamw, lib, refused  # noqa: E402


@pytest.mark.parametrize("epsilon", [0.0, -1e-8, 1e-46, 1e-39, float("nan"), float("inf"), 1e39])
def test_an_epsilon_that_is_no_normal_number_in_fp32(epsilon):
    refused(adamw(epsilon=epsilon), "epsilon")
    with pytest.raises(ValueError, match="epsilon"):
        device_ops.AdamW([torch.zeros(3)], epsilon=epsilon)


@pytest.mark.parametrize("scale", [1e-20, -1e-20, 1e-200, 1e25, -1e25, 1e160])
def test_a_gradient_scale_whose_square_fp32_does_not_hold(scale):
    refused(adamw(grad_scale=scale), "grad_scale")


def test_a_product_that_gave_up_is_an_error(monkeypatch):
    class Library:  # answers as the library does after a wait on the device has run out
        status = capi.DEVICE_STATUS

        def kge_op_product8_status(self):
            return self.status

        def kge_last_error(self, engine):
            return b"kge_op_product8: a wait on the device gave up"

    monkeypatch.setattr(capi, "load_library", Library)
    with pytest.raises(RuntimeError, match="a wait on the device gave up"):
        device_ops.check_product8()
    monkeypatch.setattr(Library, "status", capi.OK)
    device_ops.check_product8()


@pytest.mark.parametrize("rows,cols", [(0, 5), (0, 0), (3, 0), (2, 130)])
def test_dequantised_rows_have_their_shape(rows, cols):
    class Rows:  # what the values and their exponents lie in
        values = torch.zeros(rows, -(-cols // 128) * 128 if cols > 128 else -(-cols // 16) * 16, dtype=torch.uint8)
        exponents = torch.full((-(-rows // 128) * -(-cols // 512) * 512,), 127, dtype=torch.uint8)

    Rows.rows, Rows.cols = rows, cols
    got = device_ops.Rows8.dequantise(Rows)
    assert got.shape == (rows, cols) and got.dtype == torch.float32 and torch.all(got == 0)


def test_moments_that_do_not_fit_one_another():
    def bytes_(n):
        return torch.zeros(n, dtype=torch.uint8)

    for moments, text in [((bytes_(256), bytes_(1), bytes_(256), bytes_(2)), "m_exponent has shape"), ((bytes_(256), bytes_(2), bytes_(256), bytes_(1)), "v_exponent has shape"),
                          ((bytes_(256), bytes_(2).float(), bytes_(256), bytes_(2)), "m_exponent must be torch.uint8"),
                          ((bytes_(256), bytes_(4)[::2], bytes_(256), bytes_(2)), "m_exponent must be contiguous"), ((bytes_(256), bytes_(2), bytes_(256), bytes_(2)), "on a GPU")]:
        with pytest.raises(ValueError, match=text):
            device_ops._module.adamw_moments(*moments)


def optimiser_of(bits, total=256):
    """An optimiser as it is between its calls, without the GPU that its construction asks for."""
    optimiser = object.__new__(device_ops.AdamW)
    optimiser.state_bits, optimiser.step_count, optimiser.seed, optimiser.device = bits, 3, 7, torch.device("cpu")
    kind = torch.float32 if bits == 32 else torch.uint8
    optimiser.adam_m, optimiser.adam_v = torch.zeros(total, dtype=kind), torch.zeros(total, dtype=kind)
    optimiser.m_exponent, optimiser.v_exponent = torch.zeros(total // 128, dtype=torch.uint8), torch.zeros(total // 128, dtype=torch.uint8)
    return optimiser


@pytest.mark.parametrize("bits", [8, 32])
def test_a_state_that_does_not_fit_changes_nothing(bits):
    optimiser, other = optimiser_of(bits), optimiser_of(bits)
    for t in (other.adam_m, other.adam_v):
        t.fill_(5)
    whole = other.state()
    for change in (dict(step_count=None), dict(step_count=-1), dict(step_count=1.5), dict(seed=None), dict(seed="x"), dict(adam_v=whole["adam_v"][:128]), dict(adam_v=[5] * 256)):
        for state in (dict(whole, **change), {k: v for k, v in whole.items() if k not in change}):
            with pytest.raises(ValueError, match="does not fit"):
                optimiser.load_state(state)
            assert torch.all(optimiser.adam_m == 0) and torch.all(optimiser.adam_v == 0) and (optimiser.step_count, optimiser.seed) == (3, 7)
    optimiser.load_state(dict(whole, step_count=torch.tensor(9), seed=-1))
    assert torch.all(optimiser.adam_m == 5) and (optimiser.step_count, optimiser.seed) == (9, 0xFFFFFFFF)


def test_workspaces_of_sizes_that_are_refused():
    for k in (2**31, 2**38, 2**57, 2**64 - 1):
        assert lib.kge_op_product8_workspace(4, 8, k) == 0
        refused(lib.kge_op_product8(SOME, SOME, 4, SOME, SOME, 8, k, SOME, capi.F32, 8, SOME, 2**40, None), "too large")
    assert lib.kge_op_product8_workspace(2**31 - 1, 2**31 - 1, 2**31) == 0
