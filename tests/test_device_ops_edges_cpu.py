"""What the operators on device tensors refuse or do on the host, beside test_device_ops_cpu: no GPU is needed."""

import pytest

torch = pytest.importorskip("torch")

from distributed_kge_poplar_b200 import device_ops  # noqa: E402
from test_device_ops_cpu import adamw, refused  # noqa: E402


@pytest.mark.parametrize("epsilon", [0.0, -1e-8, 1e-46, 1e-39, float("nan"), float("inf"), 1e39])
def test_an_epsilon_that_is_no_normal_number_in_fp32(epsilon):
    refused(adamw(epsilon=epsilon), "epsilon")
    with pytest.raises(ValueError, match="epsilon"):
        device_ops.AdamW([torch.zeros(3)], epsilon=epsilon)


@pytest.mark.parametrize("scale", [1e-20, -1e-20, 1e-200, 1e25, -1e25, 1e160])
def test_a_gradient_scale_whose_square_fp32_does_not_hold(scale):
    refused(adamw(grad_scale=scale), "grad_scale")
