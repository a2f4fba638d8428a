"""The operators on device tensors where their definitions are easily missed: values that are not finite or far from the others, lists
that are thinned out, larger blocks, tiles and parts."""

import pytest

torch = pytest.importorskip("torch")

import device_op_forms as forms  # noqa: E402
from test_device_ops_gpu import check_log_probs, gen, ops  # noqa: E402, F401

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
