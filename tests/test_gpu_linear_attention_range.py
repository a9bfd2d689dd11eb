"""LinearAttention over the range of its operands: large and small ones.
The bounds are those of test_gpu_linear_attention.py, which are relative to the
operator on absolute values and so hold at any magnitude."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_linear_attention import check_backward, check_forward, make

pytestmark = pytest.mark.gpu


def scaled(x, **factors):
    return {**x, **{key: (x[key].float() * f).to(x[key].dtype) for key, f in factors.items()}}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(128, 128), (64, 72)])
@pytest.mark.parametrize("qk,v", [(1e12, 1.0), (1.0, 1e30), (3e16, 1.0), (1e-14, 1.0),
                                  (1e-3, 1e-18)])
def test_magnitudes(qk, v, shape, dtype):
    """Outputs that the type holds, from scores and products that f32 holds: no
    factor of a chunk's sums may leave it in between. Scores are of the order of
    qk^2 (of v in the gradients), at most 1e35 with their sums."""
    x = make([300, 1, 40, 129, 1000], 2, 4, *shape, dtype, seed=3, g=[-0.3, -0.05, -0.01, -0.39])
    x = scaled(x, q=qk, k=qk, v=v)
    check_forward(x)
    check_backward(x)
