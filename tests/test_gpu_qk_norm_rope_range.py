"""qk_norm_rope and its gradient over the range of the head vectors' norms. The
bounds are test_gpu_qk_norm_rope.py's, relative to absolute terms, so they hold at any
magnitude whose squares f32 holds."""

from __future__ import annotations

import pytest
import torch

import tests.test_gpu_qk_norm_rope as base

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens", [3, 700])
@pytest.mark.parametrize("d", [128, 33])  # both kernels
@pytest.mark.parametrize("scale,eps", [(1e14, 1e-6), (1e17, 1e-6), (1e-16, 0.0), (1e-16, 1e-30)])
def test_magnitudes(scale, eps, d, tokens, interleaved, dtype, monkeypatch):
    """The gradient's two terms are of one size, r = 1 / rms, whatever r^3 is."""
    monkeypatch.setattr(base, "EPS", eps)
    x, g = base.make(tokens, 16, 4, d, 2 * (d // 4), dtype, seed=d)
    for key in ("q", "k"):
        x[key] = (x[key].float() * scale).to(dtype)
    base.check(x, g, interleaved=interleaved)
