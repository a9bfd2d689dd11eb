"""LinearAttention's errors in the 2-norm, relative to the outputs', over random operands.
Where the bounds of test_gpu_linear_attention.py, element by element, have to allow for
every rounding in the same direction, these count them as what they are for independent
normal operands: independent.

A rounding to nearest of a value m 2^e, 1 <= m < 2, with half step u (bf16 2^-8, f16 2^-11)
is off by u 2^e / sqrt(3) in the mean square, u / sqrt(3) / m relative. Over values of many
scales (heads, positions) log2 m is uniform, the mean of 1 / m^2 is 3 / (8 ln 2), and the
relative error

    RMS = sqrt(3 / (8 ln 2) / 3) u = 0.4247 u.

An output sum_j x_j of independent terms of mean 0 has the mean square of their sum of
squares, so terms that each have an independent relative error RMS give the output that
error; with its own rounding sqrt(2) RMS. The scores and the state's copy of the bf16
chunks are such operands, one of the two in each term. 15 % more is for the
sampling of scales and of S, which outputs share.

f32 sums: a tensor core's accumulator may be truncated at each step of 16 terms, by up to 2^-23
of it, in one direction, 2^-24 in the mean; the accumulator grows as the root of its steps, so
n steps are off by at most 2 / 3 n 2^-24. Scores and outputs at f32 accuracy have 48 steps
each at most (6 products of parts, 128 terms): 2 * 32 * 2^-24 = 3.8e-6, with what
parts leave out (3 * 2^-24) and the sums over chunks below 4.5e-6. States take
24 steps a chunk (8 of 16 terms, 3 parts; in parts of 64 positions the same) and one f32 product
and sum a chunk, 21 chunks here: (16 + 21) * 2^-24 = 2.2e-6."""

from __future__ import annotations

import math

import pytest
import torch

from bunsen_b200.linear_attention import LinearAttention
from tests.test_gpu_linear_attention import TYPES, U, make, ranges, want_core

pytestmark = pytest.mark.gpu
RMS = math.sqrt(1 / (8 * math.log(2)))
F32, STATE = 4.5e-6, 2.2e-6
DECAYS = [-0.003, -0.6, 0.0, -0.02, -0.1, -0.3, -3.0, -0.0005]


def off(got, want):
    return float((got.double().reshape(want.shape) - want).norm() / want.norm())


def bound(dtype, u_op):
    u = 0.0 if dtype == torch.float32 else U[dtype]
    return 1.15 * RMS * math.hypot(u, u_op) + F32


def check(x, algo, u_op):
    rule = LinearAttention(algo=algo)
    args = (x["q"], x["k"], x["v"], x["g"])
    hq, hv, scale = x["q"].shape[-2], x["v"].shape[-2], x["q"].shape[-1] ** -0.5
    out, s1 = rule.chunked(*args, x["state"], cu_seqlens=x["cu"])
    dq, dk, dv, d0 = rule.backward(*args, x["do"], x["state"], x["ds"], cu_seqlens=x["cu"])
    tol = bound(out.dtype, u_op)
    for got, state, roles, sigma, tau, s0, rev, turn in (
            (out, s1, ("q", "k", "v"), 1.0, scale, x["state"], False, False),
            (dq, None, ("do", "v", "k"), 1.0, scale, x["state"], False, True),
            (dk, None, ("v", "do", "q"), scale, 1.0, x["ds"], True, True),
            (dv, d0, ("k", "q", "do"), scale, 1.0, x["ds"], True, False)):
        want, _, ws, _ = want_core(x, [x[r] for r in roles], sigma, tau, s0, rev, turn)
        if turn and hv > hq:
            want = want.view(len(want), hq, hv // hq, -1).sum(2)
        assert off(got, want) <= tol, (roles, off(got, want), tol)
        if state is not None:
            assert off(state, ws) <= STATE, (roles, off(state, ws))
        if want.shape[1] == hv:  # no head hides behind another
            rows = torch.cat([torch.arange(i, j, device=want.device) for i, j in ranges(x)])
            got = got.double().reshape(want.shape)[rows]
            each = (got - want[rows]).pow(2).sum((0, 2)).sqrt() / want[rows].pow(2).sum((0, 2)).sqrt()
            # (A head's outputs are of fewer scales: 1 / m^2 is at most 1.)
            assert float(each.max()) <= tol / RMS / math.sqrt(3), (roles, each.tolist())


@pytest.mark.parametrize("algo", ["auto", "tensor", "tensor_split"])
@pytest.mark.parametrize("shape", [(128, 128), (64, 64), (40, 72)])
@pytest.mark.parametrize("hq", [8, 4])
def test_bf16_chunks(hq, shape, algo):
    x = make([700, 5, 0, 1281, 1, 640, 129], hq, 8, *shape, torch.bfloat16, seed=hq, g=DECAYS)
    check(x, algo, U[torch.bfloat16])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(128, 128), (64, 64), (33, 65)])
@pytest.mark.parametrize("hq", [8, 4])
def test_chunks_at_f32_accuracy(hq, shape, dtype):
    x = make([700, 5, 0, 1281, 1, 640, 129], hq, 8, *shape, dtype, seed=hq, g=DECAYS)
    check(x, "cuda_core", 0.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[1] * 100 + [700] + [1] * 155, [64], [16], [4] * 50])
def test_small_and_skewed_calls(lens, dtype):
    x = make(lens, 8, 8, 128, 128, dtype, seed=len(lens), g=DECAYS)
    check(x, "auto", 0.0)
