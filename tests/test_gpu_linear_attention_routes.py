"""Which kernel a LinearAttention call takes, by what each promises: calls of few positions,
small prompts and packs of mostly single positions are at f32 accuracy whatever their type
(the bound of test_gpu_linear_attention.py without a rounding of operands), and a long
sequence among short ones is not walked a position at a time."""

from __future__ import annotations

import pytest
import torch

import tests.test_gpu_linear_attention as base
from bunsen_b200 import _lib
from bunsen_b200.linear_attention import LinearAttention
from tests.test_gpu_linear_attention import TYPES, check_backward, check_forward, make

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture
def strict(monkeypatch):
    monkeypatch.setattr(base, "op_rounding", lambda x, algo: 0.0)


SKEWED = {
    "a prompt among rows": [1] * 100 + [700] + [1] * 155,
    "a long one among empty ones": [0] * 300 + [1030] + [0] * 20,
    "around the limit": [4, 5, 3, 1, 0, 6, 2, 64, 1, 1, 1, 1] + [0] * 14 + [1, 0],
    "two prompts": [300] + [0, 1, 2] * 90 + [129] + [1] * 80,
    "rows alone": [1] * 77,
    "fours": [4] * 50,
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(128, 128), (33, 65), (64, 200)])
@pytest.mark.parametrize("name", list(SKEWED))
def test_skewed_packs(name, shape, dtype, strict):
    lens = SKEWED[name]
    assert 64 < sum(lens) <= 4 * len(lens)
    x = make(lens, 2, 4, *shape, dtype, seed=len(lens))
    out, s1 = check_forward(x)
    check_backward(x)
    state = x["state"].clone()  # in place
    again, _ = LinearAttention().chunked(x["q"], x["k"], x["v"], x["g"], state, cu_seqlens=x["cu"],
                                         state_out=state)
    assert torch.equal(out, again) and torch.equal(s1, state)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_more_sequences_than_the_plans_threads(dtype):
    """1500 sequences, most of a few positions, some long enough for segments: forward and
    backward, whatever kernel the mean length gives them."""
    lens = [(7 * i) % 5 for i in range(1500)]
    lens[3], lens[1100], lens[1400] = 150, 2000, 129
    for extra in (0, 20):  # more and fewer than four a sequence
        y = [n + extra if i % 7 == 0 else n for i, n in enumerate(lens)]
        assert (sum(y) <= 4 * len(y)) == (extra == 0)
        x = make(y, 1, 2, 64, 64, dtype, seed=extra)
        check_forward(x)
        check_backward(x)


@pytest.mark.parametrize("dtype", TYPES)
def test_skewed_pack_padded_captured_and_on_a_stream(dtype):
    """NaN behind the last sequence; the same bits captured, replayed and on another stream."""
    lens = SKEWED["two prompts"]
    x = make(lens, 2, 4, 64, 64, dtype, seed=1, pad=50)
    n = sum(lens)
    for key in ("q", "k", "v", "do"):
        x[key][n:] = float("nan")
    out = torch.full_like(x["v"], 7.0)

    def call():
        rule = LinearAttention()
        return [*rule.chunked(x["q"], x["k"], x["v"], x["g"], x["state"], cu_seqlens=x["cu"],
                              out=out),
                *rule.backward(x["q"], x["k"], x["v"], x["g"], x["do"], x["state"], x["ds"],
                               cu_seqlens=x["cu"])]

    def live(ts):
        return [t[:n].clone() if t.shape[0] == n + 50 else t.clone() for t in ts]

    ref = live(call())
    assert bool((out[n:] == 7.0).all()) and all(bool(torch.isfinite(t).all()) for t in ref)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = live(call())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = call()
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ref, live(outs)))
    assert _lib.load().gdr_device_error() == _lib.GDR_OK


def microseconds(call):
    call(), call()
    times = []
    for _ in range(7):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        torch.cuda.synchronize()
        a.record()
        call()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) * 1e3)
    return min(times)


def test_a_long_sequence_among_rows_is_not_walked():
    """A prompt of 3000 positions between 1000 single ones takes no longer than twice the
    prompt and the rows in calls of their own (a walk of it alone takes three times that)."""
    parts = [[1] * 500 + [3000] + [1] * 500, [3000], [1] * 1000]
    t = []
    for lens in parts:
        x = make(lens, 16, 32, 128, 128, torch.bfloat16, seed=0)
        out, s1 = torch.empty_like(x["v"]), torch.empty_like(x["state"])
        t.append(microseconds(lambda: LinearAttention().chunked(  # noqa: B023
            x["q"], x["k"], x["v"], x["g"], x["state"], cu_seqlens=x["cu"], out=out, state_out=s1)))
    assert t[0] <= 2 * (t[1] + t[2]), t


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,packed", [
    ([1], True), ([16], True), ([16], False), ([4, 4, 4, 4, 4], False), ([3, 1, 4, 4, 4, 4, 0], True),
    ([64], True), ([64], False), ([20, 0, 44], True), ([32, 32], False), ([17], True)])
def test_small_calls_at_f32_accuracy(lens, packed, dtype, strict):
    """Few positions, and 64 or fewer where every sequence and head has an SM."""
    x = make(lens, 2, 4, 128, 128, dtype, seed=sum(lens), packed=packed)
    check_forward(x)
    check_backward(x)


@pytest.mark.parametrize("shape", [(33, 65), (1, 1), (5, 128), (128, 5), (60, 64), (160, 96),
                                   (256, 256)])
def test_other_widths_at_f32_accuracy(shape, strict):
    """bf16 widths that the chunks with bf16 scores do not take."""
    x = make([200, 1, 170], 1, 2, *shape, torch.bfloat16, seed=sum(shape))
    check_forward(x)
    check_backward(x)


@pytest.mark.parametrize("dtype", TYPES)
def test_cuda_core_at_f32_accuracy(dtype, strict):
    x = make([300, 0, 513, 64], 2, 4, 128, 128, dtype, seed=14)
    check_forward(x, "cuda_core")
    check_backward(x, "cuda_core")


# Chunks of 16-bit types take scores and the state's copy in two bf16 parts, each off by at most
# 2^-8 x 2^-8 of itself, on disjoint parts of an output. Operands of f16 are two parts
# themselves: products leave out the second part of one with the second of the other, 2^-16
# again, once in the scores and once in the outputs.
PARTS = {torch.float32: 0.0, torch.bfloat16: 2.0**-16, torch.float16: 3 * 2.0**-16}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 3), (3, 1), (8, 8)])
@pytest.mark.parametrize("lens", [[5, 0, 1, 2, 4] * 50, [5] * 100, [17] * 10 + [64]])
def test_narrow_heads(lens, shape, dtype, monkeypatch):
    """Sums of few terms, where nothing averages what a part leaves out."""
    monkeypatch.setattr(base, "op_rounding", lambda x, algo: PARTS[x["q"].dtype])
    g = [-0.01, -0.39, 0.0, -0.41, -5.0, -0.0001, -1.0, -50.0, 0.0, -0.01, -0.0001, float("-inf")]
    x = make(lens, 3, 12, *shape, dtype, seed=len(lens), g=g)
    check_forward(x, "cuda_core")
    check_backward(x, "cuda_core")
