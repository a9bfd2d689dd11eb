"""LinearAttention against its definition in 64 bits.

Tolerances are derived, element by element. With A the same operator on the
absolute values of its operands (``core(|a|, |b|, |c|, |S0|)``), every
operand rounding of relative size u moves an output by at most u A, and f32
sums over n terms by at most n 2^-24 A (2^-23 where an accumulator may
truncate). So

    |out - exact| <= u_T |exact| + (u_op + (n + d + 64) 2^-23) A

u_T the half step of the output's type (bf16 2^-8, f16 2^-11, f32 2^-24), n
the longest sequence, u_op 2^-8 where the tensor cores take the chunk's scores
and the state as bf16 operands (each output sums disjoint parts of either, so
one u covers both), 0 in f32. States take no such rounding: their scaled
operand goes in as three bf16 parts (24 bits). Small values have absolute steps:
f16 has none below 2^-24, so its rounding moves a result by up to 2^-25; f32
has no normal number below 2^-126, so a decay under it is off by up to that,
times operands' sums that stay below 2^20 here: 2^-106."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from bunsen_b200 import _lib, layer
from bunsen_b200.linear_attention import LinearAttention

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
STEP = {torch.float16: 2.0**-25}


def core(a, b, c, log_decay, sigma, tau, s0, reverse):
    """One sequence in f64: a, b [T, H, n], c [T, H, m], s0 [H, n, m].
    out_t = tau a_t . S_t, S_t = w S_{t-1} + sigma b_t c_t^T, or backward in
    time with S scaled after each position."""
    a, b, c = (x.double().transpose(0, 1) for x in (a, b, c))  # [H, T, .]
    t = a.shape[1]
    i = torch.arange(t, device=a.device, dtype=torch.float64)
    g = log_decay.double()[:, None, None]
    dist = (i[None, :] - i[:, None]) if reverse else (i[:, None] - i[None, :])
    power = lambda n: torch.where(n == 0, 1.0, torch.exp(g * n.clamp_min(1)))  # noqa: E731  w^0 = 1
    m = torch.where(dist >= 0, power(dist.clamp_min(0)), 0.0)
    ahead = power((t - 1 - i if reverse else i + 1)[:, None])
    left = power((i + 1 if reverse else t - 1 - i)[:, None])
    out = tau * (sigma * ((a @ b.transpose(1, 2)) * m) @ c + ahead * (a @ s0.double()))
    s1 = power(torch.tensor([[float(t)]], device=a.device, dtype=torch.float64)) * s0.double() + \
        sigma * (b * left).transpose(1, 2) @ c
    return out.transpose(0, 1), s1


def ranges(x):
    """[start, end) of each sequence over the flat token axis."""
    if x["cu"] is None:
        t = x["q"].shape[1]
        return [(s * t, (s + 1) * t) for s in range(x["q"].shape[0])]
    cu = x["cu"].tolist()
    return list(zip(cu[:-1], cu[1:]))


def flat(x):
    return x.flatten(0, -3)


def share(x, hv):
    return x.repeat_interleave(hv // x.shape[-2], dim=-2)


def want_core(x, roles, sigma, tau, state, reverse, turn):
    """The core over every sequence, and its bound A."""
    hv = x["g"].numel()
    a, b, c = (share(flat(r), hv) for r in roles)
    outs = [torch.zeros(a.shape[0], hv, c.shape[-1], dtype=torch.float64, device=DEV)
            for _ in range(2)]
    states = [[], []]
    for s, (i, j) in enumerate(ranges(x)):
        s0 = state[s] if state is not None else torch.zeros(hv, x["q"].shape[-1],
                                                            x["v"].shape[-1], device=DEV)
        s0 = s0.transpose(-1, -2) if turn else s0
        for k, f in enumerate((lambda y: y, torch.abs)):
            o, s1 = core(f(a[i:j]), f(b[i:j]), f(c[i:j]), x["g"], abs(sigma) if k else sigma,
                         abs(tau) if k else tau, f(s0), reverse)
            outs[k][i:j] = o
            states[k].append(s1.transpose(-1, -2) if turn else s1)
    return outs[0], outs[1], torch.stack(states[0]), torch.stack(states[1])


def longest(x):
    return max([j - i for i, j in ranges(x)] + [0])


def close(got, want, bound, x, op, dtype, what):
    n = longest(x) + max(x["q"].shape[-1], x["v"].shape[-1]) + 64
    tol = U[dtype] * want.abs() + (op + n * 2.0**-23) * bound + STEP.get(dtype, 2.0**-106)
    got = got.double().reshape(want.shape)
    live = torch.zeros(want.shape[0], dtype=torch.bool, device=DEV)
    if what == "state":
        live[:] = True
    else:
        for i, j in ranges(x):
            live[i:j] = True
    err = (got - want).abs()[live]
    bad = ~(err <= tol[live])
    assert not bad.any(), (what, float(err[bad].max()), float((err / tol[live])[bad].max()),
                           int(bad.sum()))


def make(lens, hq, hv, dk, dv, dtype, seed=0, packed=True, state=True, pad=0, g=None):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    f = dict(device=DEV, generator=gen)
    t = sum(lens) + pad
    lead = (t,) if packed else (len(lens), lens[0] if lens else 0)
    r = lambda *s: torch.randn(*s, **f).to(dtype)  # noqa: E731
    x = {"q": r(*lead, hq, dk), "k": r(*lead, hq, dk), "v": r(*lead, hv, dv),
         "do": r(*lead, hv, dv), "g": -torch.exp2(-8 * torch.rand(hv, **f)) if g is None else
         torch.tensor(g, device=DEV, dtype=torch.float32),
         "state": torch.randn(len(lens), hv, dk, dv, **f) if state else None,
         "ds": torch.randn(len(lens), hv, dk, dv, **f) if state else None,
         "cu": torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32,
                            device=DEV) if packed else None}
    return x


def op_rounding(x, algo):
    """u_op of the kernels a call takes."""
    tensor = x["q"].dtype == torch.bfloat16 and algo != "cuda_core" and \
        max(x["q"].shape[-1], x["v"].shape[-1]) <= 128
    return 2.0**-8 if tensor else 0.0


def check_forward(x, algo="auto", form="chunked", split=0):
    rule = LinearAttention(algo=algo, split_chunks=split)
    out, s1 = getattr(rule, form)(x["q"], x["k"], x["v"], x["g"], x["state"], cu_seqlens=x["cu"])
    scale = x["q"].shape[-1] ** -0.5
    want, bound, ws, bs = want_core(x, (x["q"], x["k"], x["v"]), 1.0, scale, x["state"], False,
                                    False)
    assert out.dtype == x["q"].dtype and out.shape == x["v"].shape and s1.dtype == torch.float32
    op = op_rounding(x, algo) if form == "chunked" else 0.0
    close(out, want, bound, x, op, out.dtype, "out")
    close(s1, ws, bs, x, 0.0, torch.float32, "state")
    assert _lib.load().gdr_device_error() == _lib.GDR_OK
    return out, s1


def check_backward(x, algo="auto", split=0):
    rule = LinearAttention(algo=algo, split_chunks=split)
    dq, dk, dv, d0 = rule.backward(x["q"], x["k"], x["v"], x["g"], x["do"], x["state"], x["ds"],
                                   cu_seqlens=x["cu"])
    hq, hv, scale = x["q"].shape[-2], x["v"].shape[-2], x["q"].shape[-1] ** -0.5
    op = op_rounding(x, algo)
    heads = lambda y: y.view(len(y), hq, hv // hq, y.shape[-1]).sum(2)  # noqa: E731
    for got, roles, sigma, tau, state, rev, turn, name in (
            (dq, (x["do"], x["v"], x["k"]), 1.0, scale, x["state"], False, True, "dq"),
            (dk, (x["v"], x["do"], x["q"]), scale, 1.0, x["ds"], True, True, "dk"),
            (dv, (x["k"], x["q"], x["do"]), scale, 1.0, x["ds"], True, False, "dv")):
        want, bound, ws, bs = want_core(x, roles, sigma, tau, state, rev, turn)
        if name != "dv":
            want, bound = heads(want), heads(bound)
        close(got, want, bound, x, op, got.dtype, name)
        if name == "dv" and d0 is not None:
            close(d0, ws, bs, x, 0.0, torch.float32, "state")
    assert (d0 is None) == (x["state"] is None)
    assert _lib.load().gdr_device_error() == _lib.GDR_OK
    return dq, dk, dv, d0


TYPES = [torch.bfloat16, torch.float16, torch.float32]
LENS = [[1], [0], [3, 0, 1, 130], [127, 128, 129], [64, 257, 1, 63, 65], [513]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("form", ["chunked", "recurrent"])
def test_packed(form, lens, dtype):
    check_forward(make(lens, 2, 4, 128, 128, dtype, seed=len(lens)), form=form)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(8, 8), (64, 64), (40, 72), (33, 65), (1, 1), (128, 64),
                                   (64, 128), (5, 128), (160, 96), (256, 256), (96, 200)])
@pytest.mark.parametrize("form", ["chunked", "recurrent"])
def test_head_sizes(form, shape, dtype):
    check_forward(make([70, 1, 150], 1, 3, *shape, dtype, seed=sum(shape)), form=form)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,t", [(1, 1), (3, 200), (4, 128), (2, 0)])
@pytest.mark.parametrize("state", [True, False])
def test_dense(batch, t, state, dtype):
    x = make([t] * batch, 2, 2, 128, 128, dtype, packed=False, state=state, seed=t)
    check_forward(x)
    check_forward(x, form="recurrent")
    check_backward(x)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("decay", [0.0, -1e-5, -0.05, -0.9, -6.0, -200.0, float("-inf")])
def test_decays(decay, dtype):
    x = make([300, 1, 40], 1, 2, 128, 128, dtype, seed=5, g=[decay, -0.02])
    check_forward(x)
    check_forward(x, form="recurrent")
    check_backward(x)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", LENS)
def test_backward(lens, dtype):
    check_backward(make(lens, 2, 2, 128, 128, dtype, seed=len(lens)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hv", [(1, 4), (2, 4), (3, 3)])
@pytest.mark.parametrize("shape", [(64, 64), (40, 72), (33, 65), (128, 64), (160, 96)])
def test_backward_shared_heads(shape, hq, hv, dtype):
    check_backward(make([100, 0, 1, 190], hq, hv, *shape, dtype, seed=hv))


def test_no_sequences():
    for packed in (True, False):
        x = make([], 2, 4, 128, 128, torch.bfloat16, packed=packed)
        out, s1 = LinearAttention().chunked(x["q"], x["k"], x["v"], x["g"], cu_seqlens=x["cu"])
        assert out.numel() == 0 and s1.shape[0] == 0


@pytest.mark.parametrize("form", ["chunked", "recurrent"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_padding_is_neither_read_nor_written(form, dtype):
    """Positions behind the last sequence hold NaN; the outputs' stay as they
    were."""
    x = make([130, 5], 2, 4, 128, 128, dtype, pad=90, seed=3)
    y = {**x}
    for key in ("q", "k", "v", "do"):
        y[key] = x[key].clone()
        y[key][135:] = float("nan")
    out = torch.full_like(x["v"], 7.0)
    rule = LinearAttention()
    getattr(rule, form)(y["q"], y["k"], y["v"], y["g"], y["state"], cu_seqlens=y["cu"], out=out)
    ref, _ = getattr(rule, form)(x["q"], x["k"], x["v"], x["g"], x["state"], cu_seqlens=x["cu"])
    assert torch.equal(out[:135], ref[:135]) and bool((out[135:] == 7.0).all())
    got = rule.backward(y["q"], y["k"], y["v"], y["g"], y["do"], y["state"], y["ds"],
                        cu_seqlens=y["cu"])
    want = rule.backward(x["q"], x["k"], x["v"], x["g"], x["do"], x["state"], x["ds"],
                         cu_seqlens=x["cu"])
    for a, b in zip(got[:3], want[:3]):
        assert torch.equal(a[:135], b[:135])
    assert torch.equal(got[3], want[3])


@pytest.mark.parametrize("dtype", TYPES)
def test_a_bad_value_stays_in_its_sequence(dtype):
    """Sequences share tiles of positions; a NaN or an infinity in one reaches
    no other, and nothing before its own 128 positions."""
    lens = [70, 200, 61]
    x = make(lens, 2, 2, 128, 128, dtype, seed=9)
    y = {k: v.clone() if torch.is_tensor(v) else v for k, v in x.items()}
    y["v"][70 + 150, 0, 3] = float("nan")
    y["k"][70 + 160, 1, 5] = float("inf")
    rule = LinearAttention()
    args = lambda z: (z["q"], z["k"], z["v"], z["g"])  # noqa: E731
    a, sa = rule.chunked(*args(x), x["state"], cu_seqlens=x["cu"])
    b, sb = rule.chunked(*args(y), x["state"], cu_seqlens=x["cu"])
    for i, j in ((0, 70), (70, 70 + 128), (270, 331)):
        assert torch.equal(a[i:j], b[i:j])
    assert torch.equal(sa[0], sb[0]) and torch.equal(sa[2], sb[2])
    ga = rule.backward(*args(x), x["do"], x["state"], x["ds"], cu_seqlens=x["cu"])
    gb = rule.backward(*args(y), x["do"], x["state"], x["ds"], cu_seqlens=x["cu"])
    for u, v in zip(ga[:3], gb[:3]):
        assert torch.equal(u[:70], v[:70]) and torch.equal(u[270:], v[270:])


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_inputs_and_given_outputs(dtype):
    """q, k and v cut out of one projection; the state updated in place."""
    x = make([100, 29], 2, 4, 128, 128, dtype, seed=4)
    fused = torch.cat([x["q"], x["k"], x["v"]], dim=1)
    q, k, v = fused.split([2, 2, 4], dim=1)
    ref, s_ref = LinearAttention().chunked(x["q"], x["k"], x["v"], x["g"], x["state"],
                                           cu_seqlens=x["cu"])
    state, out = x["state"].clone(), torch.empty_like(x["v"])
    got, s1 = LinearAttention().chunked(q, k, v, x["g"], state, cu_seqlens=x["cu"].long(),
                                        out=out, state_out=state)
    assert got is out and s1 is state and torch.equal(out, ref) and torch.equal(state, s_ref)
    with pytest.raises(ValueError, match="out is"):
        LinearAttention().chunked(q, k, v, x["g"], cu_seqlens=x["cu"], out=out.float().double())
    with pytest.raises(ValueError, match="state_out is"):
        LinearAttention().chunked(q, k, v, x["g"], cu_seqlens=x["cu"], state_out=state[:1])


def test_pieces_make_the_whole():
    """A prompt in parts, then single tokens, each from the last one's state."""
    x = make([700], 2, 4, 128, 128, torch.float32, seed=8)
    rule = LinearAttention()
    ref, s_ref = rule.chunked(x["q"][None], x["k"][None], x["v"][None], x["g"], x["state"])
    state, outs = x["state"], []
    for i, j in ((0, 300), (300, 301), (301, 690)):
        o, state = rule.chunked(x["q"][None, i:j], x["k"][None, i:j], x["v"][None, i:j], x["g"],
                                state)
        outs.append(o)
    for i in range(690, 700):
        o, state = rule.recurrent(x["q"][None, i:i + 1], x["k"][None, i:i + 1],
                                  x["v"][None, i:i + 1], x["g"], state)
        outs.append(o)
    want, bound, ws, bs = want_core({**x, "cu": x["cu"]}, (x["q"], x["k"], x["v"]), 1.0,
                                    128**-0.5, x["state"], False, False)
    for o, s in ((ref, s_ref), (torch.cat(outs, 1), state)):
        close(o[0], want, bound, x, 0.0, torch.float32, "out")
        close(s, ws, bs, x, 0.0, torch.float32, "state")


@pytest.mark.parametrize("rows,hq,hv,dk,dv", [(1, 16, 32, 128, 128), (5, 2, 2, 64, 64),
                                              (64, 8, 8, 128, 128), (37, 4, 12, 96, 80),
                                              (3, 1, 1, 250, 7)])
@pytest.mark.parametrize("dtype", TYPES)
def test_decode_rows(rows, hq, hv, dk, dv, dtype):
    x = make([1] * rows, hq, hv, dk, dv, dtype, seed=rows, packed=False)
    out, s1 = check_forward(x, form="recurrent")
    state = x["state"].clone()
    out2, _ = LinearAttention().recurrent(x["q"], x["k"], x["v"], x["g"], state, state_out=state)
    assert torch.equal(out, out2) and torch.equal(state, s1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_equal_calls_give_equal_bits(dtype):
    x = make([900, 3, 400], 2, 4, 128, 128, dtype, seed=1)
    first = None
    for _ in range(3):
        rule = LinearAttention()
        got = [*rule.chunked(x["q"], x["k"], x["v"], x["g"], x["state"], cu_seqlens=x["cu"]),
               *rule.backward(x["q"], x["k"], x["v"], x["g"], x["do"], x["state"], x["ds"],
                              cu_seqlens=x["cu"])]
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_gradients_against_differences():
    """The loss is linear in each operand by itself, so its difference along
    any direction of one operand is the gradient's product with it, exactly."""
    x = make([90, 1, 150], 2, 4, 32, 48, torch.float32, seed=12)
    gen = torch.Generator(device=DEV).manual_seed(13)
    grads = LinearAttention().backward(x["q"], x["k"], x["v"], x["g"], x["do"], x["state"],
                                       x["ds"], cu_seqlens=x["cu"])

    def loss(y):
        out, _, s1, _ = want_core(y, (y["q"], y["k"], y["v"]), 1.0, 32**-0.5, y["state"], False,
                                  False)
        return (out * x["do"].double()).sum() + (s1 * x["ds"].double()).sum()

    for key, grad in zip(("q", "k", "v", "state"), grads):
        d = torch.randn(x[key].shape, device=DEV, generator=gen)
        up, down = {**x, key: x[key].double() + d}, {**x, key: x[key].double() - d}
        diff = (loss(up) - loss(down)) / 2
        got = (grad.double() * d).sum()
        # |grad - exact| <= (n + d + 64) 2^-23 A with A of the order of |grad|
        # times the root of its terms; 1e-4 of the sum of absolute products
        # is above (150 + 48 + 64) 2^-23 = 3.1e-5.
        assert abs(float(got - diff)) <= 1e-4 * float((grad.double() * d).abs().sum()), key


def test_streams_threads_and_graphs():
    """Calls on side streams, and captured ones replayed on new inputs and
    interleaved with an eager call, equal the same calls alone."""
    xs = [make([600, 31], 2, 4, 128, 128, dt, seed=i) for i, dt in
          enumerate((torch.bfloat16, torch.float32))]

    def call(x):
        rule = LinearAttention()
        return [*rule.chunked(x["q"], x["k"], x["v"], x["g"], x["state"], cu_seqlens=x["cu"]),
                *rule.backward(x["q"], x["k"], x["v"], x["g"], x["do"], x["state"], x["ds"],
                               cu_seqlens=x["cu"])]

    ref = [call(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for x, s in zip(xs, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(call(x))
    torch.cuda.synchronize()
    for a, b in zip(ref, got):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
    graphs = []
    for x in xs:
        static = {k: v.clone() if torch.is_tensor(v) else v for k, v in x.items()}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call(static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = call(static)
        graphs.append((graph, static, outs))
    for rep in range(2):
        for (graph, static, outs), x, want in zip(graphs, xs, ref):
            for key in ("q", "k", "v", "do"):
                static[key].copy_(x[key] if rep == 0 else -x[key])
            graph.replay()
            eager = call(x)
            torch.cuda.synchronize()
            assert all(torch.equal(u, v) for u, v in zip(eager, want))
            if rep == 0:
                assert all(torch.equal(u, v) for u, v in zip(outs, want))
            else:
                again = call(static)
                torch.cuda.synchronize()
                assert all(torch.equal(u, v) for u, v in zip(outs, again))


def test_the_layer_together():
    """Projection parts through the head norms with rotation, the rule, its
    gradients and the norms' gradients, against 64-bit autograd."""
    gen = torch.Generator(device=DEV).manual_seed(21)
    t, hq, hv, d = 150, 2, 4, 64
    fused = torch.randn(t, 2 * hq + hv, d, device=DEV, generator=gen)
    qw, kw = (1 + 0.2 * torch.randn(d, device=DEV, generator=gen) for _ in range(2))
    g = -torch.rand(hv, device=DEV, generator=gen) * 0.3
    do = torch.randn(t, hv, d, device=DEV, generator=gen)
    pos = torch.arange(t, device=DEV) + 1000
    ang = torch.arange(1200, device=DEV)[:, None].double() * 1e4 ** (
        -torch.arange(0, d, 2, device=DEV).double() / d)
    cos, sin = ang.cos().float(), ang.sin().float()
    q, k, v = fused.split([hq, hq, hv], dim=1)
    cu = torch.tensor([0, 90, t], dtype=torch.int32, device=DEV)
    qn, kn = layer.qk_norm_rope(q, k, pos, cos, sin, qw, kw)
    rule = LinearAttention()
    out, _ = rule.chunked(qn, kn, v, g, cu_seqlens=cu)
    dqn, dkn, dv, _ = rule.backward(qn, kn, v, g, do, cu_seqlens=cu)
    dq, dk, dqw, dkw = layer.qk_norm_rope_backward(dqn, dkn, q, k, pos, cos, sin, qw, kw)

    leaf = [y.double().detach().requires_grad_() for y in (q, k, v, qw, kw)]

    def turn(x, w):
        n = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
        c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
        a, b = n[..., : d // 2], n[..., d // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    qf, kf = turn(leaf[0], leaf[3]), turn(leaf[1], leaf[4])
    qs, ks = share(qf, hv), share(kf, hv)
    zero = torch.zeros(hv, d, d, device=DEV)
    want = torch.cat([core(qs[i:j], ks[i:j], leaf[2][i:j], g, 1.0, d**-0.5, zero, False)[0]
                      for i, j in ((0, 90), (90, t))])
    grads = torch.autograd.grad(want, leaf, do.double())
    # f32 throughout: each step's relative error, at most (150 + 64 + 64) 2^-23
    # = 3.4e-5 of its absolute sums, passes through four steps; absolute sums
    # are within a factor of 10 of the values' norms here, so 4 * 3.4e-4.
    for got, ref in zip((out, dq, dk, dv, dqw, dkw), (want, *grads)):
        ref = ref.detach()
        assert float((got.double() - ref).norm() / ref.norm()) < 1.4e-3


@pytest.mark.parametrize("split", [0, 1, 2, 5])
@pytest.mark.parametrize("state", [True, False])
@pytest.mark.parametrize("shape", [(128, 128), (40, 72)])
def test_segments(shape, state, split):
    """Long sequences in segments: the states before them from a first pass and a
    scan, forward and backward in time; the last segment short, one position,
    or whole."""
    x = make([700, 5, 0, 1281, 1, 640, 129], 2, 2, *shape, torch.bfloat16, seed=split, state=state,
             g=[-0.003, -0.6])
    check_forward(x, "tensor_split", split=split)
    check_backward(x, "tensor_split", split=split)


@pytest.mark.parametrize("algo", ["auto", "tensor", "cuda_core", "tensor_split"])
def test_kernel_families_agree_with_the_definition(algo):
    x = make([300, 0, 513, 64], 2, 4, 128, 128, torch.bfloat16, seed=14)
    check_forward(x, algo)
    check_backward(x, algo)
    y = make([2049], 2, 2, 64, 64, torch.bfloat16, seed=15, packed=False)
    check_forward(y, algo)
    check_backward(y, algo)


@pytest.mark.parametrize("algo", ["tensor", "tensor_split"])
@pytest.mark.parametrize("shape,dtype", [((128, 128), torch.float32), ((128, 128), torch.float16),
                                         ((136, 128), torch.bfloat16), ((60, 64), torch.bfloat16)])
def test_tensor_families_refuse_what_they_do_not_take(shape, dtype, algo):
    x = make([64], 1, 1, *shape, dtype)
    with pytest.raises(_lib.GdrError) as e:
        LinearAttention(algo=algo).chunked(x["q"], x["k"], x["v"], x["g"], cu_seqlens=x["cu"])
    assert e.value.status == _lib.GDR_ERR_UNSUPPORTED


def test_many_sequences_on_few_heads():
    """More jobs than SMs, handed out from the list: every length from 0 to 399."""
    lens = list(range(400))
    x = make(lens, 1, 2, 128, 128, torch.bfloat16, seed=16)
    check_forward(x)
    check_backward(x)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(33, 65), (64, 64), (128, 128), (128, 200)])
@pytest.mark.parametrize("packed", [True, False])
def test_long_sequences_of_every_width(packed, shape, dtype):
    """Long enough for segments in every kernel, with shared key heads."""
    x = make([1700, 0, 700] if packed else [1300, 1300], 1, 2, *shape, dtype, seed=shape[1],
             packed=packed)
    check_forward(x)
    check_backward(x)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,hv", [([6000], 2), ([20000, 130], 16)])
def test_segments_update_a_state_in_place(lens, hv, dtype):
    """The first segment reads the state that the last one writes, which may run
    first where the jobs are more than the CTAs."""
    x = make(lens, 2, hv, 64, 64, dtype, seed=len(lens))
    rule = LinearAttention(algo="auto")
    args = (x["q"], x["k"], x["v"], x["g"])
    want, s_want = rule.chunked(*args, x["state"], cu_seqlens=x["cu"])
    for _ in range(3):
        state = x["state"].clone()
        out, _ = rule.chunked(*args, state, cu_seqlens=x["cu"], state_out=state)
        assert torch.equal(out, want) and torch.equal(state, s_want)
    assert _lib.load().gdr_device_error() == _lib.GDR_OK


def test_calls_from_threads():
    """Four host threads, each with its own stream, at once."""
    import threading

    xs = [make([900, 3, 400], 2, 4, 64, 64, dt, seed=i)
          for i, dt in enumerate((torch.bfloat16, torch.float32, torch.float16, torch.bfloat16))]

    def call(x):
        rule = LinearAttention()
        return [*rule.chunked(x["q"], x["k"], x["v"], x["g"], x["state"], cu_seqlens=x["cu"]),
                *rule.backward(x["q"], x["k"], x["v"], x["g"], x["do"], x["state"], x["ds"],
                               cu_seqlens=x["cu"])]

    ref = [call(x) for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(10):
                    got = call(xs[i])
                    stream.synchronize()
                    if not all(torch.equal(u, v) for u, v in zip(got, ref[i])):
                        bad.append(i)
        except Exception as e:  # noqa: BLE001
            bad.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
    assert _lib.load().gdr_device_error() == _lib.GDR_OK


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_offsets_past_32_bits(dtype):
    """A tensor of more than 2^31 elements: the sequence at its end equals the
    same one alone, and agrees with its steps: in bf16 to the two outputs' own
    roundings and the chunk's operands' (3 x 2^-8 of the largest), else to f32
    sums of (200 + 128 + 64) terms (2^-23 each: 5e-5)."""
    t, tail, hv, d = 270000, 200, 64, 128
    assert (t - tail) * hv * d > 2**31
    gen = torch.Generator(device=DEV).manual_seed(2)
    v = torch.empty(t, hv, d, device=DEV, dtype=dtype).normal_(generator=gen)
    q, k = (torch.empty(t, 1, d, device=DEV, dtype=dtype).normal_(generator=gen) for _ in range(2))
    g = -0.2 * torch.rand(hv, device=DEV, generator=gen)
    cu = torch.tensor([0, t - tail, t], dtype=torch.int32, device=DEV)
    rule = LinearAttention()
    out, state = rule.chunked(q, k, v, g, cu_seqlens=cu)
    one = torch.tensor([0, tail], dtype=torch.int32, device=DEV)
    want, s_want = rule.chunked(q[-tail:], k[-tail:], v[-tail:], g, cu_seqlens=one)
    assert torch.equal(out[-tail:], want) and torch.equal(state[1:], s_want)
    step, s_step = rule.recurrent(q, k, v, g, cu_seqlens=cu[1:])
    tol = 2.0**-6 if dtype == torch.bfloat16 else 1e-4
    assert float((step[-tail:].float() - want.float()).abs().max()) <= \
        tol * float(want.float().abs().max())
    assert float((s_step - s_want).abs().max()) <= 1e-4 * float(s_want.abs().max())
    assert _lib.load().gdr_device_error() == _lib.GDR_OK
