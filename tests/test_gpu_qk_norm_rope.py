"""qk_norm_rope and its gradient against their definition in 64 bits.

Tolerances are derived: an output is one rounding of an f32 value whose
relative error is at most about (d/32 + 12) 2^-24 of its two products' absolute
sum, so |y - exact| <= u_T |exact| + 24 2^-24 A with A the rotation of absolute
values (f32 also rounds the sum itself: u_T covers it). Gradients pass a mean over d
features: (d + 24) 2^-24 A, A its absolute terms. The weights' gradients sum rows in f32:
at most (rows + d) 2^-24 of the absolute sum. f16 has no step below 2^-24, so
rounding to it also moves a small result by up to 2^-25."""

from __future__ import annotations

import pytest
import torch

from bunsen_b200 import _lib, layer

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
STEP = {torch.float16: 2.0**-25}
EPS = 1e-6
E32 = 2.0**-24


def make(tokens, hq, hk, d, rot, dtype, seed=0, fused=True, table=4096):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    f = dict(device=DEV, generator=gen)
    big = (torch.randn(tokens, hq + hk + 3, d, **f) * 3).to(dtype)
    ang = torch.rand(table, rot // 2, device=DEV, generator=gen) * 6.28
    x = {"q": big[:, :hq], "k": big[:, hq:hq + hk], "cos": ang.cos(), "sin": ang.sin(),
         "positions": torch.randint(0, table, (tokens,), **f),
         "q_weight": 1 + 0.3 * torch.randn(d, **f), "k_weight": 1 + 0.3 * torch.randn(d, **f)}
    if not fused:
        x["q"], x["k"] = x["q"].contiguous(), x["k"].contiguous()
    g = {"dq_out": torch.randn(tokens, hq, d, **f).to(dtype),
         "dk_out": torch.randn(tokens, hk, d, **f).to(dtype)}
    return x, g


def pairs(rot, interleaved):
    i = torch.arange(rot, device=DEV)
    return (i[0::2], i[1::2]) if interleaved else (i[: rot // 2], i[rot // 2:])


def rotated(n, x, interleaved, back=False, bound=False):
    """n [tokens, H, d] rotated by the positions' angles (back: the opposite)."""
    c = x["cos"][x["positions"].long()].double()[:, None]
    s = x["sin"][x["positions"].long()].double()[:, None]
    i, j = pairs(2 * x["cos"].shape[1], interleaved)
    y = n.clone()
    if bound:
        y[..., i] = n[..., i] * c.abs() + n[..., j] * s.abs()
        y[..., j] = n[..., j] * c.abs() + n[..., i] * s.abs()
    else:
        s = -s if back else s
        y[..., i] = n[..., i] * c - n[..., j] * s
        y[..., j] = n[..., j] * c + n[..., i] * s
    return y


def check(x, g, interleaved=False):
    d = x["q"].shape[-1]
    ys = layer.qk_norm_rope(**x, eps=EPS, interleaved=interleaved)
    grads = layer.qk_norm_rope_backward(**g, **x, eps=EPS, interleaved=interleaved)
    for n, (v, w, dy) in enumerate(((x["q"], x["q_weight"], g["dq_out"]),
                                    (x["k"], x["k_weight"], g["dk_out"]))):
        v, w1 = v.double(), torch.ones(d, device=DEV).double() if w is None else w.double()
        u, step = U[x["q"].dtype], STEP.get(x["q"].dtype, 0.0)
        r = 1 / (v.square().mean(-1, keepdim=True) + EPS).sqrt()
        want = rotated(v * r * w1, x, interleaved)
        bound = rotated((v * r * w1).abs(), x, interleaved, bound=True)
        got = ys[n]
        assert got.dtype == x["q"].dtype and got.is_contiguous()
        assert bool(((got.double() - want).abs() <=
                     u * want.abs() + 24 * E32 * bound + step).all())
        dn = rotated(dy.double(), x, interleaved, back=True)
        an = rotated(dy.double().abs(), x, interleaved, bound=True)
        mean = (v * w1 * dn).mean(-1, keepdim=True)
        want = r * (w1 * dn - v * r * r * mean)
        bound = r * (w1.abs() * an + v.abs() * r * r * (v * w1).abs().mul(an).mean(-1, keepdim=True))
        got = grads[n]
        assert got.dtype == x["q"].dtype and got.is_contiguous()
        assert bool(((got.double() - want).abs() <=
                     u * want.abs() + (d + 24) * E32 * bound + step).all())
        if w is None:
            assert grads[2 + n] is None
            continue
        rows = v.shape[0] * v.shape[1]
        want, bound = (v * r * dn).sum((0, 1)), (v.abs() * r * an).sum((0, 1))
        assert bool(((grads[2 + n].double() - want).abs() <= (rows + d) * E32 * bound).all())
    torch.cuda.synchronize()
    assert _lib.load().gdr_device_error() == _lib.GDR_OK
    return ys, grads


TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(64, 64), (64, 16), (128, 128), (128, 32), (256, 64), (96, 48),
                                   (96, 24), (80, 40), (80, 20), (7, 4), (33, 2), (8, 8),
                                   (255, 254)])
def test_widths(d, rot, interleaved, dtype):
    check(*make(37, 5, 3, d, rot, dtype, seed=d + rot), interleaved=interleaved)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [0, 1, 2, 1000])
@pytest.mark.parametrize("hq,hk", [(1, 1), (16, 4), (9, 2)])
def test_counts(tokens, hq, hk, dtype):
    x, g = make(tokens, hq, hk, 128, 128, dtype, seed=tokens)
    _, grads = check(x, g)
    if tokens == 0:
        assert not grads[2].any() and not grads[3].any()


@pytest.mark.parametrize("layout", ["contiguous", "fused", "head-major", "odd offset", "features"])
@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(layout, dtype):
    """Strided views give the bits of their contiguous copies where the same
    kernel takes them, and the same values everywhere."""
    x, g = make(50, 4, 2, 128, 64, dtype, seed=2, fused=False)
    ref = layer.qk_norm_rope(**x, eps=EPS)
    y = {**x}
    for key in ("q", "k"):
        t, h, d = x[key].shape
        if layout == "fused":
            big = torch.zeros(t, h + 2, d, dtype=dtype, device=DEV)
            big[:, 1:-1] = x[key]
            y[key] = big[:, 1:-1]
        elif layout == "head-major":
            y[key] = x[key].transpose(0, 1).contiguous().transpose(0, 1)
        elif layout == "odd offset":  # rows that are not 16-byte aligned
            big = torch.zeros(t, h, d + 3, dtype=dtype, device=DEV)
            big[..., 1:d + 1] = x[key]
            y[key] = big[..., 1:d + 1]
        elif layout == "features":  # features not contiguous: copied
            y[key] = x[key].transpose(1, 2).contiguous().transpose(1, 2)
    got, _ = check(y, g)
    if layout != "odd offset":
        assert all(torch.equal(a, b) for a, b in zip(ref, got))


@pytest.mark.parametrize("dtype", TYPES)
def test_leading_dims_and_types_of_positions(dtype):
    x, g = make(24, 4, 2, 64, 64, dtype, seed=6, fused=False)
    ref = layer.qk_norm_rope(**x, eps=EPS)
    ref_g = layer.qk_norm_rope_backward(**g, **x, eps=EPS)
    shape = lambda t: t.reshape((2, 3, 4) + t.shape[1:])  # noqa: E731
    y = {**x, "q": shape(x["q"]), "k": shape(x["k"]),
         "positions": x["positions"].reshape(2, 3, 4).to(torch.int32)}
    got = layer.qk_norm_rope(**y, eps=EPS)
    got_g = layer.qk_norm_rope_backward(shape(g["dq_out"]), shape(g["dk_out"]), **y, eps=EPS)
    for a, b in zip((*ref, *ref_g), (*got, *got_g)):
        assert torch.equal(a, b.reshape(a.shape))


def test_without_weights_and_zero_rows():
    """No weights: ones. A head vector of zeros stays zero, gradients finite."""
    x, g = make(9, 2, 2, 128, 128, torch.float32, seed=7)
    x["q_weight"] = x["k_weight"] = None
    x["q"][3] = 0
    ys, grads = check(x, g)
    assert not ys[0][3].any() and all(bool(torch.isfinite(t).all()) for t in grads[:2])


@pytest.mark.parametrize("d", [128, 33])
def test_positions_outside_the_tables(d):
    """Skipped and reported; every other row as usual; the weights' gradients
    without them."""
    x, g = make(40, 4, 2, d, 2 * (d // 4), torch.float32, seed=8, table=50)
    bad = {3: -1, 17: 50, 30: 2**31 + 5, 39: -(2**40)}
    y = {**x, "positions": x["positions"].clone()}
    for i, v in bad.items():
        y["positions"][i] = v
    keep = torch.tensor([i not in bad for i in range(40)], device=DEV)
    ref = layer.qk_norm_rope(**x, eps=EPS)
    assert _lib.load().gdr_device_error() == _lib.GDR_OK
    got = layer.qk_norm_rope(**y, eps=EPS)
    torch.cuda.synchronize()
    assert _lib.load().gdr_device_error() == _lib.GDR_ERR_INVALID
    assert all(torch.equal(a[keep], b[keep]) for a, b in zip(ref, got))
    z = {k: v[keep] if v is not None and v.shape[0] == 40 else v for k, v in {**x, **g}.items()}
    want = layer.qk_norm_rope_backward(**z, eps=EPS)
    got = layer.qk_norm_rope_backward(**g, **y, eps=EPS)
    torch.cuda.synchronize()
    assert _lib.load().gdr_device_error() == _lib.GDR_ERR_INVALID
    assert all(torch.equal(a, b[keep]) for a, b in zip(want[:2], got[:2]))
    for a, b in zip(want[2:], got[2:]):  # 40 x 4 rows of f32 sums in another grouping
        assert float((a - b).abs().max()) <= 160 * E32 * 40 * float(a.abs().max() + 1)
    assert _lib.load().gdr_device_error() == _lib.GDR_OK


def test_gradient_against_differences():
    x, g = make(11, 2, 1, 24, 16, torch.float32, seed=10)
    dq, _, dqw, _ = layer.qk_norm_rope_backward(**g, **x, eps=EPS)
    gen = torch.Generator(device=DEV).manual_seed(3)

    def loss(v, w):
        n = v / (v.square().mean(-1, keepdim=True) + EPS).sqrt() * w
        return (rotated(n, x, False) * g["dq_out"].double()).sum()

    v, w, h = x["q"].double(), x["q_weight"].double(), 1e-5
    for grad, a, b in ((dq, 1.0, 0.0), (dqw, 0.0, 1.0)):
        dv = torch.randn(v.shape, device=DEV, generator=gen).double() * a
        dw = torch.randn(w.shape, device=DEV, generator=gen).double() * b
        diff = (loss(v + h * dv, w + h * dw) - loss(v - h * dv, w - h * dw)) / (2 * h)
        dot = grad.double() * (dv if a else dw)
        # f32 gradients (48 2^-24 of the terms), differences to h^2 = 1e-10.
        assert abs(float(dot.sum() - diff)) <= 1e-5 * float(dot.abs().sum())


def test_equal_calls_graph_and_stream():
    x, g = make(3000, 8, 4, 128, 128, torch.bfloat16, seed=11)
    call = lambda: [*layer.qk_norm_rope(**x, eps=EPS),  # noqa: E731
                    *layer.qk_norm_rope_backward(**g, **x, eps=EPS)]
    ref = call()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = call()
    graph.replay()
    eager = call()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ref, outs))
    assert all(torch.equal(a, b) for a, b in zip(ref, eager))
