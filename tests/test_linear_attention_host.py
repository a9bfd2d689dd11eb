"""LinearAttention and qk_norm_rope raise on what their contracts rule out
before they touch a device, and the C entry points reject it before a launch."""

from __future__ import annotations

import ctypes
import subprocess

import pytest
import torch

from bunsen_b200 import _lib, layer
from bunsen_b200.linear_attention import LinearAttention
from tests.conftest import ROOT


def _x(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


OK = dict(q=_x(2, 5, 2, 4), k=_x(2, 5, 2, 4), v=_x(2, 5, 4, 6), log_decay=_x(4))


@pytest.mark.parametrize("change,error,match", [
    (dict(k=_x(2, 5, 2, 5)), ValueError, "must match q"),
    (dict(q=_x(5, 2, 4)), ValueError, "q is"),
    (dict(v=_x(2, 4, 4, 6)), ValueError, "leading dims"),
    (dict(v=_x(2, 5, 3, 6), log_decay=_x(3)), ValueError, "divide"),
    (dict(log_decay=_x(2)), ValueError, "log_decay is"),
    (dict(log_decay=_x(4, 1)), ValueError, "log_decay is"),
    (dict(state=_x(2, 4, 6, 4)), ValueError, "the state is"),
    (dict(k=_x(2, 5, 2, 4, dtype=torch.float16)), TypeError, "share one dtype"),
    (dict(q=_x(2, 5, 2, 4, dtype=torch.float64)), TypeError, "f32, bf16 or f16"),
    (dict(), RuntimeError, "CUDA tensors only"),
])
@pytest.mark.parametrize("form", ["recurrent", "chunked", "backward"])
def test_contract(form, change, error, match):
    args = {**OK, **change}
    if form == "backward":
        args["d_out"] = torch.zeros_like(args["v"])
    with pytest.raises(error, match=match):
        getattr(LinearAttention(), form)(**args)


def test_scale_is_finite():
    with pytest.raises(ValueError, match="finite"):
        LinearAttention(scale=float("inf")).chunked(**OK)


def test_offsets_are_one_dimensional():
    with pytest.raises(ValueError, match="offsets"):
        LinearAttention().chunked(_x(5, 2, 4), _x(5, 2, 4), _x(5, 4, 6), _x(4),
                                  cu_seqlens=torch.zeros(2, 2, dtype=torch.int32))


def _la(**kw):
    base = dict(batch=1, seq_len=4, n_seqs=0, heads_qk=2, heads_v=4, d_k=8, d_v=8,
                dtype=_lib.GDR_DTYPE_F32, algo=0, split_chunks=0, scale=1.0)
    return _lib.GdrLaParams(**{**base, **kw})


@pytest.mark.parametrize("bad,status", [
    (dict(heads_v=3), _lib.GDR_ERR_INVALID), (dict(heads_qk=0), _lib.GDR_ERR_INVALID),
    (dict(d_k=0), _lib.GDR_ERR_INVALID), (dict(dtype=_lib.GDR_DTYPE_F64), _lib.GDR_ERR_INVALID),
    (dict(batch=-1), _lib.GDR_ERR_INVALID), (dict(seq_len=-1), _lib.GDR_ERR_INVALID),
    (dict(scale=float("nan")), _lib.GDR_ERR_INVALID), (dict(algo=9), _lib.GDR_ERR_INVALID),
    (dict(split_chunks=-1), _lib.GDR_ERR_INVALID), (dict(d_v=257), _lib.GDR_ERR_UNSUPPORTED),
    (dict(batch=70000), _lib.GDR_ERR_UNSUPPORTED),
    (dict(batch=60000, seq_len=60000), _lib.GDR_ERR_UNSUPPORTED),
])
def test_entry_points_reject_bad_parameters(bad, status):
    lib, d, p = _lib.load(), ctypes.c_void_p(16), _la(**bad)  # d is never dereferenced
    for fn in (lib.gdr_la_recurrent, lib.gdr_la_chunked):
        assert fn(ctypes.byref(p), d, d, d, d, None, d, d, None, None) == status
    assert lib.gdr_la_backward(ctypes.byref(p), d, d, d, d, d, None, None, d, d, d, None, None,
                               None) == status


def test_entry_points_reject_null_buffers():
    lib, d, p = _lib.load(), ctypes.c_void_p(16), _la()
    assert lib.gdr_la_chunked(None, d, d, d, d, None, d, d, None, None) == _lib.GDR_ERR_INVALID
    for hole in (0, 1, 2, 3, 5, 6):  # q, k, v, log_decay, out, state_out
        args = [d, d, d, d, None, d, d]
        args[hole] = None
        assert lib.gdr_la_chunked(ctypes.byref(p), *args, None, None) == _lib.GDR_ERR_INVALID
    for hole in (0, 1, 2, 3, 4, 7, 8, 9):
        args = [d, d, d, d, d, None, None, d, d, d, None]
        args[hole] = None
        assert lib.gdr_la_backward(ctypes.byref(p), *args, None, None) == _lib.GDR_ERR_INVALID


@pytest.mark.parametrize("name,struct", [("gdr_la_params", _lib.GdrLaParams),
                                         ("gdr_qk_norm_rope_params", _lib.GdrQkNormRopeParams)])
def test_struct_layouts_match_the_header(tmp_path, name, struct):
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "gdr.h"\n'
                   f'int main(void) {{ printf("%zu", sizeof({name}));\n'
                   + "".join(f'printf(" %zu", offsetof({name}, {f}));\n'
                             for f, _ in struct._fields_) + "return 0; }\n")
    subprocess.run(["gcc", "-I", str(ROOT / "include"), "-o", str(tmp_path / "layout"), str(src)],
                   check=True)
    got = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True)
    assert [int(x) for x in got.stdout.split()] == [ctypes.sizeof(struct)] + [
        getattr(struct, f).offset for f, _ in struct._fields_]


ROPE = dict(q=_x(3, 2, 8), k=_x(3, 1, 8), positions=_x(3, dtype=torch.int32), cos=_x(9, 4),
            sin=_x(9, 4), q_weight=_x(8), k_weight=None)


@pytest.mark.parametrize("change,error,match", [
    (dict(k=_x(3, 1, 6)), ValueError, "leading dims"),
    (dict(k=_x(2, 1, 8)), ValueError, "leading dims"),
    (dict(q=_x(2, 8), k=_x(1, 8)), ValueError, "leading dims"),
    (dict(positions=_x(4, dtype=torch.int32)), ValueError, "positions"),
    (dict(positions=_x(3)), ValueError, "positions"),
    (dict(cos=_x(9, 5), sin=_x(9, 5)), ValueError, "rotary_dim"),
    (dict(sin=_x(8, 4)), ValueError, "rotary_dim"),
    (dict(cos=_x(9, 0), sin=_x(9, 0)), ValueError, "rotary_dim"),
    (dict(cos=_x(0, 4), sin=_x(0, 4)), ValueError, "rotary_dim"),
    (dict(q_weight=_x(7)), ValueError, "weights"),
    (dict(q=_x(3, 2, 8, dtype=torch.float64)), TypeError, "one dtype"),
    (dict(), RuntimeError, "CUDA tensors only"),
])
def test_rope_contract(change, error, match):
    args = {**ROPE, **change}
    with pytest.raises(error, match=match):
        layer.qk_norm_rope(**args)
    with pytest.raises(error, match=match):
        layer.qk_norm_rope_backward(torch.zeros_like(args["q"]), torch.zeros_like(args["k"]),
                                    **args)


@pytest.mark.parametrize("bad,status", [
    (dict(tokens=-1), _lib.GDR_ERR_INVALID), (dict(heads_k=0), _lib.GDR_ERR_INVALID),
    (dict(rotary_dim=3), _lib.GDR_ERR_INVALID), (dict(rotary_dim=0), _lib.GDR_ERR_INVALID),
    (dict(rotary_dim=10), _lib.GDR_ERR_INVALID), (dict(table_rows=0), _lib.GDR_ERR_INVALID),
    (dict(eps=-1.0), _lib.GDR_ERR_INVALID), (dict(eps=float("nan")), _lib.GDR_ERR_INVALID),
    (dict(dtype=_lib.GDR_DTYPE_F64), _lib.GDR_ERR_INVALID),
    (dict(head_dim=264), _lib.GDR_ERR_UNSUPPORTED),
    (dict(tokens=2**40), _lib.GDR_ERR_UNSUPPORTED),
])
def test_rope_entry_points_reject_bad_parameters(bad, status):
    base = dict(tokens=3, q_token_stride=16, q_head_stride=8, k_token_stride=8, k_head_stride=8,
                heads_q=2, heads_k=1, head_dim=8, rotary_dim=8, table_rows=9, interleaved=0,
                dtype=_lib.GDR_DTYPE_BF16, eps=1e-6)
    lib, d, p = _lib.load(), ctypes.c_void_p(16), _lib.GdrQkNormRopeParams(**{**base, **bad})
    assert lib.gdr_qk_norm_rope(ctypes.byref(p), *[d] * 9, None) == status
    assert lib.gdr_qk_norm_rope_backward(ctypes.byref(p), *[d] * 13, None) == status


@pytest.mark.parametrize("value", [1e39, -1e39])
def test_scales_and_epsilons_beyond_f32_are_rejected(value):
    """The kernels compute in f32: what is infinite there is not a finite scale."""
    lib, d, p = _lib.load(), ctypes.c_void_p(16), _la(scale=value)
    for fn in (lib.gdr_la_recurrent, lib.gdr_la_chunked):
        assert fn(ctypes.byref(p), d, d, d, d, None, d, d, None, None) == _lib.GDR_ERR_INVALID
    assert lib.gdr_la_backward(ctypes.byref(p), d, d, d, d, d, None, None, d, d, d, None, None,
                               None) == _lib.GDR_ERR_INVALID
    p = _lib.GdrQkNormRopeParams(tokens=3, q_token_stride=16, q_head_stride=8, k_token_stride=8,
                                 k_head_stride=8, heads_q=2, heads_k=1, head_dim=8, rotary_dim=8,
                                 table_rows=9, interleaved=0, dtype=_lib.GDR_DTYPE_BF16, eps=value)
    assert lib.gdr_qk_norm_rope(ctypes.byref(p), *[d] * 9, None) == _lib.GDR_ERR_INVALID
    assert lib.gdr_qk_norm_rope_backward(ctypes.byref(p), *[d] * 13, None) == _lib.GDR_ERR_INVALID
    with pytest.raises(ValueError, match="finite"):
        LinearAttention(scale=value).chunked(**OK)
