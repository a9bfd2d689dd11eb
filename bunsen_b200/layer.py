"""The gated DeltaNet layer's steps around the rule, on CUDA tensors, through
libgdr's C ABI (include/gdr.h):

* ``causal_conv1d`` -- bunsen's ``causal_depthwise_conv1d``
  (``ops/transformers/linear_attention/causal_conv.rs:36-69``), optionally
  with the layer's silu and its q / k / v channel split
  (``blocks/transformers/mixers/gated_delta_net.rs:396-420``);
* ``gated_norm`` -- ``GatedNorm`` (``gated_delta_net.rs:439-440``) on its own;
* ``state_reorder`` -- ``DeltaNetState::reorder`` (``state.rs:112-135``);
* ``qk_norm_rope`` and its gradient ``qk_norm_rope_backward`` -- the RMS norm of
  every query and key head with the position rotation in the same pass, which
  a mixer with norms on its heads (``LinearAttention``'s, or a softmax one) runs
  on q and k before the rule.

The gates and the gated norm run with the rule itself:
``GatedDeltaRule.chunked(..., gates=..., norm=...)``.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .rule import _DTYPES, _ptr, _stream, on_device


def causal_conv1d(x, weight, state=None, *, cu_seqlens=None, silu=False, splits=None,
                  state_out=None, with_state=True):
    """x ``[B, T, C]`` (or packed ``[T_total, C]`` with ``cu_seqlens``),
    weight ``[C, K]`` in x's dtype, state ``[N, K - 1, C]`` f32 or None.

    Returns ``(outputs, next_state)``: ``outputs`` is the convolution ``[.., C]``
    or, with ``splits=(c0, c1)``, the three channel ranges ``[0, c0)``,
    ``[c0, c1)``, ``[c1, C)`` as separate contiguous tensors; ``next_state``
    ``[N, K - 1, C]`` f32 (None when ``with_state`` is False). ``state_out``
    may be ``state`` (updated in place)."""
    if x.device.type != "cuda":
        raise RuntimeError("libgdr runs on CUDA tensors only")
    if x.dtype not in _DTYPES or weight.dtype != x.dtype:
        raise TypeError("x and weight share one dtype, f32, bf16 or f16")
    packed = cu_seqlens is not None
    if x.dim() != (2 if packed else 3):
        raise ValueError("x is [B, T, C], or [T_total, C] with cu_seqlens")
    c, k = weight.shape
    if x.shape[-1] != c:
        raise ValueError(f"weight [C, K] = {tuple(weight.shape)} against x {tuple(x.shape)}")
    x, weight = x.contiguous(), weight.contiguous()
    lead = tuple(x.shape[:-1])
    n = (cu_seqlens.numel() - 1) if packed else x.shape[0]
    c0, c1 = (c, c) if splits is None else splits
    outs = [torch.empty(lead + (w,), dtype=x.dtype, device=x.device)
            for w in (c0, c1 - c0, c - c1)]
    if state is not None:
        if tuple(state.shape) != (n, k - 1, c):
            raise ValueError(f"the state is [N, K - 1, C] = {(n, k - 1, c)}")
        state = state.to(torch.float32).contiguous()
    if with_state and state_out is None:
        state_out = torch.empty((n, k - 1, c), dtype=torch.float32, device=x.device)
    if packed:
        cu_seqlens = cu_seqlens.to(device=x.device, dtype=torch.int32).contiguous()
    p = _lib.GdrConvParams(batch=0 if packed else x.shape[0],
                           seq_len=x.shape[0] if packed else x.shape[1],
                           n_seqs=n if packed else 0, channels=c, taps=k, split0=c0, split1=c1,
                           silu=int(silu), dtype=_DTYPES[x.dtype])
    status = _lib.load().gdr_causal_conv1d(
        ctypes.byref(p), x.data_ptr(), weight.data_ptr(), _ptr(state),
        *(o.data_ptr() if o.numel() else None for o in outs),
        _ptr(state_out) if with_state else None, _ptr(cu_seqlens), _stream(x.device))
    _lib.check("gdr_causal_conv1d", status)
    return (outs[0] if splits is None else tuple(outs)), (state_out if with_state else None)


def gated_norm(x, z, weight, eps, out=None):
    """bunsen's ``GatedNorm`` (``gated_delta_net.rs:439-440``): ``rmsnorm(x) *
    weight * silu(z)`` over the last axis; x and z share shape and dtype;
    ``out`` may be ``x``."""
    if x.device.type != "cuda":
        raise RuntimeError("libgdr runs on CUDA tensors only")
    if x.dtype not in _DTYPES or z.dtype != x.dtype or z.shape != x.shape:
        raise TypeError("x and z share one shape and one dtype, f32, bf16 or f16")
    x, z = x.contiguous(), z.contiguous()
    weight = weight.to(torch.float32).contiguous()
    if out is None:
        out = torch.empty_like(x)
    width = x.shape[-1]
    status = _lib.load().gdr_gated_norm(x.numel() // width if width else 0, width, x.data_ptr(),
                                        z.data_ptr(), weight.data_ptr(), float(eps),
                                        _DTYPES[x.dtype], out.data_ptr(), _stream(x.device))
    _lib.check("gdr_gated_norm", status)
    return out


def state_reorder(src, sources, out=None):
    """Row ``r`` of the result is row ``sources[r]`` of ``src`` (any trailing
    shape, rows along dim 0); ``sources`` int32 on the device."""
    if src.device.type != "cuda":
        raise RuntimeError("libgdr runs on CUDA tensors only")
    src = src.contiguous()
    sources = sources.to(device=src.device, dtype=torch.int32).contiguous()
    rows = sources.numel()
    if out is None:
        out = torch.empty((rows,) + tuple(src.shape[1:]), dtype=src.dtype, device=src.device)
    row_bytes = src[0].numel() * src.element_size() if src.shape[0] else 0
    status = _lib.load().gdr_state_reorder(src.data_ptr(), out.data_ptr(), sources.data_ptr(),
                                           rows, src.shape[0], row_bytes, _stream(src.device))
    _lib.check("gdr_state_reorder", status)
    return out


def _rope_args(q, k, positions, cos, sin, q_weight, k_weight, eps, interleaved):
    """The checks and the call's struct, the tensors it points at and the
    device of ``qk_norm_rope``."""
    qs, ks, dtype, dev = q.shape, k.shape, q.dtype, q.device
    if dtype not in _DTYPES or k.dtype != dtype:
        raise TypeError("q and k share one dtype, f32, bf16 or f16")
    if len(qs) < 3 or len(ks) != len(qs) or ks[:-2] != qs[:-2] or ks[-1] != qs[-1]:
        raise ValueError(f"q is [..., H_q, d] and k [..., H_k, d] with the same leading dims; got "
                         f"{tuple(qs)} and {tuple(ks)}")
    d = qs[-1]
    if positions.shape != qs[:-2] or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions are int32 or int64 {tuple(qs[:-2])}, one for each token")
    table = cos.shape
    if len(table) != 2 or sin.shape != table or not 0 < 2 * table[1] <= d or table[0] == 0:
        raise ValueError("cos and sin are [positions, rotary_dim / 2], rotary_dim at most d")
    for w in (q_weight, k_weight):
        if w is not None and w.shape != (d,):
            raise ValueError(f"the weights are [d] = ({d},)")
    if dev.type != "cuda":
        raise RuntimeError("libgdr runs on CUDA tensors only")
    for x in (k, positions, cos, sin, q_weight, k_weight):
        if x is not None and x.device != dev:
            raise ValueError(f"every tensor is on q's device {dev}; got one on {x.device}")
    q, k = _token_rows(q), _token_rows(k)
    if positions.dtype is not torch.int32:  # far positions stay outside the tables
        positions = positions.clamp(-1, 2**31 - 1).to(torch.int32)
    positions = positions.contiguous()
    cos, sin, q_weight, k_weight = _f32(cos), _f32(sin), _f32(q_weight), _f32(k_weight)
    (tokens, h_q, _), (q0, q1, _), (k0, k1, _) = q.shape, q.stride(), k.stride()
    p = _lib.GdrQkNormRopeParams(tokens, q0, q1, k0, k1, h_q, k.shape[1], d, 2 * table[1], table[0],
                                 int(interleaved), _DTYPES[dtype], float(eps))
    return p, (q, k, positions, cos, sin, q_weight, k_weight), dev


def _f32(x):
    if x is None or (x.dtype is torch.float32 and x.is_contiguous()):
        return x
    return x.to(torch.float32).contiguous()


def _token_rows(x):
    """``[..., H, d]`` as ``[tokens, H, d]`` with contiguous features: a view
    where the strides allow one (a part of a fused projection), else a copy."""
    y = x if x.dim() == 3 else x.flatten(0, -3)
    return y if y.stride(2) == 1 else y.contiguous()


def qk_norm_rope(q, k, positions, cos, sin, q_weight=None, k_weight=None, eps=1e-6, *,
                 interleaved=False):
    """The RMS norm of every head vector of q ``[..., H_q, d]`` and k
    ``[..., H_k, d]`` (weights ``[d]`` or None), then the rotation of its first
    ``2 cos.shape[1]`` features by the angles of its token's position (cos and
    sin f32 ``[positions, rotary_dim / 2]``, rows picked by ``positions``
    ``[...]``): the pairs ``(i, i + rotary_dim / 2)``, or ``(2i, 2i + 1)`` when
    ``interleaved``. One pass; q and k may be strided parts of one tensor.
    Returns new contiguous ``(q, k)`` in q's dtype. A position outside the
    tables leaves its rows unwritten; ``gdr_device_error`` reports it."""
    p, x, dev = _rope_args(q, k, positions, cos, sin, q_weight, k_weight, eps, interleaved)
    q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    k_out = torch.empty(k.shape, dtype=k.dtype, device=dev)
    on_device(dev, "gdr_qk_norm_rope", ctypes.byref(p), *(_ptr(t) for t in x), q_out.data_ptr(),
              k_out.data_ptr())
    return q_out, k_out


def qk_norm_rope_backward(dq_out, dk_out, q, k, positions, cos, sin, q_weight=None, k_weight=None,
                          eps=1e-6, *, interleaved=False):
    """The gradients of ``qk_norm_rope`` from those of its outputs: ``(dq, dk,
    dq_weight, dk_weight)``, dq and dk contiguous in q's dtype, the weights' in
    f32 (None for a weight that is None), summed over all rows in a fixed order. A row
    whose position is outside the tables is left unwritten and adds nothing."""
    p, x, dev = _rope_args(q, k, positions, cos, sin, q_weight, k_weight, eps, interleaved)
    for g, y in ((dq_out, q), (dk_out, k)):
        if g.shape != y.shape or g.dtype != y.dtype or g.device != dev:
            raise ValueError("dq_out and dk_out are shaped, typed and placed like q and k")
    dq_out, dk_out = dq_out.contiguous(), dk_out.contiguous()
    dq = torch.empty(q.shape, dtype=q.dtype, device=dev)
    dk = torch.empty(k.shape, dtype=k.dtype, device=dev)
    dw = [None if w is None else torch.empty(q.shape[-1], dtype=torch.float32, device=dev)
          for w in (q_weight, k_weight)]
    on_device(dev, "gdr_qk_norm_rope_backward", ctypes.byref(p), dq_out.data_ptr(),
              dk_out.data_ptr(), *(_ptr(t) for t in x), dq.data_ptr(), dk.data_ptr(),
              *(_ptr(w) for w in dw))
    return dq, dk, dw[0], dw[1]
