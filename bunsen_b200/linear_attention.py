"""``LinearAttention`` over libgdr: linear attention with a decay for each head,
on CUDA tensors, beside :class:`bunsen_b200.rule.GatedDeltaRule`.

Per (sequence, value head h), with ``w = exp(log_decay[h])`` and the state
``S`` ``[d_k, d_v]`` in f32::

    S_t = w S_{t-1} + k_t v_t^T        o_t = scale S_t^T q_t

The same layouts as the gated delta rule: dense ``[B, T, H, d]``, or packed
``[T_total, H, d]`` with ``cu_seqlens``; ``q`` and ``k`` may carry fewer heads
than ``v`` (value head ``h`` reads key head ``h // (H_v // H_qk)``); states
``[N, H_v, d_k, d_v]`` f32, so ``state_reorder`` and snapshots work on them
alike. ``log_decay`` ``[H_v]`` is at most 0 (minus infinity: a position sees
only itself) and is a constant of the layer: it has no gradient.

``recurrent`` steps a position at a time (decode), ``chunked`` runs prompts,
``backward`` returns the gradients of either. The calls do not record an
autograd graph. Every call runs CUDA kernels of ``libgdr.so``; there is no other
path.
"""

from __future__ import annotations

import ctypes
import dataclasses

import torch

from . import _lib
from .rule import _ALGOS, _DTYPES, _ptr, on_device

_F32_MAX = torch.finfo(torch.float32).max


@dataclasses.dataclass(frozen=True)
class LinearAttention:
    """The operator's options. ``scale``: of the output, None for
    ``1 / sqrt(d_k)``. ``algo`` and ``split_chunks`` as in ``GatedDeltaRule``:
    which kernels run ``chunked`` and ``backward``. ``"auto"`` runs bf16 prompts (widths up
    to 128) with the chunks' scores and a copy of the state rounded to bf16: outputs are off
    by 2.3e-3 (relative 2-norm; their own rounding is 1.7e-3), states by 3e-7. ``"cuda_core"``
    computes them as every other type and calls of few positions are, at f32 accuracy (of
    16-bit types in chunks, scores and the state's copy to 2^-16 of their terms). The
    kernel hangs on the call's counts of positions, sequences and heads, so a sequence may be
    rounded differently in another batch."""

    scale: float | None = None
    algo: str = "auto"  # "auto", "cuda_core", "tensor" or "tensor_split"
    split_chunks: int = 0

    def recurrent(self, q, k, v, log_decay, state=None, *, cu_seqlens=None, out=None,
                  state_out=None):
        """One position at a time. Returns ``(out, state)``: the output in q's
        dtype and the f32 state after the last position. ``state_out`` may be
        ``state`` (updated in place). Positions behind the last sequence of a
        pack are not written. A NaN or an infinity stays in its sequence and head; outputs
        after an infinity may be NaN."""
        return self._forward("gdr_la_recurrent", q, k, v, log_decay, state, cu_seqlens, out,
                             state_out)

    def chunked(self, q, k, v, log_decay, state=None, *, cu_seqlens=None, out=None,
                state_out=None):
        """A chunk at a time, for prompts: the same arguments and results. A
        NaN or an infinity may reach every output of the 128 positions it is
        computed with, and of those after it; it does not reach another
        sequence. Keys wider than 128 are stepped through a position at a time (0.6 to
        1.3 us each), whatever the length."""
        return self._forward("gdr_la_chunked", q, k, v, log_decay, state, cu_seqlens, out,
                             state_out)

    def backward(self, q, k, v, log_decay, d_out, state=None, d_state=None, *, cu_seqlens=None):
        """The gradients ``(dq, dk, dv, d_state_in)`` from ``d_out`` (shaped and
        typed like the output) and ``d_state`` (of the state after the last
        position, None: zeros). ``state`` as in the forward call;
        ``d_state_in`` is None when it is None. dq, dk and dv have the type of
        q; where value heads share a key head, its gradient is their sum, in
        f32 and in a fixed order. Positions behind the last sequence of a pack
        are not written. dv of keys wider than 128, and dk and dq of values wider than 128,
        go a position at a time."""
        dev, n = self._check(q, k, v, log_decay, state, cu_seqlens)
        if tuple(d_out.shape) != tuple(v.shape) or d_out.dtype != q.dtype:
            raise ValueError("d_out is shaped and typed like the output")
        want = (n, v.shape[-2], q.shape[-1], v.shape[-1])
        if d_state is not None and tuple(d_state.shape) != want:
            raise ValueError(f"d_state is [N, H_v, d_k, d_v] = {want}; got {tuple(d_state.shape)}")
        _same_device(dev, d_out, d_state)
        q, k, v, d_out = q.contiguous(), k.contiguous(), v.contiguous(), d_out.contiguous()
        log_decay, state, d_state = _f32(log_decay), _f32(state), _f32(d_state)
        cu_seqlens = _offsets(cu_seqlens, dev)
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        d_state_in = torch.empty_like(state) if state is not None else None
        p = self._params(q, v, cu_seqlens, n)
        on_device(dev, "gdr_la_backward", ctypes.byref(p), q.data_ptr(), k.data_ptr(),
                  v.data_ptr(), log_decay.data_ptr(), d_out.data_ptr(), _ptr(state),
                  _ptr(d_state), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(d_state_in),
                  _ptr(cu_seqlens))
        return dq, dk, dv, d_state_in

    # -- plumbing ------------------------------------------------------------
    def _check(self, q, k, v, log_decay, state, cu_seqlens):
        """The shape contract; returns the device and the number of sequences."""
        qs, vs, dtype, dev = q.shape, v.shape, q.dtype, q.device
        rank = 4 if cu_seqlens is None else 3
        if len(qs) != rank:
            raise ValueError(f"q is {'[B, T, H, Dk]' if rank == 4 else '[T, H, Dk]'}; "
                             f"got {tuple(qs)}")
        if k.shape != qs:
            raise ValueError(f"k {tuple(k.shape)} must match q {tuple(qs)}")
        if len(vs) != rank or vs[:-2] != qs[:-2]:
            raise ValueError(f"v {tuple(vs)} must share q's leading dims {tuple(qs[:-2])}")
        h_qk, h_v = qs[-2], vs[-2]
        if h_qk == 0 or h_v == 0 or h_v % h_qk != 0:
            raise ValueError(f"{h_qk} key heads must divide {h_v} value heads")
        if dtype not in _DTYPES:
            raise TypeError(f"q, k, v in f32, bf16 or f16, not {dtype}")
        if k.dtype != dtype or v.dtype != dtype:
            raise TypeError("q, k and v share one dtype")
        if log_decay.shape != (h_v,):
            raise ValueError(f"log_decay is [H_v] = ({h_v},); got {tuple(log_decay.shape)}")
        if cu_seqlens is None:
            n = qs[0]
        else:
            if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
                raise ValueError("cu_seqlens holds n_seqs + 1 offsets")
            n = cu_seqlens.numel() - 1
        if state is not None:
            if state.shape != (n, h_v, qs[-1], vs[-1]):
                raise ValueError(f"the state is [N, H_v, d_k, d_v] = {(n, h_v, qs[-1], vs[-1])}; "
                                 f"got {tuple(state.shape)}")
        if self.scale is not None and not abs(self.scale) <= _F32_MAX:
            raise ValueError("scale is finite in f32")
        if dev.type != "cuda":
            raise RuntimeError("libgdr runs on CUDA tensors only")
        _same_device(dev, k, v, log_decay, state)
        return dev, n

    def _params(self, q, v, cu_seqlens, n):
        vs = v.shape
        h_qk, d_k = q.shape[-2:]
        scale = d_k ** -0.5 if self.scale is None else self.scale
        if cu_seqlens is None:
            return _lib.GdrLaParams(n, vs[1], 0, h_qk, vs[2], d_k, vs[3], _DTYPES[q.dtype],
                                    _ALGOS[self.algo], self.split_chunks, scale)
        return _lib.GdrLaParams(0, vs[0], n, h_qk, vs[1], d_k, vs[2], _DTYPES[q.dtype],
                                _ALGOS[self.algo], self.split_chunks, scale)

    def _forward(self, fn, q, k, v, log_decay, state, cu_seqlens, out, state_out):
        dev, n = self._check(q, k, v, log_decay, state, cu_seqlens)
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        log_decay, state = _f32(log_decay), _f32(state)
        cu_seqlens = _offsets(cu_seqlens, dev)
        if out is None:
            out = torch.empty_like(v)
        else:
            _output(out, v.shape, q.dtype, dev, "out")
        if state_out is None:
            state_out = torch.empty((n, v.shape[-2], q.shape[-1], v.shape[-1]),
                                    dtype=torch.float32, device=dev)
        else:
            _output(state_out, (n, v.shape[-2], q.shape[-1], v.shape[-1]), torch.float32, dev,
                    "state_out")
        p = self._params(q, v, cu_seqlens, n)
        on_device(dev, fn, ctypes.byref(p), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                  log_decay.data_ptr(), _ptr(state), out.data_ptr(), state_out.data_ptr(),
                  _ptr(cu_seqlens))
        return out, state_out


def _f32(x):
    if x is None or (x.dtype is torch.float32 and x.is_contiguous()):
        return x
    return x.to(torch.float32).contiguous()


def _offsets(cu_seqlens, dev):
    if cu_seqlens is None or (cu_seqlens.dtype is torch.int32 and cu_seqlens.device == dev
                              and cu_seqlens.is_contiguous()):
        return cu_seqlens
    return cu_seqlens.to(device=dev, dtype=torch.int32).contiguous()


def _same_device(dev, *tensors):
    for x in tensors:
        if x is not None and x.device != dev:
            raise ValueError(f"every tensor is on q's device {dev}; got one on {x.device}")


def _output(x, shape, dtype, dev, name):
    if x.shape != shape or x.dtype != dtype or x.device != dev or not x.is_contiguous():
        raise ValueError(f"{name} is a contiguous {dtype} {tuple(shape)} on {dev}")
