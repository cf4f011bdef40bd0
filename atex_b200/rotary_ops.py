"""Per-head normalisation of attention queries and keys with rotary positions on several axes.

  fused_head_norm_rotary_op / fused_head_norm_rotary_grad_op      raw ops
  head_norm_rotary                                                differentiable function
  rotary_frequencies                                              inv_freq and pair_axis from sections
  HeadNormRotary                                                  layer that owns the scales

q [batch, tokens, heads, head_dim] and k (with heads of its own) are views: only the elements of
a head must be contiguous, so the slices of a packed projection and head-major tensors (through
``transpose(1, 2)``) are read where they lie.  [tokens, heads, head_dim] is a batch of one.

Every head is normalised over head_dim - ``norm="rms"`` (scale), ``"layer"`` (mean and variance,
scale and offset) or ``"none"`` - and its pair p is turned by the angle
``positions[pair_axis[p], batch, token] * inv_freq[p]``.  The axes may be time, height and width
of a video, row and column of an image, or the one of a text.  Pair p is the elements
(p, p + pairs), or (2p, 2p + 1) with ``interleaved``; elements from 2 * pairs on are not rotated.
Angles are formed in 64 bits, everything else in float32, rounded once to the type of q and k.

The reference (NVIDIA/atex nv_norms) has no per-head norm and no rotary positions.
"""
from __future__ import annotations

import struct
from typing import Sequence, Tuple

import torch

from . import _lib
from .nv_norm_ops import (InvalidArgumentError, _check, _device_guard, _dtype_code, _param, _require,
                          _stream)

__all__ = ["fused_head_norm_rotary_op", "fused_head_norm_rotary_grad_op", "head_norm_rotary",
           "rotary_frequencies", "HeadNormRotary"]

_NORMS = {"none": (_lib.NVN_NORM_NONE, 0), "rms": (_lib.NVN_NORM_RMS, 1), "layer": (_lib.NVN_NORM_LAYER, 2)}

# nvn_heads and nvn_head_problem of include/nvnorms.h
_HEADS = struct.Struct("@Pqqqq")
_PROBLEM = struct.Struct("@iiif" "qqqq" "ii" "Pqqq" "PP" "Pqqqq" "Pqqqq" "PPPP")


def rotary_frequencies(sections: Sequence[int], base: float = 10000.0, shared: bool = False,
                       device=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(inv_freq, pair_axis) for heads whose first sections[0] pairs turn with axis 0, the next
    sections[1] with axis 1, and so on: float64 radians per position, int32 axis numbers.

    Each axis has frequencies base^(-i / sections[axis]) of its own, or with ``shared`` all pairs
    share one ladder base^(-p / pairs) that the sections cut into pieces."""
    sizes = [int(s) for s in sections]
    if not sizes or min(sizes) < 0 or sum(sizes) == 0:
        raise ValueError("sections must be non-negative numbers of pairs, one for each axis")
    axis = torch.cat([torch.full((s,), a, dtype=torch.int32) for a, s in enumerate(sizes)])
    pairs = sum(sizes)
    if shared:
        step = torch.arange(pairs, dtype=torch.float64) / pairs
    else:
        step = torch.cat([torch.arange(s, dtype=torch.float64) / max(s, 1) for s in sizes])
    return (float(base) ** -step).to(device), axis.to(device)


def _heads(t, name):
    """A [batch, tokens, heads, head_dim] tensor's (batch, tokens, heads, head_dim)."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dim() == 4:
        return tuple(t.shape)
    _require(t.dim() == 3, name, " must be [batch, tokens, heads, head_dim] or [tokens, heads, head_dim], got ", t)
    return (1,) + tuple(t.shape)


def _on_cuda(t, name, device):
    if not t.is_cuda:
        raise RuntimeError(f"{name} is on {t.device}: the fused norm ops only run on a CUDA device "
                           "(there is no CPU implementation)")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, q on {device}")


def _rows_contiguous(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _pack(t):
    """(data, heads, stride of batch, token, head) of a view."""
    s = t.stride()
    return (t.data_ptr(), t.shape[-2], s[0] if len(s) == 4 else 0, s[-3], s[-2])


def _checked_out(t, like, name):
    if (not isinstance(t, torch.Tensor) or t.shape != like.shape or t.dtype != like.dtype
            or t.device != like.device):
        raise ValueError(f"{name} must have the shape, dtype and device of its input")
    reach, fine = t.shape[-1], t.shape[-1] == 1 or t.stride(-1) == 1
    for stride, size in sorted(zip(t.stride()[:-1], t.shape[:-1])):
        if size > 1:
            fine = fine and stride >= reach
            reach += stride * (size - 1)
    if t.numel() and not fine:
        raise ValueError(f"{name} must keep the elements of a head contiguous and its heads apart")
    return t


class _Problem:
    """The checked arguments both directions share."""

    def __init__(self, q, k, positions, inv_freq, pair_axis, scales, offsets, norm, interleaved, epsilon,
                 want_offsets):
        B, T, H, D = _heads(q, "q")
        self.code = _dtype_code(q, "q")
        if k is not None:
            kb, kt, kh, kd = _heads(k, "k")
            _require(k.dim() == q.dim() and (kb, kt, kd) == (B, T, D),
                     "k must have q's batch, tokens and head_dim, but q has shape ", q, " and k has shape ", k)
            if k.dtype != q.dtype:
                raise TypeError(f"q ({q.dtype}) and k ({k.dtype}) must have the same dtype")
            _require(kh > 0, "k must have at least one head, got ", k)
        _require(H > 0 and D > 0, "q must have at least one head and one element in it, got ", q)
        if norm not in _NORMS:
            raise InvalidArgumentError(f"norm must be 'rms', 'layer' or 'none', got {norm!r}")
        self.norm, self.vectors = _NORMS[norm]
        self.parts = 1 if k is None else 2
        self.shape, self.head_dim = (B, T, H, D), D
        tensors = [(q, "q")] + ([(k, "k")] if k is not None else [])
        for what, given, wanted in (("scale", scales, norm != "none"),
                                    ("offset", offsets, norm == "layer" and want_offsets)):
            for t, side, there in zip(given, "qk", (True, k is not None)):
                name = f"{what}_{side}"
                if not (wanted and there):
                    _require(t is None, name, " does not belong to norm='", norm, "'" if there else "' without k")
                    continue
                _require(t is not None, "norm='", norm, "' needs ", name)
                _param(t, name)
                _require(t.numel() == D, name, " must have the same number of elements as a head, got ", t.numel(),
                         " and ", D)
                tensors.append((t, name))
        self.pairs = self.axes = 0
        pos = (0, 0, 0, 0, 0)
        if positions is not None:
            if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64):
                raise TypeError("positions must be an int32 or int64 tensor")
            _require(positions.dim() in (2, 3) and positions.shape[0] > 0 and positions.shape[-1] == T
                     and (positions.dim() == 2 or positions.shape[1] == B),
                     "positions must be [axes, tokens] or [axes, batch, tokens], got ", positions, " for q ", q)
            if not isinstance(inv_freq, torch.Tensor) or inv_freq.dtype != torch.float64:
                raise TypeError("inv_freq must be a float64 tensor")
            if not isinstance(pair_axis, torch.Tensor) or pair_axis.dtype != torch.int32:
                raise TypeError("pair_axis must be an int32 tensor")
            _require(inv_freq.dim() == 1 and inv_freq.shape == pair_axis.shape,
                     "inv_freq and pair_axis must be 1-dimensional and of one length, got ", inv_freq, " and ",
                     pair_axis)
            self.pairs, self.axes = inv_freq.numel(), positions.shape[0]
            _require(2 * self.pairs <= D, "inv_freq has ", self.pairs, " pairs, a head has only ", D, " elements")
            tensors += [(positions, "positions"), (inv_freq, "inv_freq"), (pair_axis, "pair_axis")]
        else:
            _require(inv_freq is None and pair_axis is None, "inv_freq and pair_axis need positions")
        for t, name in tensors:
            _on_cuda(t, name, q.device)
        self.q, self.k = _rows_contiguous(q), None if k is None else _rows_contiguous(k)
        self.params = [None if t is None else t.contiguous() for t in (scales[0], offsets[0], scales[1], offsets[1])]
        self.freq = None if positions is None else inv_freq.contiguous()
        self.axis = None if positions is None else pair_axis.contiguous()
        self.positions = positions
        if positions is not None:
            s = positions.stride()
            pos = (positions.data_ptr(), s[0], s[1] if len(s) == 3 else 0, s[-1],
                   4 if positions.dtype == torch.int32 else 8)
        self.packed = _PROBLEM.pack(
            self.code, self.norm, int(bool(interleaved)), float(epsilon), B, T, D, self.pairs, self.axes, pos[4],
            pos[0], pos[1], pos[2], pos[3], 0 if self.freq is None else self.freq.data_ptr(),
            0 if self.axis is None else self.axis.data_ptr(), *_pack(self.q),
            *((0, 0, 0, 0, 0) if self.k is None else _pack(self.k)),
            *[0 if t is None else t.data_ptr() for t in self.params])

    def outputs(self, out):
        if out is None:
            return (torch.empty(self.q.shape, dtype=self.q.dtype, device=self.q.device),
                    None if self.k is None else torch.empty(self.k.shape, dtype=self.q.dtype, device=self.q.device))
        q_out, k_out = out
        _checked_out(q_out, self.q, "out[0]")
        if self.k is not None:
            _checked_out(k_out, self.k, "out[1]")
        return q_out, k_out


def fused_head_norm_rotary_op(q, k, positions, inv_freq=None, pair_axis=None, scale_q=None, scale_k=None,
                              offset_q=None, offset_k=None, norm: str = "rms", interleaved: bool = False,
                              epsilon: float = 0.001, out=None):
    """Normalise and rotate queries and keys: returns (q_out, k_out), contiguous.

    k may be None (then so is k_out); positions None skips the rotation.  ``positions`` is int32
    or int64, [axes, tokens] or [axes, batch, tokens]; ``inv_freq`` float64 and ``pair_axis``
    int32 have one entry for each pair (rotary_frequencies makes them; a pair whose axis is not
    one of positions' is not rotated).  Scales and offsets are float32 of head_dim elements.
    ``out`` = (q_out, k_out) supplies the outputs as views of any layout; they may be q and k
    themselves."""
    p = _Problem(q, k, positions, inv_freq, pair_axis, (scale_q, scale_k), (offset_q, offset_k), norm,
                 interleaved, epsilon, True)
    q_out, k_out = p.outputs(out)
    if q.numel() == 0:
        return q_out, k_out
    device = p.q.device
    with _device_guard(device):
        st = _lib.load().nvn_head_norm_rotary_fwd(p.packed, _HEADS.pack(*_pack(q_out)),
                                                  None if k is None else _HEADS.pack(*_pack(k_out)),
                                                  _stream(device))
    _check(st, "nvn_head_norm_rotary_fwd")
    return q_out, k_out


def fused_head_norm_rotary_grad_op(q_backprop, k_backprop, q, k, positions, inv_freq=None, pair_axis=None,
                                   scale_q=None, scale_k=None, norm: str = "rms", interleaved: bool = False,
                                   epsilon: float = 0.001, out=None):
    """Gradient of fused_head_norm_rotary_op from its inputs: returns (dq, dk, dscale_q, dscale_k,
    doffset_q, doffset_k), with None for what the form does not have.  The statistics are formed
    again from q and k.  ``out`` = (dq, dk) supplies those as views of any layout, for example the
    slices of a packed projection's gradient; they may be q_backprop and k_backprop themselves."""
    p = _Problem(q, k, positions, inv_freq, pair_axis, (scale_q, scale_k), (None, None), norm, interleaved,
                 epsilon, False)
    _require((k is None) == (k_backprop is None), "k_backprop belongs to k")
    grads = []
    for g, x, name in ((q_backprop, q, "q_backprop"), (k_backprop, k, "k_backprop")):
        if x is None:
            grads.append(None)
            continue
        if not isinstance(g, torch.Tensor) or g.shape != x.shape or g.dtype != x.dtype:
            raise InvalidArgumentError(f"{name} must have the shape and dtype of its input")
        _on_cuda(g, name, x.device)
        grads.append(_rows_contiguous(g))
    dq, dk = p.outputs(out)
    device, D = p.q.device, p.head_dim
    if p.vectors:
        fresh = torch.zeros if q.numel() == 0 else torch.empty
        dparams = fresh((p.parts, p.vectors, D), dtype=torch.float32, device=device)
    if q.numel():
        lib = _lib.load()
        with _device_guard(device):
            nbytes = lib.nvn_head_norm_rotary_bwd_workspace_bytes(p.packed) if p.vectors else 0
            ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
            st = lib.nvn_head_norm_rotary_bwd(
                p.packed, _HEADS.pack(*_pack(grads[0])), None if k is None else _HEADS.pack(*_pack(grads[1])),
                _HEADS.pack(*_pack(dq)), None if k is None else _HEADS.pack(*_pack(dk)),
                dparams.data_ptr() if p.vectors else None, None if ws is None else ws.data_ptr(), nbytes,
                _stream(device))
        _check(st, "nvn_head_norm_rotary_bwd")
    if not p.vectors:
        return dq, dk, None, None, None, None
    sums = [[dparams[i, j] if i < p.parts and j < p.vectors else None for i in range(2)] for j in range(2)]
    return dq, dk, sums[0][0], sums[0][1], sums[1][0], sums[1][1]


class _head_norm_rotary_grad(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, scale_q, scale_k, offset_q, offset_k, positions, inv_freq, pair_axis, form):
        out = fused_head_norm_rotary_op(q, k, positions, inv_freq, pair_axis, scale_q, scale_k, offset_q, offset_k,
                                        **form)
        ctx.save_for_backward(q, k, scale_q, scale_k, positions, inv_freq, pair_axis)
        ctx.form = form
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    def backward(ctx, grad_q, grad_k):
        q, k, scale_q, scale_k, positions, inv_freq, pair_axis = ctx.saved_tensors
        if grad_q is None:
            grad_q = torch.zeros_like(q)
        if grad_k is None and k is not None:
            grad_k = torch.zeros_like(k)
        dq, dk, gq, gk, oq, ok = fused_head_norm_rotary_grad_op(grad_q, grad_k, q, k, positions, inv_freq, pair_axis,
                                                                scale_q, scale_k, **ctx.form)
        like = [None if g is None or s is None else g.view(s.shape)
                for g, s in ((gq, scale_q), (gk, scale_k), (oq, scale_q), (ok, scale_k))]
        return dq, dk, *like, None, None, None, None


def head_norm_rotary(q, k, positions, inv_freq=None, pair_axis=None, scale_q=None, scale_k=None, offset_q=None,
                     offset_k=None, norm: str = "rms", interleaved: bool = False, epsilon: float = 0.001):
    """Differentiable fused_head_norm_rotary_op: gradients of q, k, the scales and the offsets."""
    form = {"norm": norm, "interleaved": bool(interleaved), "epsilon": float(epsilon)}
    return _head_norm_rotary_grad.apply(q, k, scale_q, scale_k, offset_q, offset_k, positions, inv_freq, pair_axis,
                                        form)


class HeadNormRotary(torch.nn.Module):
    """The norm and rotation of an attention layer's queries and keys, with scales (and offsets)
    of its own: ``layer(q, k, positions)`` returns the pair.

    ``sections`` are the pairs of each position axis, ``base`` and ``shared`` as in
    rotary_frequencies; ``norm``, ``interleaved`` and ``epsilon`` as in the op.  Scales are
    float32 ones and offsets zeros, created on the first call."""

    def __init__(self, sections, base=10000.0, shared=False, norm="rms", interleaved=False, epsilon=1e-3):
        super().__init__()
        if norm not in _NORMS:
            raise InvalidArgumentError(f"norm must be 'rms', 'layer' or 'none', got {norm!r}")
        self.sections, self.base, self.shared = tuple(int(s) for s in sections), float(base), bool(shared)
        self.norm, self.interleaved, self.epsilon = norm, bool(interleaved), float(epsilon)
        freq, axis = rotary_frequencies(self.sections, self.base, self.shared)
        # plain attributes and not buffers: a module cast to half precision keeps 64-bit frequencies
        self._rotary = (freq, axis)
        self.gamma_q = self.gamma_k = self.beta_q = self.beta_k = None
        self.built = False

    def build(self, head_dim, device=None):
        def new(value):
            return torch.nn.Parameter(torch.full((int(head_dim),), value, dtype=torch.float32, device=device))
        if self.norm != "none":
            self.gamma_q, self.gamma_k = new(1.0), new(1.0)
        if self.norm == "layer":
            self.beta_q, self.beta_k = new(0.0), new(0.0)
        self.built = True

    def forward(self, q, k, positions):
        if not self.built:
            self.build(q.shape[-1], device=q.device)
        if self._rotary[0].device != q.device:
            self._rotary = tuple(t.to(q.device) for t in self._rotary)
        freq, axis = self._rotary
        keys = k is not None
        return head_norm_rotary(q, k, positions, freq, axis, self.gamma_q, self.gamma_k if keys else None,
                                self.beta_q, self.beta_k if keys else None, norm=self.norm,
                                interleaved=self.interleaved, epsilon=self.epsilon)

    call = forward

    def get_config(self):
        return {"head_norm_rotary": {"sections": self.sections, "base": self.base, "shared": self.shared,
                                     "norm": self.norm, "interleaved": self.interleaved, "epsilon": self.epsilon}}
