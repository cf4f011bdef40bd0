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
Angles are formed in 64 bits up to the fraction of a turn; cosine and sine (off by at most 1.5
units of 2^-24) and everything else are float32, rounded once to the type of q and k.
A head of zeros has x-hat 0, unless epsilon is 0 as well: then it is 0 / 0 and NaN, in its own
outputs and in the parameter sums.

The reference (NVIDIA/atex nv_norms) has no per-head norm and no rotary positions.
"""
from __future__ import annotations

import struct
from typing import Sequence, Tuple

import torch

from . import _lib
from .nv_norm_ops import (InvalidArgumentError, _check, _dtype_code, _first_derivatives_only, _keeping_float32, _param,
                          _remember, _require)
from .rms_norm_ops import _on_stream, _scratch

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


def _readable(t):
    """Whether the elements of a head are contiguous, so that the kernels take the view as it is."""
    return t.stride(-1) == 1 or t.shape[-1] == 1


def _rows_contiguous(t):
    return t if _readable(t) else t.contiguous()


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


def _own_views(outs, ins):
    """In place means into its own input's view: into another view, or the other input, rows would be
    written that are still to be read."""
    for i, o in enumerate(outs):
        for j, t in enumerate(ins):
            if o.data_ptr() == t.data_ptr() and o.numel() and (
                    i != j or any(a != b and n > 1 for a, b, n in zip(o.stride(), t.stride(), o.shape))):
                raise ValueError(f"out[{i}] may share memory with its own input alone, and in the same layout")
    if len(outs) > 1 and outs[0].data_ptr() == outs[1].data_ptr() and outs[0].numel():
        raise ValueError("out[0] and out[1] must be different tensors")


class _Form:
    """What the two directions need of a call's shapes, types, strides and options, once checked."""

    def __init__(self, q, k, positions, inv_freq, pair_axis, scales, offsets, norm, interleaved, epsilon,
                 want_offsets):
        B, T, H, D = _heads(q, "q")
        code = _dtype_code(q, "q")
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
        norm_code, self.vectors = _NORMS[norm]
        self.parts, self.head_dim = 1 if k is None else 2, D
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
        pairs = axes = 0
        pos = (0, 0, 0)
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
            pairs, axes = inv_freq.numel(), positions.shape[0]
            _require(2 * pairs <= D, "inv_freq has ", pairs, " pairs, a head has only ", D, " elements")
            tensors += [(positions, "positions"), (inv_freq, "inv_freq"), (pair_axis, "pair_axis")]
            s = positions.stride()
            pos = (s[0], s[1] if len(s) == 3 else 0, s[-1])
        else:
            _require(inv_freq is None and pair_axis is None, "inv_freq and pair_axis need positions")
        for t, name in tensors:
            _on_cuda(t, name, q.device)
        # views that the kernels cannot read are copied at every call
        self.copies = not all(t is None or t.is_contiguous() for t in (*scales, *offsets, inv_freq, pair_axis))
        self.copies = self.copies or any(t is not None and not _readable(t) for t in (q, k))
        self.empty = B * T == 0
        position_bytes = 8 if positions is None or positions.dtype == torch.int64 else 4
        self.head = (code, norm_code, int(interleaved), epsilon, B, T, D, pairs, axes, position_bytes)
        self.pos = pos
        self.device, self.index = q.device, q.get_device()
        # contiguous tensors of q's and k's shape: fresh outputs, copies, and most gradients
        self.q_shape, self.k_shape = q.shape, None if k is None else k.shape
        self.q_packed = (H, T * H * D, H * D, D)
        self.k_packed = None if k is None else (kh, T * kh * D, kh * D, D)
        # what the kernels read, the copy's layout where there is one: the gradient's workspace
        # follows from it
        self.q = _layout(q) if _readable(q) else self.q_packed
        self.k = (0, 0, 0, 0) if k is None else _layout(k) if _readable(k) else self.k_packed
        self.workspace = None

    def workspace_bytes(self, index):
        """Of the gradient, at the widest accesses the strides allow (addresses may narrow them)."""
        if self.workspace is None:
            if self.vectors == 0 or self.empty:
                self.workspace = 0
            else:
                somewhere = 1 << 20   # an address of full alignment; a size query reads nothing
                packed = _PROBLEM.pack(*self.head, somewhere, *self.pos, somewhere, somewhere, somewhere, *self.q,
                                       somewhere if self.parts > 1 else 0, *self.k, *([somewhere] * 4))
                with torch.cuda.device(index):
                    self.workspace = int(_lib.load().nvn_head_norm_rotary_bwd_workspace_bytes(packed))
        return self.workspace


def _layout(t):
    """(heads, strides of batch, token and head) of a view."""
    s = t.stride()
    return (t.shape[-2], s[0] if len(s) == 4 else 0, s[-3], s[-2])


def _key(t):
    return t if t is None else (t.shape, t.stride(), t.dtype, t.device)


# A call's checks depend on shapes, types, strides, devices and options alone, and a decoding step
# spends more time in them than the GPU in the kernel: what has passed is remembered (bounded).
_forms = {}


def _problem(q, k, positions, inv_freq, pair_axis, scales, offsets, norm, interleaved, epsilon, want_offsets):
    """The checked form of a call, its nvn_head_problem, and q and k as the kernels can read them."""
    interleaved, epsilon = bool(interleaved), float(epsilon)
    try:
        key = (_key(q), _key(k), _key(positions), _key(inv_freq), _key(pair_axis), _key(scales[0]), _key(scales[1]),
               _key(offsets[0]), _key(offsets[1]), norm, interleaved, epsilon, want_offsets)
        form = _forms.get(key)
    except (AttributeError, TypeError):
        form = key = None
    if form is None:
        form = _Form(q, k, positions, inv_freq, pair_axis, scales, offsets, norm, interleaved, epsilon, want_offsets)
        if key is not None:
            _remember(_forms, key, form)
    params = (scales[0], offsets[0], scales[1], offsets[1])
    if form.copies:
        params = [None if t is None else t.contiguous() for t in params]
        inv_freq = None if inv_freq is None else inv_freq.contiguous()
        pair_axis = None if pair_axis is None else pair_axis.contiguous()
        q, k = _rows_contiguous(q), None if k is None else _rows_contiguous(k)
    packed = _PROBLEM.pack(*form.head, _ptr(positions), *form.pos, _ptr(inv_freq), _ptr(pair_axis), q.data_ptr(),
                           *form.q, _ptr(k), *form.k, *[_ptr(t) for t in params])
    # the copies must outlive the launch that reads them
    return form, packed, q, k, (params, inv_freq, pair_axis)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _pack(t):
    """nvn_heads of a view."""
    return None if t is None else _HEADS.pack(t.data_ptr(), *_layout(t))


def _fresh(like):
    """A contiguous tensor like `like` (empty_like is the cheaper call, but keeps a view's strides)."""
    return torch.empty_like(like) if like.is_contiguous() else like.new_empty(like.shape)


def _outputs(form, q, k, out):
    """The two outputs, of the shapes of q and k or their gradients, and their nvn_heads."""
    if out is None:
        q_out = _fresh(q)
        if k is None:
            return q_out, None, _HEADS.pack(q_out.data_ptr(), *form.q_packed), None
        k_out = _fresh(k)
        return (q_out, k_out, _HEADS.pack(q_out.data_ptr(), *form.q_packed),
                _HEADS.pack(k_out.data_ptr(), *form.k_packed))
    q_out, k_out = out
    _checked_out(q_out, q, "out[0]")
    if k is None:
        _own_views((q_out,), (q,))
        return q_out, None, _pack(q_out), None
    _checked_out(k_out, k, "out[1]")
    _own_views((q_out, k_out), (q, k))
    return q_out, k_out, _pack(q_out), _pack(k_out)


def _gradient(g, shape, dtype, form, name):
    """A gradient as the kernels can read it."""
    if not isinstance(g, torch.Tensor) or g.shape != shape or g.dtype != dtype:
        raise InvalidArgumentError(f"{name} must have the shape and dtype of its input")
    if g.device != form.device:
        _on_cuda(g, name, form.device)
    return _rows_contiguous(g)


def fused_head_norm_rotary_op(q, k, positions, inv_freq=None, pair_axis=None, scale_q=None, scale_k=None,
                              offset_q=None, offset_k=None, norm: str = "rms", interleaved: bool = False,
                              epsilon: float = 0.001, out=None):
    """Normalise and rotate queries and keys: returns (q_out, k_out), contiguous.

    k may be None (then so is k_out); positions None skips the rotation.  ``positions`` is int32
    or int64, [axes, tokens] or [axes, batch, tokens]; ``inv_freq`` float64 and ``pair_axis``
    int32 have one entry for each pair (rotary_frequencies makes them; a pair whose axis is not
    one of positions' is not rotated).  Scales and offsets are float32 of head_dim elements.
    ``out`` = (q_out, k_out) supplies the outputs as views of any layout; they may be q and k
    themselves, and overlap nothing else that the call reads or writes."""
    form, packed, q, k, alive = _problem(q, k, positions, inv_freq, pair_axis, (scale_q, scale_k),
                                         (offset_q, offset_k), norm, interleaved, epsilon, True)
    q_out, k_out, to_q, to_k = _outputs(form, q, k, out)
    if form.empty:
        return q_out, k_out
    st = _on_stream(form.index, _lib.load().nvn_head_norm_rotary_fwd, packed, to_q, to_k)
    _check(st, "nvn_head_norm_rotary_fwd")
    return q_out, k_out


def fused_head_norm_rotary_grad_op(q_backprop, k_backprop, q, k, positions, inv_freq=None, pair_axis=None,
                                   scale_q=None, scale_k=None, norm: str = "rms", interleaved: bool = False,
                                   epsilon: float = 0.001, out=None):
    """Gradient of fused_head_norm_rotary_op from its inputs: returns (dq, dk, dscale_q, dscale_k,
    doffset_q, doffset_k), with None for what the form does not have.  The statistics are formed
    again from q and k.  ``out`` = (dq, dk) supplies those as views of any layout, for example the
    slices of a packed projection's gradient; they may be q_backprop and k_backprop themselves, and
    overlap nothing else that the call reads or writes."""
    form, packed, q, k, alive = _problem(q, k, positions, inv_freq, pair_axis, (scale_q, scale_k), (None, None), norm,
                                         interleaved, epsilon, False)
    _require((k is None) == (k_backprop is None), "k_backprop belongs to k")
    q_backprop = _gradient(q_backprop, form.q_shape, q.dtype, form, "q_backprop")
    if k is not None:
        k_backprop = _gradient(k_backprop, form.k_shape, q.dtype, form, "k_backprop")
    dq, dk, to_q, to_k = _outputs(form, q_backprop, k_backprop, out)
    if out is not None and form.vectors:   # q and k are read as well
        _own_views([t for t in (dq, dk) if t is not None], [t for t in (q, k) if t is not None])
    dparams = ws = None
    if form.vectors:
        dparams = scale_q.new_empty((form.parts * form.vectors, form.head_dim))
        if form.empty:
            dparams.zero_()
    if not form.empty:
        nbytes = form.workspace_bytes(form.index)
        if nbytes:
            ws = _scratch(scale_q, nbytes)
        st = _on_stream(form.index, _lib.load().nvn_head_norm_rotary_bwd, packed, _pack(q_backprop),
                        _pack(k_backprop), to_q, to_k, _ptr(dparams), _ptr(ws), nbytes)
        _check(st, "nvn_head_norm_rotary_bwd")
    if dparams is None:
        return dq, dk, None, None, None, None
    sums = dparams.unbind() + (None,) * 4   # scale (and offset) of q, then of k
    if form.vectors == 1:
        return dq, dk, sums[0], sums[1], None, None
    return dq, dk, sums[0], sums[2], sums[1], sums[3]


class _head_norm_rotary_grad(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, scale_q, scale_k, offset_q, offset_k, positions, inv_freq, pair_axis, form):
        out = fused_head_norm_rotary_op(q, k, positions, inv_freq, pair_axis, scale_q, scale_k, offset_q, offset_k,
                                        **form)
        ctx.save_for_backward(q, k, scale_q, scale_k, positions, inv_freq, pair_axis)
        ctx.form = form
        ctx.shapes = [None if t is None else t.shape for t in (scale_q, scale_k, offset_q, offset_k)]
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    @_first_derivatives_only
    def backward(ctx, grad_q, grad_k):
        q, k, scale_q, scale_k, positions, inv_freq, pair_axis = ctx.saved_tensors
        if grad_q is None:
            grad_q = torch.zeros_like(q)
        if grad_k is None and k is not None:
            grad_k = torch.zeros_like(k)
        dq, dk, gq, gk, oq, ok = fused_head_norm_rotary_grad_op(grad_q, grad_k, q, k, positions, inv_freq, pair_axis,
                                                                scale_q, scale_k, **ctx.form)
        sums = [None if g is None else g.view(s) for g, s in zip((gq, gk, oq, ok), ctx.shapes)]
        return dq, dk, *sums, None, None, None, None


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
        # plain attributes and not buffers: a module cast to half precision keeps 64-bit frequencies,
        # and its scales and offsets in 32 (_apply)
        self._rotary = (freq, axis)
        self.gamma_q = self.gamma_k = self.beta_q = self.beta_k = None
        self.built = False

    def _apply(self, fn, *args, **kwargs):
        return super()._apply(_keeping_float32(fn), *args, **kwargs)

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
