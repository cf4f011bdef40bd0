"""RMS normalisation, and the gradients of the norms that stand behind a residual add.

  fused_rms_norm_op / fused_rms_norm_grad_op                 y = x scale / sqrt(mean(x^2) + eps)
  fused_rms_norm_residual_op / fused_rms_norm_residual_grad_op   the same on s = T(x + residual)
  fused_layer_norm_residual_grad_op    gradient of fused_layer_norm_residual_op
  rms_norm / rms_norm_residual / layer_norm_residual          differentiable functions
  RMSNormalization                                            layer, like LayerNormalization

The gradient of a residual norm takes two gradients: y_backprop, from what follows the norm,
and sum_backprop, from the residual stream that passes it by.  Both reach s, so
x_backprop = T(norm gradient + sum_backprop) in one pass and with one rounding; it is the
gradient of x and of residual.

The reference normalises by mean and variance only and leaves the residual stream to
TensorFlow (atex/nv_norms/python/ops/nv_norm_ops.py:85-99): argument names, output order and
checks follow its LayerNorm ops (atex/nv_norms/cc/ops/norm_ops.cc:148-174).  scale / offset are
float32, the activations float32, float16 or bfloat16, all arithmetic is float32.
"""
from __future__ import annotations

from typing import Iterable

import torch

from . import _lib
from .nv_norm_ops import (InvalidArgumentError, LayerNormalization, _axis_list, _check, _dtype_code,
                          _first_derivatives_only, _grad_outputs, _keeping_float32, _like_output, _ln_dims,
                          _on_device, _param, _remember, _require, fused_layer_norm_grad_op,
                          fused_layer_norm_residual_op)

__all__ = [
    "fused_rms_norm_op", "fused_rms_norm_grad_op", "fused_rms_norm_residual_op",
    "fused_rms_norm_residual_grad_op", "fused_layer_norm_residual_grad_op",
    "rms_norm", "rms_norm_residual", "layer_norm_residual", "RMSNormalization",
]


def _on_stream(index: int, fn, *args) -> int:
    """fn(*args, stream) with device `index` current, on torch's current stream of that device."""
    if torch._C._cuda_getDevice() == index:
        return fn(*args, torch._C._cuda_getCurrentRawStream(index))
    with torch.cuda.device(index):
        return fn(*args, torch._C._cuda_getCurrentRawStream(index))


def _scratch(like: torch.Tensor, nbytes: int) -> torch.Tensor:
    """Workspace of one call (nbytes a multiple of 256), on the device of the float32 tensor `like`.
    From the caching allocator on the current stream, so that calls on different streams and
    captured graphs never share one, and a captured graph owns its own."""
    return like.new_empty(nbytes // 4)


class _Rows:
    """A checked pair of x and scale: dtype code, rows, features, and the gradients' workspaces."""
    __slots__ = ("code", "N", "D", "bytes")

    def __init__(self, code, N, D):
        self.code, self.N, self.D, self.bytes = code, N, D, {}

    def workspace_bytes(self, fn_name: str, index: int) -> int:
        """A size, asked for once with device `index` current (it follows from the device's SMs)."""
        n = self.bytes.get((fn_name, index))
        if n is None:
            with torch.cuda.device(index):
                n = int(getattr(_lib.load(), fn_name)(self.code, self.N, self.D))
            self.bytes[fn_name, index] = n
        return n


# The checks of x and scale depend on their shapes and types alone; a small decoding step spends
# more time in them than the GPU in the kernel, so what has passed is remembered (bounded).
_rows_cache = {}


def _rows(x, scale, axis) -> _Rows:
    """Checks x and scale against each other."""
    try:
        return _rows_cache[x.shape, x.dtype, scale.shape, scale.dtype, axis]
    except (KeyError, AttributeError, TypeError):
        pass
    _require(isinstance(x, torch.Tensor) and x.dim() > 0, "input must be at least 1-dimensional",
             x if isinstance(x, torch.Tensor) else "")
    code = _dtype_code(x, "x")
    _param(scale, "scale")
    axis = tuple(_axis_list(axis))
    N, D = _ln_dims(x, axis)
    _require(scale.numel() == D, "scale must have the same number of elements as the features "
             "of x, got ", scale.numel(), " and ", D)
    return _remember(_rows_cache, (x.shape, x.dtype, scale.shape, scale.dtype, axis), _Rows(code, N, D))


def _like_x(t, x, name):
    if not isinstance(t, torch.Tensor) or t.shape != x.shape or t.dtype != x.dtype:
        raise InvalidArgumentError(f"{name} must have the shape and dtype of x")


def _saved(t, name, N):
    if isinstance(t, torch.Tensor) and t.dtype == torch.float32 and t.shape == (N,):
        return
    _param(t, name)
    _require(t.dim() == 1, name, " must be 1-dimensional", t)
    _require(t.numel() == N, name, " must have the same number of elements as the batches of x, got ",
             t.numel(), " and ", N)


def _together(*named):
    """Contiguous CUDA tensors, all on one device."""
    device = named[0][0].device
    for t, _ in named:
        if not (t.is_cuda and t.is_contiguous() and t.device == device):
            break
    else:
        return [t for t, _ in named]
    out = _on_device(*named)
    for t, (_, name) in zip(out, named):
        if t.device != out[0].device:
            raise ValueError(f"{name} is on {t.device}, {named[0][1]} on {out[0].device}")
    return out


def _one_output(like_numel, scale, out, name):
    if out is None:
        return scale.new_empty(like_numel)
    device = scale.device
    if out.dtype != torch.float32 or out.numel() != like_numel or not out.is_contiguous() or out.device != device:
        raise ValueError(f"{name} must be a contiguous float32 tensor of {like_numel} elements on {device}")
    return out


# ---------------------------------------------------------------------------
# raw ops
# ---------------------------------------------------------------------------
def fused_rms_norm_op(x, scale, axis: Iterable[int] = (-1,), epsilon: float = 0.001,
                      out: torch.Tensor | None = None, out_stats: torch.Tensor | None = None):
    """y = x * scale / sqrt(mean(x^2) + epsilon) over the packed trailing `axis`: returns
    (y, reserve_space_1), reserve_space_1 the per-row 1/sqrt(mean(x^2) + epsilon), float32 [N].

    `out` may be `x` itself; `out_stats` optionally supplies the reserve_space_1 buffer."""
    rows = _rows(x, scale, axis)
    code, N, D = rows.code, rows.N, rows.D
    x, scale = _together((x, "x"), (scale, "scale"))
    y = _like_output(x, out, "out")
    inv = _one_output(N, scale, out_stats, "out_stats")
    st = _on_stream(x.get_device(), _lib.load().nvn_rms_fwd, code, x.data_ptr(), scale.data_ptr(), N, D,
                    float(epsilon), y.data_ptr(), inv.data_ptr())
    _check(st, "nvn_rms_fwd")
    return y, inv


def fused_rms_norm_residual_op(x, residual, scale, axis: Iterable[int] = (-1,), epsilon: float = 0.001,
                               out: torch.Tensor | None = None, out_sum: torch.Tensor | None = None,
                               out_stats: torch.Tensor | None = None):
    """Residual add + RMS normalisation in one pass: returns (y, s, reserve_space_1) with
    s = (x + residual) rounded to x's dtype and y the norm of s.

    `out_sum` may be `x` or `residual` (the residual stream updated in place), `out` may be `x`
    or `residual`; the two must not be the same tensor."""
    rows = _rows(x, scale, axis)
    code, N, D = rows.code, rows.N, rows.D
    _like_x(residual, x, "residual")
    x, residual, scale = _together((x, "x"), (residual, "residual"), (scale, "scale"))
    y = _like_output(x, out, "out")
    s = _like_output(x, out_sum, "out_sum")
    if N * D and y.data_ptr() == s.data_ptr():
        raise ValueError("out and out_sum must be different tensors")
    inv = _one_output(N, scale, out_stats, "out_stats")
    st = _on_stream(x.get_device(), _lib.load().nvn_rms_fwd_residual, code, x.data_ptr(), residual.data_ptr(),
                    scale.data_ptr(), N, D, float(epsilon), s.data_ptr(), y.data_ptr(), inv.data_ptr())
    _check(st, "nvn_rms_fwd_residual")
    return y, s, inv


def _rms_grad(dy, dsum, x, scale, inv, axis, out_grads, out):
    rows = _rows(x, scale, axis)
    code, N, D = rows.code, rows.N, rows.D
    _like_x(dy, x, "y_backprop")
    _saved(inv, "reserve_space_1", N)
    if dsum is None:
        x, dy, scale, inv = _together((x, "x"), (dy, "y_backprop"), (scale, "scale"), (inv, "reserve_space_1"))
    else:
        _like_x(dsum, x, "sum_backprop")
        x, dy, dsum, scale, inv = _together((x, "x"), (dy, "y_backprop"), (dsum, "sum_backprop"), (scale, "scale"),
                                            (inv, "reserve_space_1"))
    dx = _like_output(x, out, "out")
    dscale = torch.empty_like(scale) if out_grads is None else _one_output(D, scale, out_grads, "out_grads")
    index = x.get_device()
    nbytes = rows.workspace_bytes("nvn_rms_bwd_workspace_bytes", index)
    ws = _scratch(scale, nbytes)
    st = _on_stream(index, _lib.load().nvn_rms_bwd, code, dy.data_ptr(), 0 if dsum is None else dsum.data_ptr(),
                    x.data_ptr(), scale.data_ptr(), inv.data_ptr(), N, D, dx.data_ptr(), dscale.data_ptr(),
                    ws.data_ptr(), nbytes)
    _check(st, "nvn_rms_bwd")
    return dx, dscale


def fused_rms_norm_grad_op(y_backprop, x, scale, reserve_space_1, axis: Iterable[int] = (-1,),
                           epsilon: float = 0.001, out_grads: torch.Tensor | None = None,
                           out: torch.Tensor | None = None):
    """Gradient of fused_rms_norm_op from its saved statistics: returns (x_backprop,
    scale_backprop), the latter in the shape of `scale`.  `out_grads` optionally supplies the
    scale_backprop buffer, `out` the x_backprop buffer."""
    return _rms_grad(y_backprop, None, x, scale, reserve_space_1, axis, out_grads, out)


def fused_rms_norm_residual_grad_op(y_backprop, sum_backprop, s, scale, reserve_space_1,
                                    axis: Iterable[int] = (-1,), epsilon: float = 0.001,
                                    out_grads: torch.Tensor | None = None,
                                    out: torch.Tensor | None = None):
    """Gradient of fused_rms_norm_residual_op: returns (x_backprop, scale_backprop).  `s` is the
    op's sum output, sum_backprop the gradient that reaches it from the residual stream;
    x_backprop is the gradient of x and of residual.  `out` may be sum_backprop."""
    if sum_backprop is None:
        raise InvalidArgumentError("sum_backprop must have the shape and dtype of x")
    return _rms_grad(y_backprop, sum_backprop, s, scale, reserve_space_1, axis, out_grads, out)


def fused_layer_norm_residual_grad_op(y_backprop, sum_backprop, s, scale, reserve_space_1,
                                      reserve_space_2, axis: Iterable[int] = (-1,),
                                      epsilon: float = 0.001, out_grads=None,
                                      out: torch.Tensor | None = None):
    """Gradient of fused_layer_norm_residual_op: returns (x_backprop, scale_backprop,
    offset_backprop).  `s` is the op's sum output, sum_backprop the gradient that reaches it
    from the residual stream; x_backprop is the gradient of x and of residual.  `out` may be
    sum_backprop; `out_grads` optionally supplies the (scale_backprop, offset_backprop) pair."""
    rows = _rows(s, scale, axis)
    code, N, D = rows.code, rows.N, rows.D
    _like_x(y_backprop, s, "y_backprop")
    _like_x(sum_backprop, s, "sum_backprop")
    _saved(reserve_space_1, "reserve_space_1", N)
    _saved(reserve_space_2, "reserve_space_2", N)
    x, dy, dsum, scale, mean, inv = _together((s, "s"), (y_backprop, "y_backprop"), (sum_backprop, "sum_backprop"),
                                              (scale, "scale"), (reserve_space_1, "reserve_space_1"),
                                              (reserve_space_2, "reserve_space_2"))
    dx = _like_output(x, out, "out")
    dscale, doffset = _grad_outputs(scale, out_grads)
    index = x.get_device()
    nbytes = rows.workspace_bytes("nvn_ln_bwd_residual_workspace_bytes", index)
    ws = _scratch(scale, nbytes)
    st = _on_stream(index, _lib.load().nvn_ln_bwd_residual, code, dy.data_ptr(), dsum.data_ptr(), x.data_ptr(),
                    scale.data_ptr(), mean.data_ptr(), inv.data_ptr(), N, D, dx.data_ptr(), dscale.data_ptr(),
                    doffset.data_ptr(), ws.data_ptr(), nbytes)
    _check(st, "nvn_ln_bwd_residual")
    return dx, dscale, doffset


# ---------------------------------------------------------------------------
# differentiable functions
# ---------------------------------------------------------------------------
class _rms_norm_grad(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, axis, epsilon):
        y, inv = fused_rms_norm_op(x, gamma, axis=axis, epsilon=epsilon)
        ctx.save_for_backward(x, gamma, inv)
        ctx.axis = axis
        return y

    @staticmethod
    @_first_derivatives_only
    def backward(ctx, grad_y):
        x, gamma, inv = ctx.saved_tensors
        dx, dgamma = fused_rms_norm_grad_op(grad_y, x, gamma, inv, axis=ctx.axis)
        return dx, dgamma, None, None


class _rms_norm_residual_grad(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, gamma, axis, epsilon):
        y, s, inv = fused_rms_norm_residual_op(x, residual, gamma, axis=axis, epsilon=epsilon)
        ctx.save_for_backward(s, gamma, inv)
        ctx.axis = axis
        ctx.set_materialize_grads(False)
        return y, s

    @staticmethod
    def backward(ctx, grad_y, grad_s):
        if grad_y is None:   # only the sum was used: its gradient passes, with whatever graph it has
            return grad_s, grad_s, None, None, None
        return _rms_norm_residual_grad.through_norm(ctx, grad_y, grad_s)

    @staticmethod
    @_first_derivatives_only
    def through_norm(ctx, grad_y, grad_s):
        s, gamma, inv = ctx.saved_tensors
        dx, dgamma = _rms_grad(grad_y, grad_s, s, gamma, inv, ctx.axis, None, None)
        return dx, dx, dgamma, None, None


class _layer_norm_residual_grad(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, gamma, beta, axis, epsilon):
        y, s, mean, inv = fused_layer_norm_residual_op(x, residual, gamma, beta, axis=axis, epsilon=epsilon)
        ctx.save_for_backward(s, gamma, mean, inv)
        ctx.axis = axis
        ctx.set_materialize_grads(False)
        return y, s

    @staticmethod
    def backward(ctx, grad_y, grad_s):
        if grad_y is None:
            return grad_s, grad_s, None, None, None, None
        return _layer_norm_residual_grad.through_norm(ctx, grad_y, grad_s)

    @staticmethod
    @_first_derivatives_only
    def through_norm(ctx, grad_y, grad_s):
        s, gamma, mean, inv = ctx.saved_tensors
        if grad_s is None:
            dx, dgamma, dbeta = fused_layer_norm_grad_op(grad_y, s, gamma, mean, inv, axis=ctx.axis)
        else:
            dx, dgamma, dbeta = fused_layer_norm_residual_grad_op(grad_y, grad_s, s, gamma, mean, inv,
                                                                  axis=ctx.axis)
        return dx, dx, dgamma, dbeta, None, None


def rms_norm(x, gamma, axis=(-1,), epsilon=0.001):
    """Differentiable y = fused_rms_norm_op(x)."""
    return _rms_norm_grad.apply(x, gamma, tuple(_axis_list(axis)), float(epsilon))


def rms_norm_residual(x, residual, gamma, axis=(-1,), epsilon=0.001):
    """Differentiable (y, s): s = x + residual, y = RMS norm of s."""
    return _rms_norm_residual_grad.apply(x, residual, gamma, tuple(_axis_list(axis)), float(epsilon))


def layer_norm_residual(x, residual, gamma, beta, axis=(-1,), epsilon=0.001):
    """Differentiable (y, s): s = x + residual, y = LayerNorm of s."""
    return _layer_norm_residual_grad.apply(x, residual, gamma, beta, tuple(_axis_list(axis)), float(epsilon))


class RMSNormalization(LayerNormalization):
    """LayerNormalization's counterpart without mean and offset: keyword arguments ``axis``
    (int or list, default -1; the packed trailing dims), ``epsilon`` (default 1e-3) and
    ``scale``; gamma is float32 and created on the first call.  Called with a residual it
    returns (y, s) of the residual form."""

    def __init__(self, axis=-1, epsilon=1e-3, scale=True, **kwargs):
        super().__init__(axis=axis, epsilon=epsilon, center=False, scale=scale, **kwargs)

    def _apply(self, fn, *args, **kwargs):
        return super()._apply(_keeping_float32(fn), *args, **kwargs)

    def build(self, input_shape, device=None):
        super().build(input_shape, device=device)
        self.beta = None

    def forward(self, inputs, residual=None):
        if not self.built:
            self.build(tuple(inputs.shape), device=inputs.device)
        axis = _axis_list(self.axis)
        if axis != sorted(set(axis)):
            raise ValueError("We only support sorted and unique axis to make sure the weights "
                             "have the same data layout with the keras layers.")
        if residual is None:
            return rms_norm(inputs, self.gamma, axis=axis, epsilon=self.epsilon)
        return rms_norm_residual(inputs, residual, self.gamma, axis=axis, epsilon=self.epsilon)

    call = forward

    def get_weights(self):
        return [self.gamma.detach().cpu().numpy()]

    def set_weights(self, weights):
        (g,) = weights
        with torch.no_grad():
            self.gamma.copy_(torch.as_tensor(g, dtype=torch.float32).reshape(self.gamma.shape))

    @property
    def variables(self):
        return [self.gamma]

    weights = variables

    def get_config(self):
        cfg = {"axis": self.axis, "epsilon": self.epsilon, "scale": self.scale}
        cfg.update(self._extra)
        return {"rms_norm": cfg}
