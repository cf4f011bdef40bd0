"""RMS normalisation and residual norm gradients: refusals and host-side behaviour.  No GPU."""
import ctypes

import pytest
import torch

import atex_b200 as A
from atex_b200 import _lib as L


def test_shape_and_type_checks(lib):
    x, g, m = torch.zeros(2, 3, 4), torch.ones(4), torch.zeros(6)
    with pytest.raises(A.InvalidArgumentError, match="axis is not packed from last dim"):
        A.fused_rms_norm_op(x, g, axis=[0])
    with pytest.raises(A.InvalidArgumentError, match="axis contains invalid value: 7"):
        A.fused_rms_norm_op(x, g, axis=[7])
    with pytest.raises(A.InvalidArgumentError, match="features of x, got 3 and 4"):
        A.fused_rms_norm_op(x, torch.ones(3))
    with pytest.raises(A.InvalidArgumentError, match="at least 1-dimensional"):
        A.fused_rms_norm_op(torch.zeros(()), g)
    with pytest.raises(TypeError, match="float32"):
        A.fused_rms_norm_op(x, g.half())
    with pytest.raises(TypeError):
        A.fused_rms_norm_op(x.double(), g)
    with pytest.raises(A.InvalidArgumentError, match="residual must have the shape and dtype of x"):
        A.fused_rms_norm_residual_op(x, x[:1], g)
    with pytest.raises(A.InvalidArgumentError, match="residual must have the shape and dtype of x"):
        A.fused_rms_norm_residual_op(x, x.half(), g)
    with pytest.raises(A.InvalidArgumentError, match="y_backprop must have the shape"):
        A.fused_rms_norm_grad_op(x[:1], x, g, m)
    with pytest.raises(A.InvalidArgumentError, match="reserve_space_1 must have the same number"):
        A.fused_rms_norm_grad_op(x, x, g, torch.zeros(5))
    with pytest.raises(A.InvalidArgumentError, match="reserve_space_1 must be 1-dimensional"):
        A.fused_rms_norm_grad_op(x, x, g, m.view(2, 3))
    for bad in (None, x[:1], x.half()):
        with pytest.raises(A.InvalidArgumentError, match="sum_backprop must have the shape"):
            A.fused_rms_norm_residual_grad_op(x, bad, x, g, m)
        with pytest.raises(A.InvalidArgumentError, match="sum_backprop must have the shape"):
            A.fused_layer_norm_residual_grad_op(x, bad, x, g, m, m)
    with pytest.raises(A.InvalidArgumentError, match="reserve_space_2 must have the same number"):
        A.fused_layer_norm_residual_grad_op(x, x, x, g, m, torch.zeros(4))


def test_cpu_tensors_are_refused(lib):
    x, g, m = torch.zeros(6, 4), torch.ones(4), torch.zeros(6)
    for call in (lambda: A.fused_rms_norm_op(x, g), lambda: A.fused_rms_norm_residual_op(x, x, g),
                 lambda: A.fused_rms_norm_grad_op(x, x, g, m),
                 lambda: A.fused_rms_norm_residual_grad_op(x, x, x, g, m),
                 lambda: A.fused_layer_norm_residual_grad_op(x, x, x, g, m, m)):
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            call()


def test_abi_refuses_before_it_touches_cuda(lib):
    n = None
    bad = L.NVN_ERR_INVALID_ARGUMENT
    assert lib.nvn_rms_fwd(7, n, n, 4, 4, 1e-3, n, n, n) == bad
    assert lib.nvn_rms_fwd(0, n, n, -1, 4, 1e-3, n, n, n) == bad
    assert lib.nvn_rms_fwd(0, n, n, 4, 4, 1e-3, n, n, n) == bad
    assert lib.nvn_rms_fwd(0, n, n, 0, 4, 1e-3, n, n, n) == L.NVN_OK
    assert lib.nvn_rms_fwd_residual(0, n, n, n, 4, 4, 1e-3, n, n, n, n) == bad
    assert lib.nvn_rms_fwd_residual(2, n, n, n, 4, 0, 1e-3, n, n, n, n) == L.NVN_OK
    buf = (ctypes.c_float * 64)()
    p = ctypes.cast(buf, ctypes.c_void_p)
    assert lib.nvn_rms_fwd_residual(0, p, p, p, 4, 4, 1e-3, p, p, n, n) == bad      # one place for two outputs
    assert lib.nvn_rms_bwd(0, n, n, n, n, n, 4, 4, n, n, n, 0, n) == bad
    assert lib.nvn_rms_bwd(0, n, n, n, n, n, 4, 0, n, n, n, 0, n) == L.NVN_OK
    assert lib.nvn_ln_bwd_residual(0, n, n, n, n, n, n, 4, 4, n, n, n, n, 0, n) == bad
    off = ctypes.c_void_p((p.value + 255) // 256 * 256 + 4)
    # a workspace that is missing or misaligned is an error and not a write
    for ws in (n, off):
        assert lib.nvn_rms_bwd(0, p, n, p, p, p, 4, 4, p, p, ws, 1 << 20, n) == L.NVN_ERR_WORKSPACE
        assert lib.nvn_ln_bwd_residual(0, p, p, p, p, p, p, 4, 4, p, p, p, ws, 1 << 20, n) == L.NVN_ERR_WORKSPACE
    for fn in (lib.nvn_rms_bwd_workspace_bytes, lib.nvn_ln_bwd_residual_workspace_bytes):
        assert fn(0, 0, 4) == 0 and fn(9, 4, 4) == 0


def test_layer_interface(lib):
    layer = A.RMSNormalization(axis=[1, 2], epsilon=1e-5, name="n")
    layer.build((4, 3, 5))
    assert layer.gamma.shape == (3, 5) and layer.beta is None and len(list(layer.parameters())) == 1
    assert layer.get_config() == {"rms_norm": {"axis": [1, 2], "epsilon": 1e-5, "scale": True, "name": "n"}}
    layer.set_weights([torch.full((3, 5), 2.0).numpy()])
    assert float(layer.get_weights()[0].sum()) == 30.0
    assert not A.RMSNormalization(scale=False)._parameters
    with pytest.raises(ValueError, match="Invalid axis"):
        A.RMSNormalization(axis=5).build((2, 3))
    with pytest.raises(ValueError, match="sorted and unique"):
        bad = A.RMSNormalization(axis=[2, 1])
        bad(torch.zeros(2, 3, 4))
