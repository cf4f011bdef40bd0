"""The operators of a transformer block at the edges of what their documentation allows."""
import pytest
import torch

import atex_b200 as A
from atex_b200 import testing as T

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


# ---------------------------------------------------------------------------
# gradients of views whose heads are not contiguous: the call copies them
# ---------------------------------------------------------------------------
def transposed(t):
    """The same values with the heads, and not the elements of a head, contiguous."""
    return t.transpose(-1, -2).contiguous().transpose(-1, -2)


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("B,T_,dtype", [(1, 300, "bf16"), (2, 2048, "f16"), (1, 2048, "f32")])
def test_gradient_of_views_that_are_copied(lib, B, T_, dtype, norm):
    hq, hk, hd = 32, 8, 128
    g, dt = gen(B + T_), T.TORCH_DTYPE[dtype]

    def r(*shape):
        return torch.randn(*shape, generator=g, device=DEV).to(dt)
    q, k, dq, dk = r(B, T_, hq, hd), r(B, T_, hk, hd), r(B, T_, hq, hd), r(B, T_, hk, hd)
    sq, sk = (torch.rand(hd, generator=g, device=DEV) + 0.5 for _ in range(2))
    off = (sq - 1, sk - 1) if norm == "layer" else (None, None)
    f, ax = A.rotary_frequencies((16, 24, 24), device=DEV)
    pos = torch.randint(0, 1000, (3, B, T_), generator=g, device=DEV)
    want = A.fused_head_norm_rotary_grad_op(dq, dk, q, k, pos, f, ax, sq, sk, norm=norm)
    qt, kt = transposed(q), transposed(k)
    assert qt.stride(-1) == hq and kt.stride(-1) == hk
    for a, b in ((qt, kt), (qt, k), (q, kt)):
        got = A.fused_head_norm_rotary_grad_op(dq, dk, a, b, pos, f, ax, sq, sk, norm=norm)
        assert all(y is None or torch.equal(x, y) for x, y in zip(got, want))
    leaves = [t.detach().clone().requires_grad_() for t in (qt, kt)]
    assert leaves[0].stride(-1) == hq
    out = A.head_norm_rotary(*leaves, pos, f, ax, sq, sk, *off, norm=norm)
    torch.autograd.backward(out, [dq, dk])
    assert torch.equal(leaves[0].grad, want[0]) and torch.equal(leaves[1].grad, want[1])


# ---------------------------------------------------------------------------
# RMS rows of no elements
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_statistics_of_rows_without_elements(lib, dtype):
    """The mean of nothing is not a number; the buffer's former content is not an answer."""
    x, g = torch.empty(5, 0, dtype=T.TORCH_DTYPE[dtype], device=DEV), torch.ones(0, device=DEV)
    stats = torch.full((5,), 7.0, device=DEV)
    assert torch.isnan(A.fused_rms_norm_op(x, g, out_stats=stats)[1]).all() and torch.isnan(stats).all()
    stats.fill_(7.0)
    assert torch.isnan(A.fused_rms_norm_residual_op(x, x, g, out_stats=stats)[2]).all()


# ---------------------------------------------------------------------------
# LayerNorm and InstanceNorm of no elements
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_layer_norm_statistics_of_rows_without_elements(lib, dtype):
    x, g = torch.empty(5, 0, dtype=T.TORCH_DTYPE[dtype], device=DEV), torch.ones(0, device=DEV)
    stats = torch.full((2, 5), 7.0, device=DEV)
    A.fused_layer_norm_op(x, g, g, out_stats=(stats[0], stats[1]))
    assert torch.isnan(stats).all()
    stats.fill_(7.0)
    A.fused_layer_norm_residual_op(x, x, g, g, out_stats=(stats[0], stats[1]))
    assert torch.isnan(stats).all()


@pytest.mark.parametrize("shape,fmt", [((3, 2, 0, 4), "NC..."), ((3, 0, 4, 2), "N...C")])
def test_instance_norm_statistics_of_items_without_elements(lib, shape, fmt):
    x, g = torch.empty(shape, device=DEV), torch.ones(2, device=DEV)
    stats = torch.full((2, 3, 2), 7.0, device=DEV)
    A.fused_instance_norm_op(x, g, g, data_format=fmt, out_stats=(stats[0], stats[1]))
    assert torch.isnan(stats).all()
