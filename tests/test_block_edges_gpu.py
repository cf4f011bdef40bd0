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


# ---------------------------------------------------------------------------
# second derivatives: refused, not silently left out
# ---------------------------------------------------------------------------
def differentiable_calls():
    g = gen(3)
    x, r = torch.randn(6, 64, generator=g, device=DEV), torch.randn(6, 64, generator=g, device=DEV)
    w, b = torch.rand(64, generator=g, device=DEV) + 0.5, torch.randn(64, generator=g, device=DEV)
    q, k = torch.randn(1, 3, 2, 64, generator=g, device=DEV), torch.randn(1, 3, 1, 64, generator=g, device=DEV)
    f, ax = A.rotary_frequencies((32,), device=DEV)
    pos = torch.arange(3, device=DEV)[None]
    return {
        "rms": (x, lambda t: A.rms_norm(t, w)),
        "rms_residual": (x, lambda t: A.rms_norm_residual(t, r, w)[0]),
        "rms_residual_both": (x, lambda t: sum(A.rms_norm_residual(t, r, w))),
        "layer_residual": (x, lambda t: A.layer_norm_residual(t, r, w, b)[0]),
        "layer_residual_both": (x, lambda t: sum(A.layer_norm_residual(t, r, w, b))),
        "rotary": (q, lambda t: A.head_norm_rotary(t, k, pos, f, ax, w, w)[0]),
        "rotary_none": (q, lambda t: A.head_norm_rotary(t, None, pos, f, ax, norm="none")[0]),
    }


@pytest.mark.parametrize("name", ["rms", "rms_residual", "rms_residual_both", "layer_residual", "layer_residual_both",
                                  "rotary", "rotary_none"])
def test_second_derivatives_are_refused(lib, name):
    x, call = differentiable_calls()[name]
    up = torch.randn(x.shape, generator=gen(4), device=DEV)
    a = x.clone().requires_grad_()
    want, = torch.autograd.grad(call(a), a, up)
    for grads_too in (False, True):
        a, u = x.clone().requires_grad_(), up.clone().requires_grad_(grads_too)
        got, = torch.autograd.grad(call(a), a, u, create_graph=True)
        assert torch.equal(got, want)     # the first derivative is there
        with pytest.raises(RuntimeError, match="first derivatives only"):
            (got * up).sum().backward()   # of the gradient itself
        a = x.clone().requires_grad_()
        got, = torch.autograd.grad(call(a) * a.detach() + a * a, a, up, create_graph=True)
        with pytest.raises(RuntimeError, match="first derivatives only"):
            got.square().sum().backward()   # beside a part that has one


def test_second_derivatives_of_the_sum_alone(lib):
    """The sum passes its gradient on unchanged, so what is built on that gradient has a derivative."""
    g = gen(5)
    x, r = (torch.randn(6, 64, generator=g, device=DEV) for _ in range(2))
    w = torch.ones(64, device=DEV)
    for call in (lambda a: A.rms_norm_residual(a, r, w)[1], lambda a: A.layer_norm_residual(a, r, w, w)[1]):
        a = x.clone().requires_grad_()
        first, = torch.autograd.grad((call(a) ** 3).sum(), a, create_graph=True)
        second, = torch.autograd.grad(first.sum(), a)
        assert torch.allclose(second, 6 * (x + r), rtol=1e-6)


# ---------------------------------------------------------------------------
# the older functions' derivatives
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("name", ["layer", "instance"])
def test_second_derivatives_of_layer_and_instance_norm_are_refused(lib, name):
    """As in the reference, whose gradient ops have no gradient registered (nv_norm_ops.py:27-67)."""
    g = gen(6)
    x = torch.randn(3, 5, 4, 8, generator=g, device=DEV)
    w = torch.rand(8, generator=g, device=DEV) + 0.5
    up = torch.randn(x.shape, generator=g, device=DEV)

    def call(t):
        return A.layer_norm(t, w, w) if name == "layer" else A.instance_norm(t, w, w)
    a = x.clone().requires_grad_()
    want, = torch.autograd.grad(call(a), a, up)
    a = x.clone().requires_grad_()
    got, = torch.autograd.grad(call(a), a, up, create_graph=True)
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="first derivatives only"):
        (got * got + a).sum().backward()


# ---------------------------------------------------------------------------
# wide rows whose mean square is near fp32's end
# ---------------------------------------------------------------------------
def huge(shape, dtype, seed, top):
    """Magnitudes top to top / 16 with both signs, the root mean square at most top."""
    g = gen(seed)
    m = torch.exp2(-4 * torch.rand(shape, generator=g, device=DEV))
    m[..., ::3] = 1.0
    sign = torch.randint(0, 2, shape, generator=g, device=DEV) * 2 - 1
    return (m * sign * top).to(T.TORCH_DTYPE[dtype])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [1, 5, 64, 100, 512, 1001, 1024, 2044, 4096, 8192, 16384, 20001, 40000])
def test_rms_of_rows_whose_mean_square_just_fits(lib, dtype, D):
    """1.8e19 squared is 3.24e38, of 3.40e38 that fp32 holds: mean squares fit, sums of two do not.
    The bounds are those of every row, with two roundings more for the scaled squares and their
    scale, (64 + D / 512) / 2 + 12 units of 2^-24; the squares of the small values, scaled down by a
    power of two, are far from fp32's lower end."""
    for N in (1, 40):
        x = huge((N, D), dtype, D + N, 1.8e19)
        gamma = torch.rand(D, generator=gen(D), device=DEV) + 0.5
        x64 = x.double()
        inv64 = 1 / torch.sqrt((x64 * x64).mean(1) + 1e-5)
        want = x64 * inv64[:, None] * gamma.double()
        allow = U * ((64 + D / 512) / 2 + 12)
        half = torch.finfo(x.dtype).eps / 2 if dtype != "f32" else 0.0
        zero = torch.zeros_like(x)
        for y, inv in (A.fused_rms_norm_op(x, gamma, epsilon=1e-5),
                       A.fused_rms_norm_residual_op(x, zero, gamma, epsilon=1e-5)[::2]):
            assert ((inv.double() - inv64).abs() <= allow * inv64).all()
            assert ((y.double() - want).abs() <= (allow + half * 1.001) * want.abs()).all()


# ---------------------------------------------------------------------------
# narrow heads whose mean square is near fp32's end
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd,rows", [(1, 5), (7, 50), (33, 50), (64, 5), (64, 4000), (80, 3000), (128, 7), (128, 3000),
                                     (256, 1500), (320, 40), (511, 40)])
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_heads_whose_mean_square_just_fits(lib, dtype, hd, rows, norm):
    """Forward: 40 units of 2^-24 of the magnitudes, as for every head, and two more for the scaled
    squares.  For a norm with mean the values are 0.9e19, so that a value less the mean, at most 1.8e19,
    squares to no more than fits, and a sum of 16 of them is far below fp32's end."""
    top = 1.8e19 if norm == "rms" else 0.9e19
    q = huge((1, rows, 2, hd), dtype, hd + rows, top)
    scale = torch.rand(hd, generator=gen(hd), device=DEV) + 0.5
    off = torch.zeros(hd, device=DEV) if norm == "layer" else None
    x = q.double()
    c = x - x.mean(-1, keepdim=True) if norm == "layer" else x
    mag = x.abs() + x.abs().mean(-1, keepdim=True) if norm == "layer" else x.abs()
    inv = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-6)
    half = torch.finfo(q.dtype).eps / 2 if dtype != "f32" else 0.0
    y, _ = A.fused_head_norm_rotary_op(q, None, None, scale_q=scale, offset_q=off, norm=norm, epsilon=1e-6)
    want = c * inv * scale.double()
    assert ((y.double() - want).abs() <= 42 * U * mag * inv * scale.double() + half * 1.001 * want.abs()).all()
    # the gradient forms the statistics again; its terms are 1 / 1e19 and their products with c of order one
    dy = torch.randn(q.shape, generator=gen(9), device=DEV).to(q.dtype)
    dx, _, dscale, _, _, _ = A.fused_head_norm_rotary_grad_op(dy, None, q, None, None, scale_q=scale, norm=norm,
                                                              epsilon=1e-6)
    xh, xm = c * inv, mag * inv
    gy = dy.double() * scale.double()
    lift = gy.mean(-1, keepdim=True) if norm == "layer" else 0.0
    want = inv * (gy - lift - xh * (gy * xh).mean(-1, keepdim=True))
    big = inv * (gy.abs() + gy.abs().mean(-1, keepdim=True) + xm * (gy.abs() * xm).mean(-1, keepdim=True))
    assert ((dx.double() - want).abs() <= 98 * U * big + half * 1.001 * want.abs()).all()
    terms = dy.double() * xh
    allow = U * (34 + 64 + 2 * rows / 16) * (dy.double().abs() * xm).sum((0, 1, 2))
    assert ((dscale.double() - terms.sum((0, 1, 2))).abs() <= allow).all()


# ---------------------------------------------------------------------------
# cosines and sines
# ---------------------------------------------------------------------------
def test_cosines_and_sines_keep_their_last_bit(lib):
    """A pair (1, 0) turned by an angle is its cosine and sine.  The function on the rounded fraction of a
    turn is off by at most one unit of 2^-24 below one (1 ulp, CUDA's bound for sinpif and cospif), the
    correction by the part that fp32 drops rounds once more, by half a unit, and its second order,
    (2 pi 2^-26)^2 / 2, is below 1e-14.  Without the correction the dropped part alone is up to
    2 pi 2^-26 = 1.57 units."""
    rows, pairs = 4096, 64
    f = 10000.0 ** -(torch.arange(pairs, dtype=torch.float64, device=DEV) / pairs)
    ax = torch.zeros(pairs, dtype=torch.int32, device=DEV)
    pos = torch.randint(0, 100000, (1, rows), generator=gen(1), device=DEV)
    q = torch.zeros(1, rows, 1, 2 * pairs, device=DEV)
    q[..., :pairs] = 1.0
    y = A.fused_head_norm_rotary_op(q, None, pos, f, ax, norm="none")[0][0, :, 0].double()
    ang = pos[0, :, None].double() * f
    # an angle's own rounding in 64 bits: 1e5 2^-53 2, in the product here and in turns there
    err = (y - torch.cat((torch.cos(ang), torch.sin(ang)), -1)).abs()
    assert float(err.max()) <= 1.5 * U + 1e-10, float(err.max()) / U


# ---------------------------------------------------------------------------
# column sums of very wide rows
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("N,D", [(8192, 151553), (8192, 131080)])
def test_column_sums_of_many_very_wide_rows(lib, N, D):
    """Rows wider than the row-cached kernels leave few slices of rows, so a thread adds thousands of
    terms.  Equal terms are the worst case: every addition to a growing sum rounds the same way.  Sums
    of at most 256 terms at a time, joined one after the other, are off by 256 + N / 256 units of 2^-24
    and a tree's 32."""
    x = torch.ones(N, D, dtype=torch.bfloat16, device=DEV)
    gamma = torch.ones(D, device=DEV)
    inv = torch.full((N,), 0.1, device=DEV)
    term = float(inv[0])
    want, allow = N * term, U * (256 + N / 256 + 32 + 4) * N * term
    dscale = A.fused_rms_norm_grad_op(x, x, gamma, inv)[1]
    assert float((dscale.double() - want).abs().max()) <= allow, float((dscale.double() - want).abs().max()) / allow
    # 1 - 0.5 = 0.5, times 0.1 rounded: exact halves of the terms above; the offset's terms are one
    mean = torch.full((N,), 0.5, device=DEV)
    _, dscale, doffset = A.fused_layer_norm_residual_grad_op(x, x, x, gamma, mean, inv)
    assert float((dscale.double() - want / 2).abs().max()) <= allow / 2
    assert float((doffset - N).abs().max()) == 0.0     # whole numbers below 2^24 are exact


# ---------------------------------------------------------------------------
# heads of zeros
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("hd,tokens", [(128, 9), (128, 2000), (96, 9), (33, 9)])
def test_heads_of_zeros_leave_the_others_alone(lib, norm, hd, tokens):
    """x-hat of a head of zeros is zero: it adds nothing to the scale's gradient, and its own gradient is
    that of the others with 1/rms = 1/sqrt(eps)."""
    g = gen(hd + tokens)
    q = torch.randn(1, tokens, 2, hd, generator=g, device=DEV)
    dy = torch.randn(1, tokens, 2, hd, generator=g, device=DEV)
    q[0, ::3] = 0.0
    scale = torch.rand(hd, generator=g, device=DEV) + 0.5
    dx, _, dscale, _, doffset, _ = A.fused_head_norm_rotary_grad_op(dy, None, q, None, None, scale_q=scale, norm=norm,
                                                                    epsilon=1e-6)
    gy = dy.double() * scale.double()
    want = (gy - gy.mean(-1, keepdim=True) if norm == "layer" else gy)[0, ::3] * 1e3
    # 1/sqrt(1e-6) in fp32 is off by the 2^-24 of eps and 2 ulp of the root; two products and a mean
    assert ((dx[0, ::3].double() - want).abs() <= 32 * U * (gy.abs() + gy.abs().mean(-1, keepdim=True))[0, ::3] * 1e3).all()
    keep = torch.ones(tokens, dtype=torch.bool, device=DEV)
    keep[::3] = False
    x = q.double()[:, keep]
    c = x - x.mean(-1, keepdim=True) if norm == "layer" else x
    mag = x.abs() + x.abs().mean(-1, keepdim=True) if norm == "layer" else x.abs()
    inv = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-6)
    terms = dy.double()[:, keep] * c * inv
    allow = U * (32 + 64 + 2 * tokens / 16) * (dy.double()[:, keep].abs() * mag * inv).sum((0, 1, 2))
    assert ((dscale.double() - terms.sum((0, 1, 2))).abs() <= allow).all()
    if norm == "layer":
        allow = U * (32 + 64 + 2 * tokens / 16) * dy.double().abs().sum((0, 1, 2))
        assert ((doffset.double() - dy.double().sum((0, 1, 2))).abs() <= allow).all()


@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_heads_of_zeros_without_an_epsilon(lib, norm):
    """0 / 0 is not a number, as in the formula: in the head's own outputs, and in the parameter sums, which
    it is part of.  The other heads' outputs do not see it."""
    g = gen(12)
    q, dy = (torch.randn(1, 9, 2, 64, generator=g, device=DEV) for _ in range(2))
    scale, off = torch.rand(64, generator=g, device=DEV) + 0.5, (torch.zeros(64, device=DEV) if norm == "layer" else None)
    calls = []
    for x in (q.clone(), q):
        if x is q:
            q[0, 4, 1] = 0.0
        calls.append((A.fused_head_norm_rotary_op(x, None, None, scale_q=scale, offset_q=off, norm=norm, epsilon=0.0)[0],
                      A.fused_head_norm_rotary_grad_op(dy, None, x, None, None, scale_q=scale, norm=norm, epsilon=0.0)))
    (y0, grads0), (y, grads) = calls
    others = torch.ones(1, 9, 2, dtype=torch.bool, device=DEV)
    others[0, 4, 1] = False
    assert torch.isnan(y[0, 4, 1]).all() and torch.isnan(grads[0][0, 4, 1]).all() and torch.isnan(grads[2]).all()
    assert torch.equal(y[others], y0[others]) and torch.equal(grads[0][others], grads0[0][others])
    if norm == "layer":
        assert torch.equal(grads[4], grads0[4])     # the offset's sum has no 1/rms in it


# ---------------------------------------------------------------------------
# layers cast to half precision
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("norm", ["rms", "layer", "none"])
def test_a_cast_layer_keeps_its_parameters_in_32_bits(lib, dtype, norm):
    q = torch.randn(1, 5, 2, 64, generator=gen(1), device=DEV).to(dtype)
    layer = A.HeadNormRotary((16, 16), norm=norm)
    pos = torch.arange(10, device=DEV).view(2, 5)
    want = layer(q, q, pos)
    layer = layer.to(dtype)
    assert all(p.dtype == torch.float32 for p in layer.parameters())
    got = layer(q, q, pos)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    rms = A.RMSNormalization()
    want = rms(q)
    assert torch.equal(rms.to(dtype)(q), want)


# ---------------------------------------------------------------------------
# captured graphs of the older ops
# ---------------------------------------------------------------------------
def test_graphs_of_the_layer_norm_gradient_share_no_scratch(lib):
    """Two graphs captured on one stream (torch.cuda.graph's own), replayed at once on two, and an eager call
    that needs more scratch between capture and replay."""
    g = gen(8)

    def inputs(n):
        x, dy = (torch.randn(n, 1024, generator=g, device=DEV).bfloat16() for _ in range(2))
        return x, dy, torch.rand(1024, generator=g, device=DEV) + 0.5
    problems = [inputs(3000), inputs(3000)]

    def step(x, dy, w):
        y, mean, inv = A.fused_layer_norm_op(x, w, w)
        return (y, *A.fused_layer_norm_grad_op(dy, x, w, mean, inv))
    want = [step(*p) for p in problems]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for p in problems:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*p))
        graphs.append(graph)
    x = torch.randn(64, 1 << 18, generator=g, device=DEV).bfloat16()
    w = torch.ones(1 << 18, device=DEV)
    A.fused_layer_norm_grad_op(x, x, w, *A.fused_layer_norm_op(x, w, w)[1:])   # partial rows of 512 KB
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(10):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(want, outs):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


# ---------------------------------------------------------------------------
# outputs that are not their own input's view
# ---------------------------------------------------------------------------
def test_outputs_in_another_inputs_place_are_refused(lib):
    g = gen(2)
    B, T_, h, hd = 2, 6, 4, 64
    q, k = (torch.randn(B, T_, h, hd, generator=g, device=DEV).bfloat16() for _ in range(2))
    f, ax = A.rotary_frequencies((32,), device=DEV)
    pos = torch.arange(T_, device=DEV)[None]
    fresh = torch.empty_like(q)
    other = q.view(-1).view(B, h, T_, hd).transpose(1, 2)     # q's memory, the heads in another order
    args = (pos, f, ax)
    for out in ((k, q), (k, fresh), (fresh, q), (fresh, fresh), (other, fresh)):
        with pytest.raises(ValueError, match="own input|different tensors"):
            A.fused_head_norm_rotary_op(q, k, *args, norm="none", out=out)
        with pytest.raises(ValueError, match="own input|different tensors"):
            A.fused_head_norm_rotary_grad_op(q, k, fresh.clone(), fresh.clone(), *args, norm="none", out=out)
    with pytest.raises(ValueError, match="own input"):
        A.fused_head_norm_rotary_op(q, None, *args, norm="none", out=(other, None))
    # a gradient with a norm reads q and k too; without one it does not
    w, dq, dk = torch.ones(hd, device=DEV), q.clone(), k.clone()
    want = A.fused_head_norm_rotary_grad_op(dq, dk, q, k, *args, w, w)
    for out in ((k, q), (k, fresh), (fresh, q), (other, fresh)):
        with pytest.raises(ValueError, match="own input"):
            A.fused_head_norm_rotary_grad_op(dq, dk, q, k, *args, w, w, out=out)
    qq, kk = q.clone(), k.clone()
    A.fused_head_norm_rotary_grad_op(dq, dk, qq, kk, *args, w, w, out=(qq, kk))
    assert torch.equal(qq, want[0]) and torch.equal(kk, want[1])
    want = A.fused_head_norm_rotary_grad_op(dq, dk, q, k, *args, norm="none")
    got = A.fused_head_norm_rotary_grad_op(dq, dk, q, k, *args, norm="none", out=(k, q))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # a size of one has no stride, and nothing at all has no address
    one = torch.randn(1, 1, 1, hd, device=DEV)
    want = A.fused_head_norm_rotary_op(one, None, pos[:, :1], f, ax, norm="none")[0]
    same = one.as_strided(one.shape, (7, 9, 200, 1))
    A.fused_head_norm_rotary_op(one, None, pos[:, :1], f, ax, norm="none", out=(same, None))
    assert torch.equal(one, want)
    empty = torch.empty(0, T_, h, hd, device=DEV)
    A.fused_head_norm_rotary_op(empty, empty, *args, norm="none", out=(empty, empty))


# ---------------------------------------------------------------------------
# gradients written over the residual branch's
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("N,D", [(300, 64), (300, 260), (300, 1001), (300, 1024), (300, 2044), (9000, 2048), (9000, 4096),
                                 (300, 8192), (2100, 8192), (40, 16384), (40, 40000)])
def test_a_gradient_in_the_residual_branchs_place(lib, dtype, N, D):
    g, dt = gen(N + D), T.TORCH_DTYPE[dtype]
    s, dy, ds = (torch.randn(N, D, generator=g, device=DEV).to(dt) for _ in range(3))
    gamma = torch.rand(D, generator=g, device=DEV) + 0.5
    mean, inv = torch.randn(N, generator=g, device=DEV), torch.rand(N, generator=g, device=DEV) + 0.5
    want = A.fused_rms_norm_residual_grad_op(dy, ds, s, gamma, inv)
    here = ds.clone()
    got = A.fused_rms_norm_residual_grad_op(dy, here, s, gamma, inv, out=here)
    assert got[0] is here and all(torch.equal(a, b) for a, b in zip(got, want))
    want = A.fused_layer_norm_residual_grad_op(dy, ds, s, gamma, mean, inv)
    here = ds.clone()
    got = A.fused_layer_norm_residual_grad_op(dy, here, s, gamma, mean, inv, out=here)
    assert got[0] is here and all(torch.equal(a, b) for a, b in zip(got, want))
