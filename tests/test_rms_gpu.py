"""RMS normalisation and the gradients of the residual norms on the GPU, against their
formulas in 64 bits.

Tolerances follow from the arithmetic.  u = 2^-24 is the fp32 rounding; a sum of n terms of
which L are added one after the other in a thread is off by at most (L + tree) u sum|terms|.
Rows: a thread adds at most 32 values of a row-cached row, D / 512 of any other, and the tree
over threads is below 32 deep, so L = 64 + D / 512 covers both; columns: at most a sixteenth of
the rows one after the other.  Results in 16 bits are rounded once more, by eps / 2 of their
value (fp16 below its normal range by half of 2^-24).
"""
import pytest
import torch

import atex_b200 as A
from atex_b200 import _lib
from atex_b200 import testing as T

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
DTYPES = ["f32", "f16", "bf16"]

# every kind of shape: single elements, widths of 1, 2, 4 and 8 elements per access, widths that
# fill a thread layout and that do not, the last width of the row-cached kernels and wider rows
WIDTHS = [1, 2, 7, 8, 33, 64, 100, 128, 250, 256, 384, 768, 1000, 1001, 1024, 2044, 2048, 2050, 4096, 4097, 5120,
          8192, 8200, 16384, 16392, 20001, 32768, 40000]


def rnd(t):
    return torch.finfo(t).eps / 2 if t != torch.float32 else 0.0


def tiny(t):
    return 2.0 ** -25 if t == torch.float16 else 0.0


def close(got, ref, bound, what):
    """|got - ref| <= rounding of ref to got's type + bound, everywhere."""
    g = got.double()
    allow = rnd(got.dtype) * ref.abs() * (1 + 1e-3) + bound + tiny(got.dtype)
    bad = ~((g - ref).abs() <= allow)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst "
                           f"{float(((g - ref).abs() / (allow + 1e-300)).max()):.3f} of the allowance")


def data(N, D, dtype, seed, shift=0.3):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = T.TORCH_DTYPE[dtype]

    def r(*shape):
        return torch.randn(*shape, generator=g, device=DEV)
    x = (r(N, D) * 2 + shift).to(dt)
    res = (r(N, D) * 1.5).to(dt)
    dy, ds = r(N, D).to(dt), r(N, D).to(dt)
    gamma = torch.rand(D, generator=g, device=DEV) + 0.5
    beta = r(D) * 0.1
    return x, res, dy, ds, gamma, beta


def rms_reference(s, gamma, eps):
    s = s.double()
    inv = 1 / torch.sqrt((s * s).mean(1) + eps)
    return s * inv[:, None] * gamma.double(), inv


def check_forward(x, res, gamma, eps, y, s, inv):
    D = x.shape[1]
    if res is not None:
        want = (x.float() + res.float()).to(x.dtype)
        assert torch.equal(s, want), "the residual sum is one fp32 addition rounded once"
        x = want
    y64, inv64 = rms_reference(x, gamma, eps)
    L = 64 + D / 512
    close(inv, inv64, U * (L / 2 + 8) * inv64, "inv_rms")
    close(y, y64, U * (L / 2 + 10) * y64.abs(), "y")


def grad_reference(dy, ds, x, gamma, inv, mean=None):
    """dx, dgamma, dbeta and the sums of magnitudes that bound their errors, in 64 bits."""
    dy, x, gamma, inv = dy.double(), x.double(), gamma.double(), inv.double()[:, None]
    c = x if mean is None else x - mean.double()[:, None]
    xh, gy = c * inv, dy * gamma
    along = (gy * xh).mean(1, keepdim=True)
    lift = gy.mean(1, keepdim=True) if mean is not None else 0.0
    dx = inv * (gy - lift - xh * along)
    big = inv * (gy.abs() + xh.abs() * (gy * xh).abs().mean(1, keepdim=True))
    if mean is not None:
        # x - mean rounds once relative to the larger of the two
        off = inv * (x.abs() + mean.double().abs()[:, None])
        big = big + inv * (gy.abs().mean(1, keepdim=True) + off * (gy * xh).abs().mean(1, keepdim=True)
                           + xh.abs() * (gy.abs() * off).mean(1, keepdim=True))
    if ds is not None:
        dx = dx + ds.double()
        big = big + ds.double().abs()
    terms = dy * xh
    big_g = terms.abs().sum(0)
    if mean is not None:
        big_g = big_g + (dy.abs() * off).sum(0)
    return dx, terms.sum(0), dy.sum(0), big, big_g, dy.abs().sum(0)


def check_grad(dy, ds, x, gamma, inv, dx, dg, mean=None, db=None):
    N, D = x.shape
    r = grad_reference(dy, ds, x, gamma, inv, mean)
    close(dx, r[0], U * (64 + D / 512 + 12) * r[3], "dx")
    L = 64 + N / 16
    close(dg, r[1], U * L * r[4], "dgamma")
    if db is not None:
        close(db, r[2], U * L * r[5], "dbeta")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", WIDTHS)
def test_forward_and_gradients_over_the_widths(lib, dtype, D):
    for N in (1, 37) if D > 2048 else (1, 5, 333):
        x, res, dy, ds, gamma, beta = data(N, D, dtype, 7 * D + N)
        y, inv = A.fused_rms_norm_op(x, gamma, epsilon=1e-5)
        check_forward(x, None, gamma, 1e-5, y, None, inv)
        dx, dg = A.fused_rms_norm_grad_op(dy, x, gamma, inv)
        check_grad(dy, None, x, gamma, inv, dx, dg)
        y, s, inv = A.fused_rms_norm_residual_op(x, res, gamma, epsilon=1e-5)
        check_forward(x, res, gamma, 1e-5, y, s, inv)
        dx, dg = A.fused_rms_norm_residual_grad_op(dy, ds, s, gamma, inv)
        check_grad(dy, ds, s, gamma, inv, dx, dg)
        _, s, mean, iv = A.fused_layer_norm_residual_op(x, res, gamma, beta, epsilon=1e-5)
        dx, dg, db = A.fused_layer_norm_residual_grad_op(dy, ds, s, gamma, mean, iv)
        check_grad(dy, ds, s, gamma, iv, dx, dg, mean, db)
    assert lib.nvn_device_status() == _lib.NVN_OK


# tensors of 32 MB and more take the kernels that hold a row batch in shared memory
@pytest.mark.parametrize("dtype,N,D", [("bf16", 8197, 4096), ("f16", 131, 262144), ("f32", 16401, 1024),
                                       ("bf16", 16389, 2048), ("f16", 4101, 8192), ("f32", 2053, 8192),
                                       ("bf16", 30000, 1152), ("f16", 262147, 128), ("f16", 20003, 1024),
                                       ("bf16", 40001, 512), ("f16", 80003, 256), ("bf16", 25001, 768),
                                       ("bf16", 4099, 5120), ("f32", 3001, 4096), ("f16", 3001, 6144),
                                       ("bf16", 1501, 12288), ("f32", 1101, 8000), ("bf16", 2001, 9000),
                                       ("f16", 1501, 16384), ("f32", 12001, 768), ("bf16", 7001, 2600)])
def test_large_tensors(lib, dtype, N, D):
    x, res, dy, ds, gamma, beta = data(N, D, dtype, N + D)
    y, s, inv = A.fused_rms_norm_residual_op(x, res, gamma, epsilon=1e-6)
    check_forward(x, res, gamma, 1e-6, y, s, inv)
    y, inv2 = A.fused_rms_norm_op(s, gamma, epsilon=1e-6)
    check_forward(s, None, gamma, 1e-6, y, None, inv2)
    dx, dg = A.fused_rms_norm_residual_grad_op(dy, ds, s, gamma, inv)
    check_grad(dy, ds, s, gamma, inv, dx, dg)
    dx, dg = A.fused_rms_norm_grad_op(dy, s, gamma, inv)
    check_grad(dy, None, s, gamma, inv, dx, dg)
    _, s, mean, iv = A.fused_layer_norm_residual_op(x, res, gamma, beta, epsilon=1e-6)
    dx, dg, db = A.fused_layer_norm_residual_grad_op(dy, ds, s, gamma, mean, iv)
    check_grad(dy, ds, s, gamma, iv, dx, dg, mean, db)
    assert lib.nvn_device_status() == _lib.NVN_OK


@pytest.mark.parametrize("dtype", DTYPES)
def test_buffers_of_every_alignment(lib, dtype):
    dt = T.TORCH_DTYPE[dtype]
    for D in (64, 1024, 4096, 24000):
        for off in (1, 2, 4):
            N = 11
            x, res, dy, ds, gamma, beta = data(N, D, dtype, D + off)

            def moved(t):
                base = torch.empty(t.numel() + off, dtype=t.dtype, device=DEV)
                v = base[off:].view(t.shape)
                v.copy_(t)
                return v
            y, s, inv = A.fused_rms_norm_residual_op(moved(x), moved(res), moved(gamma), epsilon=1e-5)
            check_forward(x, res, gamma, 1e-5, y, s, inv)
            dx, dg = A.fused_rms_norm_residual_grad_op(moved(dy), moved(ds), s, moved(gamma), inv)
            check_grad(dy, ds, s, gamma, inv, dx, dg)
            out = moved(x)
            A.fused_rms_norm_op(out, gamma, epsilon=1e-5, out=out)
            check_forward(x, None, gamma, 1e-5, out, None, inv=A.fused_rms_norm_op(x, gamma, epsilon=1e-5)[1])
            _, s, mean, iv = A.fused_layer_norm_residual_op(x, res, gamma, beta, epsilon=1e-5)
            dx, dg, db = A.fused_layer_norm_residual_grad_op(moved(dy), moved(ds), s, moved(gamma), mean, iv)
            check_grad(dy, ds, s, gamma, iv, dx, dg, mean, db)


def test_higher_ranks_and_strided_inputs(lib):
    x, res, dy, ds, gamma, _ = data(6 * 35, 96, "bf16", 2)
    x4, r4 = x.view(6, 35, 12, 8), res.view(6, 35, 12, 8)
    g2 = gamma.view(12, 8)
    y, s, inv = A.fused_rms_norm_residual_op(x4, r4, g2, axis=[2, 3], epsilon=1e-5)
    assert y.shape == x4.shape and inv.shape == (210,)
    check_forward(x, res, gamma, 1e-5, y.view(210, 96), s.view(210, 96), inv)
    dx, dg = A.fused_rms_norm_residual_grad_op(dy.view_as(x4), ds.view_as(x4), s, g2, inv, axis=[-2, -1])
    assert dg.shape == g2.shape
    check_grad(dy, ds, s.view(210, 96), gamma, inv, dx.view(210, 96), dg.view(-1))
    wide = torch.zeros(210, 200, dtype=torch.bfloat16, device=DEV)
    wide[:, 50:146] = x
    y2, inv2 = A.fused_rms_norm_op(wide[:, 50:146], gamma, epsilon=1e-5)
    check_forward(x, None, gamma, 1e-5, y2, None, inv2)


@pytest.mark.parametrize("D", [4096, 20001])
def test_in_place_forms(lib, D):
    x, res, dy, ds, gamma, beta = data(300, D, "bf16", 5)
    y, s, inv = A.fused_rms_norm_residual_op(x, res, gamma, epsilon=1e-5)
    x2, r2 = x.clone(), res.clone()
    # the stream in `residual` is updated, the norm lands in `x`
    A.fused_rms_norm_residual_op(x2, r2, gamma, epsilon=1e-5, out=x2, out_sum=r2)
    assert torch.equal(x2, y) and torch.equal(r2, s)
    x2, r2 = x.clone(), res.clone()
    A.fused_rms_norm_residual_op(x2, r2, gamma, epsilon=1e-5, out=r2, out_sum=x2)
    assert torch.equal(r2, y) and torch.equal(x2, s)
    dx, dg = A.fused_rms_norm_residual_grad_op(dy, ds, s, gamma, inv)
    d2, g2 = ds.clone(), torch.empty_like(gamma)
    a, b = A.fused_rms_norm_residual_grad_op(dy, d2, s, gamma, inv, out=d2, out_grads=g2)
    assert a is d2 and b is g2 and torch.equal(d2, dx) and torch.equal(g2, dg)
    _, s, mean, iv = A.fused_layer_norm_residual_op(x, res, gamma, beta)
    dx = A.fused_layer_norm_residual_grad_op(dy, ds, s, gamma, mean, iv)[0]
    d2 = ds.clone()
    A.fused_layer_norm_residual_grad_op(dy, d2, s, gamma, mean, iv, out=d2)
    assert torch.equal(d2, dx)


def test_values_at_the_edges(lib):
    D = 1024
    x, res, dy, ds, gamma, _ = data(64, D, "bf16", 9)
    x[3] = 0                       # a row of zeros: y = 0, 1/rms = 1/sqrt(eps)
    x[5] = float("inf")
    x[9, 17] = float("nan")
    x[11] = 1e18                   # squares stay finite in fp32
    x[12] = 1e-18                  # squares vanish beside eps
    y, inv = A.fused_rms_norm_op(x, gamma, epsilon=1e-6)
    fine = [i for i in range(64) if i not in (5, 9)]
    check_forward(x[fine], None, gamma, 1e-6, y[fine], None, inv[fine])
    assert torch.equal(y[3], torch.zeros_like(y[3])) and abs(float(inv[3]) - 1e3) < 1e-2
    assert torch.isnan(y[5]).all() and torch.isnan(y[9]).all()     # 0 * inf, and a NaN statistic
    dx, _ = A.fused_rms_norm_residual_grad_op(dy, ds, x, gamma, inv)
    check_grad(dy[fine], ds[fine], x[fine], gamma, inv[fine], dx[fine],
               A.fused_rms_norm_residual_grad_op(dy[fine], ds[fine], x[fine], gamma, inv[fine])[1])


def test_workspace_too_small_is_an_error(lib):
    x, _, dy, ds, gamma, _ = data(64, 1024, "f32", 1)
    inv = torch.ones(64, device=DEV)
    for D, fn, args in ((1024, lib.nvn_rms_bwd, (inv,)), (1024, lib.nvn_ln_bwd_residual, (inv, inv))):
        size = lib.nvn_rms_bwd_workspace_bytes if len(args) == 1 else lib.nvn_ln_bwd_residual_workspace_bytes
        need = size(0, 64, D)
        assert need >= D * 4
        ws = torch.empty(need, dtype=torch.uint8, device=DEV)
        outs = [torch.empty_like(gamma) for _ in args]
        call = [0, dy.data_ptr(), ds.data_ptr(), x.data_ptr(), gamma.data_ptr(), *[a.data_ptr() for a in args], 64,
                D, torch.empty_like(x).data_ptr(), *[o.data_ptr() for o in outs], ws.data_ptr()]
        stream = torch.cuda.current_stream().cuda_stream
        assert fn(*call, 512, stream) == _lib.NVN_ERR_WORKSPACE
        assert fn(*call, need, stream) == _lib.NVN_OK
    torch.cuda.synchronize()


def test_empty_problems(lib):
    g = torch.ones(8, device=DEV)
    for dt in (torch.float32, torch.bfloat16):
        e = torch.empty(0, 8, dtype=dt, device=DEV)
        y, inv = A.fused_rms_norm_op(e, g)
        assert y.shape == (0, 8) and inv.shape == (0,)
        y, s, inv = A.fused_rms_norm_residual_op(e, e, g)
        assert s.shape == (0, 8)
        dx, dg = A.fused_rms_norm_residual_grad_op(e, e, e, g, inv)
        assert dx.shape == (0, 8) and torch.equal(dg, torch.zeros_like(g))
        dx, dg, db = A.fused_layer_norm_residual_grad_op(e, e, e, g, inv, inv)
        assert torch.equal(dg, torch.zeros_like(g)) and torch.equal(db, torch.zeros_like(g))
        z = torch.empty(5, 0, dtype=dt, device=DEV)
        g0 = torch.ones(0, device=DEV)
        y, inv = A.fused_rms_norm_op(z, g0)
        dx, dg = A.fused_rms_norm_grad_op(z, z, g0, inv)
        assert y.shape == (5, 0) and dg.shape == (0,)


@pytest.mark.parametrize("N,D", [(5000, 1024), (700, 20001)])
def test_the_same_bits_every_run(lib, N, D):
    x, res, dy, ds, gamma, _ = data(N, D, "f32", 21)
    y, s, inv = A.fused_rms_norm_residual_op(x, res, gamma)
    first = A.fused_rms_norm_residual_grad_op(dy, ds, s, gamma, inv)
    for _ in range(3):
        again = A.fused_rms_norm_residual_grad_op(dy, ds, s, gamma, inv)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_streams_and_captured_graphs(lib):
    """Two graphs and eager calls of the same ops, replayed at once on streams of their own."""
    x, res, dy, ds, gamma, _ = data(2000, 1024, "bf16", 31)
    y0, s0, inv0 = A.fused_rms_norm_residual_op(x, res, gamma)
    dx0, dg0 = A.fused_rms_norm_residual_grad_op(dy, ds, s0, gamma, inv0)
    graphs, outs = [], []
    for _ in range(2):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y, s, inv = A.fused_rms_norm_residual_op(x, res, gamma)
            A.fused_rms_norm_residual_grad_op(dy, ds, s, gamma, inv)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y, s, inv = A.fused_rms_norm_residual_op(x, res, gamma)
            dx, dg = A.fused_rms_norm_residual_grad_op(dy, ds, s, gamma, inv)
        graphs.append(g)
        outs.append((y, s, dx, dg))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        dx, dg = A.fused_rms_norm_residual_grad_op(dy, ds, s0, gamma, inv0)
    torch.cuda.synchronize()
    assert torch.equal(dx, dx0) and torch.equal(dg, dg0)
    for y, s, dx, dg in outs:
        assert torch.equal(y, y0) and torch.equal(s, s0) and torch.equal(dx, dx0) and torch.equal(dg, dg0)


def test_differentiable_functions_and_layer(lib):
    """A pre-norm block: two residual norms in a row, against autograd of the formula in 64 bits."""
    x, res, dy, ds, gamma, beta = data(50, 256, "f32", 41)

    def leaves():
        return [t.clone().requires_grad_() for t in (x, res, gamma, beta)]
    a = leaves()
    y1, s1 = A.layer_norm_residual(a[0], a[1], a[2], a[3], epsilon=1e-5)
    y2, s2 = A.rms_norm_residual(y1, s1, a[2], epsilon=1e-5)
    y3 = A.rms_norm(s2, a[2], epsilon=1e-5)
    torch.autograd.backward([y2, y3], [dy, ds])
    b = [t.detach().double().requires_grad_() for t in (x, res, gamma, beta)]
    t1 = b[0] + b[1]
    n1 = torch.nn.functional.layer_norm(t1, (256,), b[2], b[3], 1e-5)
    t2 = n1 + t1

    def rms(t):
        return t / torch.sqrt((t * t).mean(1, keepdim=True) + 1e-5) * b[2]
    torch.autograd.backward([rms(t2), rms(t2)], [dy.double(), ds.double()])
    for p, q in zip(a, b):
        # three norms deep, every value below 10 and gradients of order one: 1e-5 of the largest
        scale = float(q.grad.abs().max())
        assert float((p.grad.double() - q.grad).abs().max()) <= 1e-5 * scale
    # only one of the two outputs is used
    a = leaves()
    A.rms_norm_residual(a[0], a[1], a[2])[1].sum().backward()
    assert torch.equal(a[0].grad, torch.ones_like(x)) and a[2].grad is None
    a = leaves()
    A.rms_norm_residual(a[0], a[1], a[2])[0].backward(dy)
    assert torch.equal(a[0].grad, a[1].grad) and a[2].grad is not None
    layer = A.RMSNormalization(epsilon=1e-5)
    y, s = layer(x, res)
    check_forward(x, res, layer.gamma.detach(), 1e-5, y.detach(), s.detach(), A.fused_rms_norm_op(s.detach(), layer.gamma.detach(), epsilon=1e-5)[1])
    layer(x).backward(dy)
    assert layer.gamma.grad is not None and layer.variables == [layer.gamma]


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_gradients_against_differences(lib, kind):
    """<gradient, v> against the central difference of the formula in 64 bits along v."""
    N, D, eps, h = 17, 320, 1e-5, 1e-4
    x, res, dy, ds, gamma, beta = data(N, D, "f32", 51)
    g = torch.Generator(device=DEV).manual_seed(3)
    vs = torch.randn(N, D, generator=g, device=DEV).double()
    vg = torch.randn(D, generator=g, device=DEV).double()
    s = x + res

    def loss(t, gam):
        c = t - t.mean(1, keepdim=True) if kind == "layer" else t
        y = c / torch.sqrt((c * c).mean(1, keepdim=True) + eps) * gam
        return (y * dy.double()).sum() + (t * ds.double()).sum()
    s64, g64 = s.double(), gamma.double()
    if kind == "rms":
        inv = A.fused_rms_norm_op(s, gamma, epsilon=eps)[1]
        dx, dg = A.fused_rms_norm_residual_grad_op(dy, ds, s, gamma, inv)
    else:
        _, mean, inv = A.fused_layer_norm_op(s, gamma, beta, epsilon=eps)
        dx, dg, _ = A.fused_layer_norm_residual_grad_op(dy, ds, s, gamma, mean, inv)
    along_x = (loss(s64 + h * vs, g64) - loss(s64 - h * vs, g64)) / (2 * h)
    along_g = (loss(s64, g64 + h * vg) - loss(s64, g64 - h * vg)) / (2 * h)
    # the difference is off by h^2 / 6 times a third derivative of order |v|^3; sums of 5440 fp32
    # values of order one are off by far less than 1e-5 of sum|terms|
    assert abs(float((dx.double() * vs).sum() - along_x)) <= 1e-5 * float((dx.double() * vs).abs().sum())
    assert abs(float((dg.double() * vg).sum() - along_g)) <= 1e-5 * float((dg.double() * vg).abs().sum())


@pytest.mark.parametrize("dtype,N,D", [("f32", 200003, 3), ("bf16", 100001, 17), ("f16", 3, 1000003), ("bf16", 2, 500008)])
def test_many_short_rows_and_few_long_ones(lib, dtype, N, D):
    x, res, dy, ds, gamma, beta = data(N, D, dtype, D)
    y, s, inv = A.fused_rms_norm_residual_op(x, res, gamma, epsilon=1e-5)
    check_forward(x, res, gamma, 1e-5, y, s, inv)
    dx, dg = A.fused_rms_norm_residual_grad_op(dy, ds, s, gamma, inv)
    check_grad(dy, ds, s, gamma, inv, dx, dg)
    _, s, mean, iv = A.fused_layer_norm_residual_op(x, res, gamma, beta, epsilon=1e-5)
    dx, dg, db = A.fused_layer_norm_residual_grad_op(dy, ds, s, gamma, mean, iv)
    check_grad(dy, ds, s, gamma, iv, dx, dg, mean, db)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_another_device_than_the_current_one(lib):
    x, res, dy, ds, gamma, _ = data(2000, 1024, "bf16", 4)
    y, s, inv = A.fused_rms_norm_residual_op(x, res, gamma)
    want = (y, s, inv, *A.fused_rms_norm_residual_grad_op(dy, ds, s, gamma, inv))
    x, res, dy, ds, gamma = (t.to("cuda:1") for t in (x, res, dy, ds, gamma))
    with torch.cuda.device(0):
        y, s, inv = A.fused_rms_norm_residual_op(x, res, gamma)
        got = (y, s, inv, *A.fused_rms_norm_residual_grad_op(dy, ds, s, gamma, inv))
    assert all(b.device.index == 1 and torch.equal(a, b.to(DEV)) for a, b in zip(want, got))
    with pytest.raises(ValueError, match="residual is on"):
        A.fused_rms_norm_residual_op(x, res.to(DEV), gamma)
