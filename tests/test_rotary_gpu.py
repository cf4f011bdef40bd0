"""Per-head normalisation with rotary positions on the GPU, against its formula in 64 bits.

Tolerances follow from the arithmetic (u = 2^-24).  A cosine or sine: the fraction of a turn is
exact to 1e-9, its rounding to fp32 moves the angle by 2 u, the function is off by 2 ulp: 6 u.  A
lane adds 16 values and a tree of 5 follows: means are off by 22 u of the mean magnitude, 1/rms by
11 u + 4 u.  Forward: 15 + 10 + a few roundings, 40 u of |u| + |v| of the pair.  Gradient: the
rotation (10 u), the sums (22 u) and 1/rms up to three times (45 u): 96 u of the sum of the
magnitudes of all terms.  Parameter sums: 32 u a term and at most 64 + rows / 16 additions one
after the other.  Results in 16 bits are rounded once more, by eps / 2 of their value.
"""
import pytest
import torch

import atex_b200 as A
from atex_b200 import _lib
from atex_b200 import testing as T

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
EPS = 1e-6


def close(got, ref, bound, what):
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    small = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    allow = half * ref.abs() * (1 + 1e-3) + bound + small
    bad = ~((got.double() - ref).abs() <= allow)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst "
                           f"{float(((got.double() - ref).abs() / (allow + 1e-300)).max()):.3f} of the allowance")


def turn(x, cos, sin, interleaved):
    """Rotated x and, with |x|, |cos| + |sin| in place of the angles, the magnitudes."""
    pairs = cos.shape[-1]
    y = x.clone()
    i = torch.arange(pairs, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., a] * sin + x[..., b] * cos
    return y


def spread(x, pairs, interleaved):
    """|u| + |v| in the place of both members of a pair."""
    y = x.clone()
    i = torch.arange(pairs, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
    y[..., a] = y[..., b] = x[..., a] + x[..., b]
    return y


def angles(c):
    if c["positions"] is None:
        z = torch.zeros(1, 1, 1, 0, dtype=torch.float64, device=DEV)
        return z, z
    pos = c["positions"]
    pos = pos[:, None] if pos.dim() == 2 else pos
    ok = (c["axis"] >= 0) & (c["axis"] < pos.shape[0])
    ang = pos[torch.where(ok, c["axis"], 0).long()].permute(1, 2, 0).double() * torch.where(ok, c["freq"], 0.0)
    return torch.cos(ang)[:, :, None], torch.sin(ang)[:, :, None]


def stats(x, norm):
    """x-hat's numerator, 1/rms, and the magnitude that bounds the numerator's error."""
    if norm == "layer":
        c = x - x.mean(-1, keepdim=True)
        return c, 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + EPS), c.abs() + x.abs().mean(-1, keepdim=True)
    return x, 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS), x.abs()


def as4(t):
    return t if t.dim() == 4 else t[None]


def check(c, which, x, out, scale, offset):
    x = as4(x).double()
    cos, sin = angles(c)
    if c["norm"] == "none":
        n, m = x, x.abs()
    else:
        k, inv, mag = stats(x, c["norm"])
        g = scale.double()
        n, m = k * inv * g, mag * inv * g.abs()
        if offset is not None:
            n, m = n + offset.double(), m + offset.double().abs()
    close(as4(out), turn(n, cos, sin, c["interleaved"]), 40 * U * spread(m, cos.shape[-1], c["interleaved"]), which)


def check_grad(c, which, dy, x, scale, dx, dscale, doffset):
    x, dy = as4(x).double(), as4(dy).double()
    cos, sin = angles(c)
    dn = turn(dy, cos, -sin, c["interleaved"])
    mag = spread(dy.abs(), cos.shape[-1], c["interleaved"])
    if c["norm"] == "none":
        close(as4(dx), dn, 16 * U * mag, "d" + which)
        assert dscale is None and doffset is None
        return
    k, inv, km = stats(x, c["norm"])
    g = scale.double()
    xh, xm, gy, gm = k * inv, km * inv, dn * g, mag * g.abs()
    lift = gy.mean(-1, keepdim=True) if c["norm"] == "layer" else 0.0
    ref = inv * (gy - lift - xh * (gy * xh).mean(-1, keepdim=True))
    big = inv * (gm + gm.mean(-1, keepdim=True) + xm * (gm * xm).mean(-1, keepdim=True))
    close(as4(dx), ref, 96 * U * big, "d" + which)
    L = 32 + 64 + x.numel() / x.shape[-1] / 16
    close(dscale, (dn * xh).sum((0, 1, 2)), L * U * (mag * xm).sum((0, 1, 2)), "dscale_" + which)
    if c["norm"] == "layer":
        close(doffset, dn.sum((0, 1, 2)), L * U * mag.sum((0, 1, 2)), "doffset_" + which)
    else:
        assert doffset is None


def case(B, T_, hq, hk, hd, pairs, norm, interleaved, dtype, seed, axes=3, far=1000, layout="bthd", int32=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = T.TORCH_DTYPE[dtype]

    def r(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    def laid(h):
        if layout == "bhtd":
            return (r(B, h, T_, hd) * 2 + 0.3).to(dt).transpose(1, 2)
        return (r(B, T_, h, hd) * 2 + 0.3).to(dt)
    c = {"norm": norm, "interleaved": interleaved}
    if layout == "packed":
        qkv = (r(B, T_, hq + 2 * hk, hd) * 2 + 0.3).to(dt)
        c["q"], c["k"] = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
    else:
        c["q"], c["k"] = laid(hq), laid(hk)
    c["dq"], c["dk"] = r(B, T_, hq, hd).to(dt), r(B, T_, hk, hd).to(dt)
    c["positions"] = c["freq"] = c["axis"] = None
    if pairs:
        c["positions"] = torch.randint(-5, far, (axes, B, T_), generator=g, device=DEV,
                                       dtype=torch.int32 if int32 else torch.int64)
        c["freq"] = 10000.0 ** -(torch.arange(pairs, device=DEV, dtype=torch.float64) / pairs)
        c["axis"] = torch.randint(0, axes, (pairs,), generator=g, device=DEV, dtype=torch.int32)
    for s in "qk":
        c["scale_" + s] = None if norm == "none" else torch.rand(hd, generator=g, device=DEV) + 0.5
        c["offset_" + s] = r(hd) * 0.2 if norm == "layer" else None
    return c


def forward(c, **kw):
    return A.fused_head_norm_rotary_op(c["q"], c["k"], c["positions"], c["freq"], c["axis"], c["scale_q"],
                                       c["scale_k"], c["offset_q"], c["offset_k"], norm=c["norm"],
                                       interleaved=c["interleaved"], epsilon=EPS, **kw)


def backward(c, **kw):
    return A.fused_head_norm_rotary_grad_op(c["dq"], c["dk"], c["q"], c["k"], c["positions"], c["freq"], c["axis"],
                                            c["scale_q"], c["scale_k"], norm=c["norm"],
                                            interleaved=c["interleaved"], epsilon=EPS, **kw)


def check_both(c):
    q, k = forward(c)
    check(c, "q", c["q"], q, c["scale_q"], c["offset_q"])
    dq, dk, gq, gk, oq, ok = backward(c)
    check_grad(c, "q", c["dq"], c["q"], c["scale_q"], dq, gq, oq)
    if c["k"] is not None:
        check(c, "k", c["k"], k, c["scale_k"], c["offset_k"])
        check_grad(c, "k", c["dk"], c["k"], c["scale_k"], dk, gk, ok)
    else:
        assert k is None and dk is None and gk is None and ok is None


HEADS = [(1, 0), (2, 1), (3, 1), (7, 3), (16, 8), (32, 16), (33, 16), (64, 32), (72, 36), (80, 24), (96, 48),
         (100, 50), (128, 64), (128, 20), (128, 0), (160, 80), (192, 96), (256, 128), (320, 100), (510, 255),
         (511, 254), (512, 256)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", ["none", "rms", "layer"])
@pytest.mark.parametrize("hd,pairs", HEADS)
def test_head_sizes_norms_and_types(lib, hd, pairs, norm, interleaved):
    for i, dtype in enumerate(("f32", "f16", "bf16")):
        check_both(case(2, 19, 5, 2, hd, pairs, norm, interleaved, dtype, 100 * hd + pairs + i))


@pytest.mark.parametrize("layout", ["bthd", "bhtd", "packed"])
@pytest.mark.parametrize("B,T_,hq,hk", [(1, 1, 1, 1), (1, 1, 32, 8), (16, 1, 32, 8), (3, 1025, 10, 2), (1, 4099, 1, 1),
                                        (64, 33, 4, 4), (5, 7, 129, 3), (2, 2500, 16, 16)])
def test_batches_tokens_heads_and_layouts(lib, layout, B, T_, hq, hk):
    for dtype, hd, il in (("bf16", 128, False), ("f16", 64, True), ("f32", 80, False)):
        for norm in ("rms", "layer"):
            check_both(case(B, T_, hq, hk, hd, hd // 2, norm, il, dtype, B + T_ + hq, layout=layout))


@pytest.mark.parametrize("norm", ["none", "rms", "layer"])
@pytest.mark.parametrize("hd,pairs", [(48, 24), (64, 32), (64, 8), (80, 40), (96, 48), (112, 56), (128, 64), (128, 16),
                                      (160, 80), (192, 96), (192, 40), (240, 120), (256, 128), (256, 64)])
def test_two_heads_at_once(lib, hd, pairs, norm):
    """Even numbers of heads and enough rows: the kernels that take neighbouring heads together, with
    lanes to spare (sizes between the powers of two) and rotated ranges that end inside the head."""
    for dtype, il in (("bf16", False), ("f16", True)):
        check_both(case(2, 1301, 8, 4, hd, pairs, norm, il, dtype, hd + pairs, layout="packed"))
    check_both(case(1, 2603, 8, 4, hd, pairs, norm, True, "f32", hd + pairs))


@pytest.mark.parametrize("axes,far,int32", [(1, 4, True), (2, 2 ** 31 - 1, True), (4, 10 ** 6, False), (1, 2 ** 40, False)])
def test_positions(lib, axes, far, int32):
    """Far positions keep their angles: 2^40 times a frequency is still known to 1e-4 of a turn in 64
    bits, and the reference rounds the same product, so both see the same fraction to 2^-53 * 2^40."""
    c = case(2, 50, 3, 2, 64, 32, "none", False, "f32", axes, axes=axes, far=far, int32=int32)
    slack = 2.0 ** -50 * far     # of an angle, from the products' rounding in 64 bits
    for x, y in zip((c["q"], c["k"]), forward(c)):
        cos, sin = angles(c)
        ref = turn(x.double(), cos, sin, False)
        close(y, ref, (40 * U + slack) * spread(x.double().abs(), 32, False), "rotated")


def test_position_forms(lib):
    c = case(3, 40, 4, 2, 64, 32, "rms", False, "bf16", 3)
    shared = c["positions"][:, 0].contiguous()
    c["positions"] = shared[:, None].expand(3, 3, 40)
    want = forward(c)
    c["positions"] = shared
    assert all(torch.equal(a, b) for a, b in zip(want, forward(c)))
    c["positions"] = shared[:, None].expand(3, 3, 40).permute(2, 1, 0).contiguous().permute(2, 1, 0)   # other strides
    assert all(torch.equal(a, b) for a, b in zip(want, forward(c)))
    check_both(c)
    # pairs of an axis that is not there are left as they are
    c["axis"][::3] = -1
    c["axis"][1::5] = 7
    check_both(c)
    # three dimensions: a batch of one
    d = {k: (v[0] if k in ("q", "k", "dq", "dk") else v) for k, v in c.items()}
    d["positions"] = shared
    check_both(d)
    # queries alone
    e = dict(c, k=None, dk=None, scale_k=None)
    check_both(e)


def test_frequencies_of_sections(lib):
    f, a = A.rotary_frequencies((3, 5), base=100.0, device=DEV)
    assert f.dtype == torch.float64 and a.tolist() == [0] * 3 + [1] * 5
    assert torch.allclose(f.cpu(), torch.tensor([100.0 ** (-i / 3) for i in range(3)] + [100.0 ** (-i / 5) for i in range(5)],
                                                dtype=torch.float64), rtol=1e-15)
    f, _ = A.rotary_frequencies((3, 5), base=100.0, shared=True)
    assert torch.allclose(f, torch.tensor([100.0 ** (-i / 8) for i in range(8)], dtype=torch.float64), rtol=1e-15)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_alignments(lib, dtype):
    """Views whose strides or addresses rule out wide accesses, and outputs of any layout."""
    dt = T.TORCH_DTYPE[dtype]
    for extra, off in ((0, 1), (1, 0), (2, 2), (4, 4), (8, 0)):
        c = case(2, 21, 3, 2, 64, 32, "layer", False, dtype, extra + off)
        for s, h in (("q", 3), ("k", 2)):
            for name in (s, "d" + s):
                base = torch.zeros(2 * 21 * h * (64 + extra) + off, dtype=dt, device=DEV)
                v = base[off:].view(2, 21, h, 64 + extra)[..., :64]
                v.copy_(c[name])
                c[name] = v
        check_both(c)
        # into the slices of one packed tensor, whose other elements stay as they are
        packed = torch.full((2, 21, 9, 64 + extra), 7.0, dtype=dt, device=DEV)
        out = (packed[:, :, 1:4, :64], packed[:, :, 5:7, :64])
        want = forward(c)
        got = forward(c, out=out)
        assert got[0] is out[0] and all(torch.equal(a, b) for a, b in zip(want, got))
        want = backward(c)
        backward(c, out=out)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        rest = torch.ones(9, 64 + extra, dtype=torch.bool, device=DEV)
        rest[1:4, :64] = rest[5:7, :64] = False
        assert (packed[:, :, rest] == 7).all()
    # a last dimension that is not contiguous is copied
    c = case(2, 21, 3, 2, 64, 32, "rms", False, dtype, 77)
    c["q"] = c["q"].transpose(2, 3).contiguous().transpose(2, 3)
    check_both(c)


def test_in_place(lib):
    c = case(2, 300, 8, 2, 128, 64, "rms", False, "bf16", 8, layout="packed")
    q, k = forward(c)
    dq, dk = backward(c)[:2]
    kept = c["q"].clone(), c["k"].clone()
    forward(c, out=(c["q"], c["k"]))
    assert torch.equal(c["q"], q) and torch.equal(c["k"], k)
    c["q"].copy_(kept[0])
    c["k"].copy_(kept[1])
    backward(c, out=(c["dq"], c["dk"]))
    assert torch.equal(c["dq"], dq) and torch.equal(c["dk"], dk)


def test_values_at_the_edges(lib):
    c = case(1, 8, 4, 2, 128, 32, "rms", False, "bf16", 9)
    c["q"][0, 0, 0] = 0
    c["q"][0, 1, 1, 5] = float("inf")
    c["q"][0, 2, 2, 5] = float("nan")
    c["q"][0, 3, 3] = 1e18
    q, _ = forward(c)
    fine = torch.ones(1, 8, 4, dtype=torch.bool, device=DEV)
    fine[0, 1, 1] = fine[0, 2, 2] = False
    assert (q[0, 0, 0] == 0).all() and torch.isfinite(q[fine]).all()
    assert not torch.isfinite(q[0, 1, 1]).all() and torch.isnan(q[0, 2, 2]).all()
    dq = backward(c)[0]
    assert torch.isfinite(dq[fine]).all()
    # without a norm an infinity spoils its own pair alone, and none behind the rotated elements
    for il in (False, True):
        c = case(1, 8, 4, 2, 128, 32, "none", il, "bf16", 9)
        c["q"][0, 1, 1, 100] = float("inf")
        q, _ = forward(c)
        assert torch.isinf(q[0, 1, 1, 100]) and int(torch.isfinite(q).logical_not().sum()) == 1
    # nor where the rotated elements end inside a vector
    for hd, pairs, at in ((72, 11, 22), (72, 11, 23), (64, 5, 10), (100, 3, 7)):
        c = case(1, 8, 4, 2, hd, pairs, "none", True, "bf16", 9)
        c["q"][0, 1, 1, at] = float("inf")
        q, _ = forward(c)
        assert torch.isinf(q[0, 1, 1, at]) and int(torch.isfinite(q).logical_not().sum()) == 1
    # a gradient's infinity reaches its own head's row and columns, and nothing of a step's empty rows
    c = case(1, 3, 3, 1, 128, 64, "layer", False, "bf16", 11)
    c["dq"][0, 0, 0, 0] = float("inf")
    dq, dk, gq, gk, oq, ok = backward(c)
    assert torch.isfinite(dq[0, 1:]).all() and torch.isfinite(dq[0, 0, 1:]).all() and torch.isfinite(dk).all()
    assert all(torch.isfinite(t).all() for t in (gk, ok, gq[1:64], gq[65:], oq[1:64], oq[65:]))
    # every token's row of zeros without epsilon: nothing from it reaches the parameter sums of the others
    c = case(1, 9, 1, 1, 96, 48, "rms", False, "f32", 10)
    check_both(c)


def test_offsets_beyond_32_bits(lib):
    """The second sequence of a batch whose stride passes 2^31 elements."""
    T_, h, hd = 5, 2, 64
    base = torch.empty(2 ** 31 + 4096, dtype=torch.bfloat16, device=DEV)
    c = case(2, T_, h, h, hd, 32, "rms", False, "bf16", 12)
    far = torch.as_strided(base, (2, T_, h, hd), (2 ** 31 + 64, h * hd, hd, 1))
    want, grads = forward(c), backward(c)
    far.copy_(c["q"])
    c["q"] = far
    assert all(torch.equal(a, b) for a, b in zip(want, forward(c)))
    assert all(b is None or torch.equal(a, b) for a, b in zip(grads, backward(c)))
    out = (far, torch.empty_like(c["k"]))
    c["q"] = c["q"].contiguous()
    forward(c, out=out)
    assert torch.equal(far, want[0])


def test_workspace_too_small_is_an_error_and_not_a_write(lib):
    from atex_b200 import rotary_ops as R
    c = case(2, 300, 4, 2, 64, 32, "layer", False, "bf16", 1)
    form, packed, q, k, alive = R._problem(c["q"], c["k"], c["positions"], c["freq"], c["axis"],
                                           (c["scale_q"], c["scale_k"]), (None, None), "layer", False, EPS, False)
    need = lib.nvn_head_norm_rotary_bwd_workspace_bytes(packed)
    assert need == form.workspace_bytes(0) and need >= 4 * 64 * 4
    ws = torch.full((need // 4,), 7.0, device=DEV)
    out = torch.full((2, 2, 64), 7.0, device=DEV)
    dq, dk = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    args = (packed, R._pack(c["dq"]), R._pack(c["dk"]), R._pack(dq), R._pack(dk), out.data_ptr(), ws.data_ptr())
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.nvn_head_norm_rotary_bwd(*args, 256, stream) == _lib.NVN_ERR_WORKSPACE
    torch.cuda.synchronize()
    assert all((t == 7).all() for t in (ws, out, dq, dk))
    assert lib.nvn_head_norm_rotary_bwd(*args, need, stream) == _lib.NVN_OK
    want = backward(c)
    assert torch.equal(dq, want[0]) and torch.equal(dk, want[1]) and torch.equal(out[0, 0], want[2])


def test_empty_batches(lib):
    for B, T_ in ((0, 5), (3, 0)):
        c = case(B, T_, 4, 2, 64, 32, "layer", False, "bf16", 1)
        q, k = forward(c)
        assert q.shape == (B, T_, 4, 64) and k.shape == (B, T_, 2, 64)
        dq, dk, *sums = backward(c)
        assert dq.shape == q.shape and all(torch.equal(s, torch.zeros(64, device=DEV)) for s in sums)


def test_the_same_bits_every_run(lib):
    c = case(4, 3000, 8, 8, 128, 64, "layer", False, "bf16", 2)
    first = backward(c)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, backward(c)))


def test_streams_and_captured_graphs(lib):
    c = case(2, 1500, 8, 2, 128, 64, "rms", False, "bf16", 4)
    want = (*forward(c), *backward(c)[:4])
    graphs, outs = [], []
    for _ in range(2):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            forward(c)
            backward(c)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append((*forward(c), *backward(c)[:4]))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = (*forward(c), *backward(c)[:4])
    torch.cuda.synchronize()
    for got in (*outs, eager):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("norm", ["rms", "layer", "none"])
def test_differentiable_function_and_layer(lib, norm):
    """Through autograd from a packed projection, against autograd of the formula in 64 bits."""
    B, T_, hq, hk, hd = 2, 9, 4, 2, 32
    c = case(B, T_, hq, hk, hd, 16, norm, True, "f32", 6)
    g = torch.Generator(device=DEV).manual_seed(1)
    qkv = torch.randn(B, T_, hq + 2 * hk, hd, generator=g, device=DEV, requires_grad=True)
    params = [c[n] for n in ("scale_q", "scale_k", "offset_q", "offset_k")]
    leaves = [None if p is None else p.clone().requires_grad_() for p in params]
    q, k = A.head_norm_rotary(qkv[:, :, :hq], qkv[:, :, hq:hq + hk], c["positions"], c["freq"], c["axis"], *leaves,
                              norm=norm, interleaved=True, epsilon=EPS)
    torch.autograd.backward([q, k], [c["dq"], c["dk"]])
    ref = qkv.detach().double().requires_grad_()
    wide = [None if p is None else p.double().requires_grad_() for p in params]
    cos, sin = angles(c)

    def form(x, scale, offset):
        if norm != "none":
            m, inv, _ = stats(x, norm)
            x = m * inv * scale
        if offset is not None:
            x = x + offset
        return turn(x, cos, sin, True)
    torch.autograd.backward([form(ref[:, :, :hq], wide[0], wide[2]), form(ref[:, :, hq:hq + hk], wide[1], wide[3])],
                            [c["dq"].double(), c["dk"].double()])
    # values of order one: 96 u of a handful of terms stays below 1e-4
    assert float((qkv.grad.double() - ref.grad).abs().max()) <= 1e-4 * float(ref.grad.abs().max())
    assert (qkv.grad[:, :, hq + hk:] == 0).all()
    for a, b in zip(leaves, wide):
        if a is not None:
            assert float((a.grad.double() - b.grad).abs().max()) <= 1e-4 * float(b.grad.abs().max())
    layer = A.HeadNormRotary((4, 6, 6), norm=norm, epsilon=EPS)
    q, k = layer(c["q"], c["k"], c["positions"])
    f, ax = A.rotary_frequencies((4, 6, 6), device=DEV)
    one, zero = torch.ones(hd, device=DEV), torch.zeros(hd, device=DEV)
    pick = {"none": (None,) * 4, "rms": (one, one, None, None), "layer": (one, one, zero, zero)}[norm]
    want = A.fused_head_norm_rotary_op(c["q"], c["k"], c["positions"], f, ax, *pick, norm=norm, epsilon=EPS)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert len(list(layer.parameters())) == {"none": 0, "rms": 2, "layer": 4}[norm]
    assert layer(c["q"], None, c["positions"])[1] is None


@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_gradients_against_differences(lib, norm):
    c = case(1, 13, 3, 2, 64, 24, norm, False, "f32", 14)
    dq, dk, gq, gk, oq, ok = backward(c)
    cos, sin = angles(c)
    g = torch.Generator(device=DEV).manual_seed(5)
    h = 1e-5

    def loss(x, scale, offset, dy):
        m, inv, _ = stats(x, norm)
        n = m * inv * scale
        return (turn(n + offset if offset is not None else n, cos, sin, False) * dy).sum()
    for x, s, o, dy, dx, gs, go in ((c["q"], c["scale_q"], c["offset_q"], c["dq"], dq, gq, oq),
                                    (c["k"], c["scale_k"], c["offset_k"], c["dk"], dk, gk, ok)):
        x, s, dy = x.double(), s.double(), dy.double()
        o = None if o is None else o.double()
        for at, grad in ((0, dx), (1, gs), (2, go)):
            if grad is None:
                continue
            v = torch.randn(grad.shape, generator=g, device=DEV).double()
            up, down = [x, s, o], [x, s, o]
            up[at], down[at] = up[at] + h * v, down[at] - h * v
            diff = (loss(*up, dy) - loss(*down, dy)) / (2 * h)
            terms = grad.double() * v
            # h^2 times a third derivative, and fp32 sums of a few thousand terms: far below 1e-5 of sum|terms|
            assert abs(float(terms.sum() - diff)) <= 1e-5 * float(terms.abs().sum())


def test_a_captured_training_step(lib):
    """Forward and backward through autograd in one captured graph, replayed on new values."""
    B, T_, hq, hk, hd = 2, 40, 4, 2, 64
    c = case(B, T_, hq, hk, hd, 32, "rms", False, "bf16", 61)
    x = torch.randn(B, T_, (hq + 2 * hk) * hd, device=DEV).bfloat16()
    up = torch.randn(B, T_, hq, hd, device=DEV).bfloat16()

    def step(leaf, sq, sk):
        qkv = leaf.view(B, T_, hq + 2 * hk, hd)
        q, k = A.head_norm_rotary(qkv[:, :, :hq], qkv[:, :, hq:hq + hk], c["positions"], c["freq"], c["axis"], sq, sk,
                                  epsilon=EPS)
        torch.autograd.backward([q, k], [up, up[:, :, :hk]])

    def leaves():
        return x.clone().requires_grad_(), c["scale_q"].clone().requires_grad_(), c["scale_k"].clone().requires_grad_()
    static = leaves()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(*static)
    torch.cuda.current_stream().wait_stream(side)
    for t in static:
        t.grad = None
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(*static)
    x = torch.randn_like(x)
    with torch.no_grad():
        static[0].copy_(x)
    g.replay()
    torch.cuda.synchronize()
    eager = leaves()
    step(*eager)
    for a, b in zip(static, eager):
        assert torch.equal(a.grad, b.grad)


def test_refusals_that_need_a_device(lib):
    c = case(2, 6, 4, 2, 64, 32, "rms", False, "bf16", 1)
    with pytest.raises(RuntimeError, match="exceeds a built-in capacity"):
        x = torch.zeros(1, 2, 1, 520, device=DEV)
        A.fused_head_norm_rotary_op(x, None, None, norm="none")
    with pytest.raises(ValueError, match="heads apart"):
        forward(c, out=(c["q"][:, :1].expand(2, 6, 4, 64), c["k"]))
    with pytest.raises(ValueError, match="shape, dtype and device"):
        forward(c, out=(c["q"].float(), c["k"]))
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        A.fused_head_norm_rotary_op(c["q"], c["k"], c["positions"].cpu(), c["freq"], c["axis"], c["scale_q"],
                                    c["scale_k"])
    with pytest.raises(A.InvalidArgumentError, match="q_backprop must have the shape"):
        backward(dict(c, dq=c["dq"][:, :3]))
    with pytest.raises(A.InvalidArgumentError, match="k_backprop belongs to k"):
        backward(dict(c, dk=None))


def test_a_block_forward_and_backward(lib):
    """The operators in a run as a transformer block uses them: residual norm, projection, per-head
    norm and rotation, and all the way back, against autograd of the formulas in 64 bits."""
    B, T_, hq, hk, hd, D = 2, 24, 4, 2, 32, 128
    g = torch.Generator(device=DEV).manual_seed(9)

    def r(*s):
        return torch.randn(*s, generator=g, device=DEV)
    x, res, W = r(B * T_, D), r(B * T_, D), r(D, (hq + 2 * hk) * hd) / D ** 0.5
    gam, gq, gk = torch.rand(D, generator=g, device=DEV) + 0.5, torch.rand(hd, generator=g, device=DEV) + 0.5, \
        torch.rand(hd, generator=g, device=DEV) + 0.5
    f, ax = A.rotary_frequencies((4, 6, 6), device=DEV)
    pos = torch.randint(0, 500, (3, B, T_), generator=g, device=DEV)
    up = [r(B, T_, hq, hd), r(B, T_, hk, hd), r(B * T_, D)]
    a = [t.clone().requires_grad_() for t in (x, res, gam, gq, gk, W)]
    y, s = A.rms_norm_residual(a[0], a[1], a[2], epsilon=EPS)
    # a product that keeps fp32 whatever the library's default: sums of exact 64-bit products
    qkv = (y.double() @ a[5].double()).float().view(B, T_, hq + 2 * hk, hd)
    q, k = A.head_norm_rotary(qkv[:, :, :hq], qkv[:, :, hq:hq + hk], pos, f, ax, a[3], a[4], epsilon=EPS)
    torch.autograd.backward([q, k, s], up)
    b = [t.double().requires_grad_() for t in (x, res, gam, gq, gk, W)]
    t = b[0] + b[1]
    n = t / torch.sqrt((t * t).mean(1, keepdim=True) + EPS) * b[2]
    z = (n @ b[5]).view(B, T_, hq + 2 * hk, hd)
    cos, sin = angles({"positions": pos, "freq": f, "axis": ax})

    def head(v, w):
        return turn(v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * w, cos, sin, False)
    torch.autograd.backward([head(z[:, :, :hq], b[3]), head(z[:, :, hq:hq + hk], b[4]), t],
                            [u.double() for u in up])
    for p, w in zip(a, b):
        # a few hundred roundings of 2^-24 along the way, sums of at most 192 terms
        assert float((p.grad.double() - w.grad).abs().max()) <= 1e-4 * float(w.grad.abs().max())
    assert lib.nvn_device_status() == _lib.NVN_OK


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_another_device_than_the_current_one(lib):
    c = case(2, 300, 8, 2, 128, 64, "layer", False, "bf16", 4)
    want = (*forward(c), *backward(c))
    other = {k: v.to("cuda:1") if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    with torch.cuda.device(0):
        got = (*forward(other), *backward(other))
    assert all(b.device.index == 1 and torch.equal(a, b.to(DEV)) for a, b in zip(want, got))
    with pytest.raises(ValueError, match="positions is on"):
        forward(dict(other, positions=c["positions"]))
