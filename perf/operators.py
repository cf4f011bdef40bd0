"""The transformer-block operators beside LayerNorm, as plain torch and as the framework's calls.

  rms_fwd      RMS normalisation, alone or behind the residual add:  s = T(x + r),
               y = s * scale / sqrt(mean(s^2) + eps); returns y, (s,) and the saved 1/rms.
  rms_grad     its gradient from the saved 1/rms; with a residual branch the gradient that
               arrives at s from there is added before the one rounding.
  ln_res_grad  the gradient of the residual LayerNorm, the residual branch's gradient included.
  rotary_fwd   attention queries and keys, normalised per head (root mean square, mean and
               variance, or not at all) and rotated by positions on one to four axes.
  rotary_grad  its gradient: of q and k, and of the per-head scales and offsets, which all
               heads and tokens share.

With `own` false `run` computes these from elementary torch operations in 32 bits (angles in
64: a position of a million times a frequency has no fraction left in 32), rounded once at
the end.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _rows(name, op, dtype, n, d, residual):
    return {"name": name, "op": op, "dtype": dtype, "n": n, "d": d, "residual": residual}


def _heads(name, op, dtype, batch, tokens, hq, hk, hd, sections, norm, interleaved, shared, layout, far):
    return {"name": name, "op": op, "dtype": dtype, "batch": batch, "tokens": tokens, "hq": hq, "hk": hk,
            "hd": hd, "sections": sections, "norm": norm, "interleaved": interleaved, "shared": shared,
            "layout": layout, "far": far}


def listed():
    return [
        # one decoding step of sixteen sequences: the block's residual add and norm, where latency counts
        _rows("rms_decode", "rms_fwd", "bf16", 16, 4096, True),
        # the same block over a training batch of 16 sequences of 2048 tokens
        _rows("rms_batch", "rms_fwd", "bf16", 32768, 4096, True),
        # a norm without a residual on a width that no vector access divides
        _rows("rms_odd", "rms_fwd", "f16", 12345, 1001, False),
        # backward of the training batch, the residual stream's gradient added on the way
        _rows("rms_grad_batch", "rms_grad", "bf16", 32768, 4096, True),
        # backward of a final norm in 32 bits
        _rows("rms_grad_f32", "rms_grad", "f32", 4096, 1024, False),
        # residual LayerNorm backward, many rows of an encoder's width
        _rows("ln_res_grad_batch", "ln_res_grad", "f16", 65536, 1024, True),
        # the same on a ragged batch of a wider model
        _rows("ln_res_grad_ragged", "ln_res_grad", "bf16", 4099, 5120, True),
        # queries and keys of one decoding step: one token for each of sixteen sequences, far into their contexts
        _heads("rotary_decode", "rotary_fwd", "bf16", 16, 1, 32, 8, 128, "16,24,24", "rms", False, True, "packed", 100000),
        # the training batch: q and k read where they lie in the packed projection
        _heads("rotary_batch", "rotary_fwd", "bf16", 16, 2048, 32, 8, 128, "16,24,24", "rms", False, True, "packed", 0),
        # a ragged video clip: time, height and width with frequencies of their own, head-major tensors
        _heads("rotary_video", "rotary_fwd", "f16", 2, 17550, 16, 16, 64, "8,12,12", "layer", True, False, "bhtd", 0),
        # backward of the training batch
        _heads("rotary_grad_batch", "rotary_grad", "bf16", 8, 2048, 32, 8, 128, "16,24,24", "rms", False, True, "packed", 0),
        # backward in 32 bits: heads of 80 of which 48 are rotated, few keys, an odd number of tokens
        _heads("rotary_grad_partial", "rotary_grad", "f32", 3, 1025, 10, 2, 80, "12,12", "layer", False, False, "bthd", 0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rms_fwd", "rms_grad", "ln_res_grad", "rotary_fwd", "rotary_grad"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    room = (1 << 27) * 2 // _BYTES[dtype]   # elements of one tensor of the largest listed case
    if not op.startswith("rotary"):
        d = _log(rng, 64, 16384)
        d = rng.choice([d, d // 8 * 8, d // 64 * 64, d // 256 * 256]) or 64
        n = _log(rng, 1, min(131072, max(1, room // d)))
        return {"op": op, "dtype": dtype, "n": n, "d": d,
                "residual": True if op == "ln_res_grad" else rng.random() < 0.6}
    hd = rng.choice([32, 40, 64, 64, 72, 80, 96, 112, 128, 128, 128, 160, 192, 256, rng.randrange(34, 256)])
    pairs = rng.choice([hd // 2, hd // 2, hd // 2, rng.randrange(4, hd // 2 + 1)])
    axes = min(rng.choice([1, 2, 3, 3, 4]), pairs)
    cuts = sorted(rng.sample(range(1, pairs), axes - 1)) if axes > 1 else []
    sections = ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [pairs]))
    hk = rng.choice([1, 2, 4, 8, 8, 16, rng.randrange(1, 17)])
    hq = hk * rng.choice([1, 1, 2, 4, 5, 8])
    most = (room * 5 // 4 if op == "rotary_fwd" else room * 5 // 8) // ((hq + hk) * hd)
    tokens = _log(rng, 1, max(1, min(131072, most)))
    batch = _log(rng, 1, max(1, min(64, most // tokens)))
    return {"op": op, "dtype": dtype, "batch": batch, "tokens": tokens, "hq": hq, "hk": hk, "hd": hd,
            "sections": sections, "norm": rng.choice(["rms", "rms", "layer", "none"]),
            "interleaved": rng.random() < 0.4, "shared": rng.random() < 0.5,
            "layout": rng.choice(["packed", "bthd", "bhtd"]), "far": rng.choice([0, 0, 5000, 1000000])}


def work(case):
    e = _BYTES[case["dtype"]]
    if not case["op"].startswith("rotary"):
        n, d, res = case["n"], case["d"], bool(case["residual"])
        if case["op"] == "rms_fwd":
            return {"bytes": n * d * e * (4 if res else 2) + 4 * d + 4 * n, "flops": n * d * (5 if res else 4)}
        if case["op"] == "rms_grad":
            return {"bytes": n * d * e * (4 if res else 3) + 8 * d + 4 * n, "flops": n * d * (9 if res else 8)}
        return {"bytes": n * d * e * 4 + 12 * d + 8 * n, "flops": n * d * 12}
    rows = case["batch"] * case["tokens"]
    cells = rows * (case["hq"] + case["hk"]) * case["hd"]
    axes = len(case["sections"].split(","))
    vectors = {"none": 0, "rms": 2, "layer": 4}[case["norm"]] * case["hd"] * 4
    if case["op"] == "rotary_fwd":
        return {"bytes": cells * e * 2 + rows * axes * 8 + vectors, "flops": cells * 8}
    return {"bytes": cells * e * 3 + rows * axes * 8 + 2 * vectors, "flops": cells * 16}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _frequencies(case):
    """Radians per position of every pair, in 64 bits, and the axis that turns it."""
    sizes = [int(s) for s in case["sections"].split(",")]
    pairs, base = sum(sizes), 10000.0
    axis = torch.cat([torch.full((s,), a, dtype=torch.int32) for a, s in enumerate(sizes)])
    if case["shared"]:      # one ladder over all pairs, cut into sections
        step = torch.arange(pairs, dtype=torch.float64) / pairs
    else:                   # a ladder for each axis
        step = torch.cat([torch.arange(s, dtype=torch.float64) / s for s in sizes])
    return base ** -step, axis


def _positions(case, g, dev):
    """[axes, batch, tokens]: the cells of a grid in row order, each sequence from a start of its own."""
    axes, t = len(case["sections"].split(",")), case["tokens"]
    side = max(1, int(round(t ** (1.0 / axes))))
    index, out = torch.arange(t, dtype=torch.int64, device=dev), []
    for a in range(axes - 1):
        out.append(index % side)
        index = index // side
    out.append(index)
    grid = torch.stack(out[::-1])[:, None, :].expand(axes, case["batch"], t)
    start = torch.randint(0, case["far"] + 1, (axes, case["batch"], 1), generator=g, device=dev)
    return (grid + start).contiguous()


def _laid_out(case, heads, g, dev, dtype):
    b, t, hd = case["batch"], case["tokens"], case["hd"]
    shape = (b, heads, t, hd) if case["layout"] == "bhtd" else (b, t, heads, hd)
    x = torch.randn(shape, generator=g, device=dev)
    x = (x * (0.5 + 2 * torch.rand(hd, generator=g, device=dev)) + 0.2).to(dtype)
    return x.transpose(1, 2) if case["layout"] == "bhtd" else x


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(1000003 * int(seed) + 17)
    dtype = _TYPES[case["dtype"]]
    st = {"case": case}
    if not case["op"].startswith("rotary"):
        n, d = case["n"], case["d"]
        # a residual stream: channels of unlike size, rows with a common offset
        x = torch.randn(n, d, generator=g, device=dev)
        x = x * (0.3 + 3 * torch.rand(d, generator=g, device=dev)) + torch.randn(n, 1, generator=g, device=dev)
        st["x"] = x.to(dtype)
        st["scale"] = 0.5 + torch.rand(d, generator=g, device=dev)
        st["eps"] = 1e-5
        if case["op"] == "rms_fwd":
            if case["residual"]:
                st["residual"] = (2 * torch.randn(n, d, generator=g, device=dev)).to(dtype)
            return st
        st["dy"] = torch.randn(n, d, generator=g, device=dev).to(dtype)
        if case["residual"]:
            st["dsum"] = torch.randn(n, d, generator=g, device=dev).to(dtype)
        # what the forward pass has saved
        xf = st["x"].float()
        if case["op"] == "rms_grad":
            st["inv"] = torch.rsqrt((xf * xf).mean(1) + st["eps"])
        else:
            st["mean"] = xf.mean(1)
            st["inv"] = torch.rsqrt(xf.var(1, unbiased=False) + st["eps"])
        return st
    hq, hk, hd = case["hq"], case["hk"], case["hd"]
    if case["layout"] == "packed":     # q, k and v side by side, as the projection leaves them
        qkv = _laid_out(case, hq + 2 * hk, g, dev, dtype)
        st["q"], st["k"] = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
    else:
        st["q"], st["k"] = _laid_out(case, hq, g, dev, dtype), _laid_out(case, hk, g, dev, dtype)
    freq, axis = _frequencies(case)
    st["inv_freq"], st["pair_axis"] = freq.to(dev), axis.to(dev)
    st["positions"] = _positions(case, g, dev)
    st["eps"] = 1e-6
    for name in ("q", "k"):
        st["scale_" + name] = None if case["norm"] == "none" else 0.5 + torch.rand(hd, generator=g, device=dev)
        st["offset_" + name] = 0.1 * torch.randn(hd, generator=g, device=dev) if case["norm"] == "layer" else None
    if case["op"] == "rotary_grad":
        for name, heads in (("q", hq), ("k", hk)):
            st["d" + name] = torch.randn(case["batch"], case["tokens"], heads, hd, generator=g, device=dev).to(dtype)
    return st


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _rms_fwd(st):
    x, out = st["x"], {}
    if "residual" in st:
        x = (x.float() + st["residual"].float()).to(x.dtype)
        out["s"] = x
    xf = x.float()
    inv = torch.rsqrt((xf * xf).mean(1) + st["eps"])
    out["y"] = (xf * inv[:, None] * st["scale"]).to(x.dtype)
    out["inv"] = inv
    return out


def _rms_grad(st):
    x, dy = st["x"].float(), st["dy"].float()
    xh = x * st["inv"][:, None]
    gy = dy * st["scale"]
    dx = (gy - xh * (gy * xh).mean(1, keepdim=True)) * st["inv"][:, None]
    if "dsum" in st:
        dx = dx + st["dsum"].float()
    return {"dx": dx.to(st["x"].dtype), "dscale": (dy * xh).sum(0)}


def _ln_res_grad(st):
    x, dy = st["x"].float(), st["dy"].float()
    xh = (x - st["mean"][:, None]) * st["inv"][:, None]
    gy = dy * st["scale"]
    dx = (gy - gy.mean(1, keepdim=True) - xh * (gy * xh).mean(1, keepdim=True)) * st["inv"][:, None]
    dx = dx + st["dsum"].float()
    return {"dx": dx.to(st["x"].dtype), "dscale": (dy * xh).sum(0), "doffset": dy.sum(0)}


def _angles(st):
    """cos and sin of [batch, tokens, 1, pairs], from angles in 64 bits."""
    turn = st["positions"][st["pair_axis"].long()].permute(1, 2, 0).double() * st["inv_freq"]
    return torch.cos(turn).float()[:, :, None], torch.sin(turn).float()[:, :, None]


def _turned(x, cos, sin, interleaved):
    pairs = cos.shape[-1]
    a, b = (x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]) if interleaved else (x[..., :pairs], x[..., pairs:2 * pairs])
    u, v = a * cos - b * sin, a * sin + b * cos
    y = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    return torch.cat((y, x[..., 2 * pairs:]), -1)


def _head_stats(x, norm, eps):
    if norm == "rms":
        inv = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
        return x * inv, inv
    c = x - x.mean(-1, keepdim=True)
    inv = torch.rsqrt((c * c).mean(-1, keepdim=True) + eps)
    return c * inv, inv


def _rotary_fwd(st):
    case, out = st["case"], {}
    cos, sin = _angles(st)
    for name in ("q", "k"):
        x = st[name].float()
        if case["norm"] != "none":
            x = _head_stats(x, case["norm"], st["eps"])[0] * st["scale_" + name]
        if case["norm"] == "layer":
            x = x + st["offset_" + name]
        out[name] = _turned(x, cos, sin, case["interleaved"]).to(st[name].dtype)
    return out


def _rotary_grad(st):
    case, out = st["case"], {}
    cos, sin = _angles(st)
    for name in ("q", "k"):
        g = _turned(st["d" + name].float(), cos, -sin, case["interleaved"])
        if case["norm"] != "none":
            xh, inv = _head_stats(st[name].float(), case["norm"], st["eps"])
            out["dscale_" + name] = (g * xh).sum((0, 1, 2))
            if case["norm"] == "layer":
                out["doffset_" + name] = g.sum((0, 1, 2))
            g = g * st["scale_" + name]
            mean = g.mean(-1, keepdim=True) if case["norm"] == "layer" else 0.0
            g = (g - mean - xh * (g * xh).mean(-1, keepdim=True)) * inv
        out["d" + name] = g.to(st[name].dtype)
    return out


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _own(st):
    import atex_b200 as A
    case = st["case"]
    op = case["op"]
    if op == "rms_fwd":
        if "residual" in st:
            y, s, inv = A.fused_rms_norm_residual_op(st["x"], st["residual"], st["scale"], epsilon=st["eps"])
            return {"y": y, "s": s, "inv": inv}
        y, inv = A.fused_rms_norm_op(st["x"], st["scale"], epsilon=st["eps"])
        return {"y": y, "inv": inv}
    if op == "rms_grad":
        if "dsum" in st:
            dx, dscale = A.fused_rms_norm_residual_grad_op(st["dy"], st["dsum"], st["x"], st["scale"], st["inv"])
        else:
            dx, dscale = A.fused_rms_norm_grad_op(st["dy"], st["x"], st["scale"], st["inv"])
        return {"dx": dx, "dscale": dscale}
    if op == "ln_res_grad":
        dx, dscale, doffset = A.fused_layer_norm_residual_grad_op(st["dy"], st["dsum"], st["x"], st["scale"],
                                                                  st["mean"], st["inv"])
        return {"dx": dx, "dscale": dscale, "doffset": doffset}
    form = {"norm": case["norm"], "interleaved": case["interleaved"], "epsilon": st["eps"]}
    if op == "rotary_fwd":
        q, k = A.fused_head_norm_rotary_op(st["q"], st["k"], st["positions"], st["inv_freq"], st["pair_axis"],
                                           scale_q=st["scale_q"], scale_k=st["scale_k"],
                                           offset_q=st["offset_q"], offset_k=st["offset_k"], **form)
        return {"q": q, "k": k}
    dq, dk, gq, gk, oq, ok = A.fused_head_norm_rotary_grad_op(
        st["dq"], st["dk"], st["q"], st["k"], st["positions"], st["inv_freq"], st["pair_axis"],
        scale_q=st["scale_q"], scale_k=st["scale_k"], **form)
    out = {"dq": dq, "dk": dk}
    if case["norm"] != "none":
        out["dscale_q"], out["dscale_k"] = gq, gk
    if case["norm"] == "layer":
        out["doffset_q"], out["doffset_k"] = oq, ok
    return out


def run(state):
    if own:
        return _own(state)
    return {"rms_fwd": _rms_fwd, "rms_grad": _rms_grad, "ln_res_grad": _ln_res_grad,
            "rotary_fwd": _rotary_fwd, "rotary_grad": _rotary_grad}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_rows(case, st):
    x = st["x"].double()
    w = st["scale"].double()
    d = case["d"]
    if case["op"] == "rms_fwd":
        out = {}
        if case["residual"]:
            # s is by definition the sum in the activations' type
            out["s"] = (x + st["residual"].double()).to(st["x"].dtype).double()
            x = out["s"]
        power = torch.einsum("nd,nd->n", x, x) / d
        out["inv"] = 1.0 / torch.sqrt(power + st["eps"])
        out["y"] = torch.einsum("nd,n,d->nd", x, out["inv"], w)
        return out
    # the gradient written out: y_j = w_j inv c_j with c = x (- mean), inv from the mean square of c
    dy, inv = st["dy"].double(), st["inv"].double()
    c = x if case["op"] == "rms_grad" else x - st["mean"].double()[:, None]
    along = torch.einsum("nd,nd,d->n", dy, c, w) * inv ** 3 / d
    dx = torch.einsum("nd,d,n->nd", dy, w, inv) - c * along[:, None]
    out = {"dscale": torch.einsum("nd,nd,n->d", dy, c, inv)}
    if case["op"] == "ln_res_grad":
        dx -= (torch.einsum("nd,d->n", dy, w) * inv / d)[:, None]
        out["doffset"] = dy.sum(0)
    if case["residual"]:
        dx += st["dsum"].double()
    out["dx"] = dx
    return out


def _exact_rotary(case, st):
    out = {}
    freq, axis, eps, hd = st["inv_freq"], st["pair_axis"], st["eps"], case["hd"]
    pairs = freq.numel()
    at = torch.arange(pairs, device=freq.device)
    first, second = (2 * at, 2 * at + 1) if case["interleaved"] else (at, at + pairs)
    turn = torch.stack([st["positions"][int(a)].double() * f for a, f in zip(axis.tolist(), freq.tolist())], -1)
    point = torch.polar(torch.ones_like(turn), turn)[:, :, None]          # exp(i angle)
    for name in ("q", "k"):
        x = st[name].double()
        c = x - x.mean(-1, keepdim=True) if case["norm"] == "layer" else x
        inv = 1.0 / torch.sqrt(c.square().mean(-1, keepdim=True) + eps)
        w = None if case["norm"] == "none" else st["scale_" + name].double()
        if case["op"] == "rotary_fwd":
            y = x if w is None else c * inv * w
            if case["norm"] == "layer":
                y = y + st["offset_" + name].double()
            y = y.clone()
            z = torch.complex(y[..., first], y[..., second]) * point
            y[..., first], y[..., second] = z.real, z.imag
            out[name] = y
            continue
        g = st["d" + name].double().clone()
        z = torch.complex(g[..., first], g[..., second]) * point.conj()
        g[..., first], g[..., second] = z.real, z.imag
        if w is not None:
            out["dscale_" + name] = torch.einsum("bthd,bthd->d", g, c * inv)
            if case["norm"] == "layer":
                out["doffset_" + name] = torch.einsum("bthd->d", g)
            g = g * w
            along = (g * c).sum(-1, keepdim=True) * inv ** 3 / hd
            lift = g.sum(-1, keepdim=True) * inv / hd if case["norm"] == "layer" else 0.0
            g = g * inv - c * along - lift
        out["d" + name] = g
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return _exact_rotary(case, st) if case["op"].startswith("rotary") else _exact_rows(case, st)
