"""Per-head normalisation with rotary positions: refusals and host-side behaviour.  No GPU."""
import ctypes

import pytest
import torch

import atex_b200 as A
from atex_b200 import _lib as L
from atex_b200 import rotary_ops as R


def args(**kw):
    f, a = A.rotary_frequencies((2, 2))
    d = {"q": torch.zeros(2, 3, 4, 8), "k": torch.zeros(2, 3, 2, 8), "positions": torch.zeros(2, 2, 3, dtype=torch.int64),
         "inv_freq": f, "pair_axis": a, "scale_q": torch.ones(8), "scale_k": torch.ones(8)}
    d.update(kw)
    return d


@pytest.mark.parametrize("change,error,text", [
    ({"q": torch.zeros(3, 8)}, A.InvalidArgumentError, "q must be \\[batch, tokens, heads, head_dim\\]"),
    ({"q": None}, TypeError, "q must be a torch.Tensor"),
    ({"q": torch.zeros(2, 3, 4, 8).double()}, TypeError, "float32, float16 or bfloat16"),
    ({"q": torch.zeros(2, 3, 0, 8)}, A.InvalidArgumentError, "at least one head"),
    ({"k": torch.zeros(2, 4, 2, 8)}, A.InvalidArgumentError, "k must have q's batch, tokens and head_dim"),
    ({"k": torch.zeros(2, 3, 2, 8).half()}, TypeError, "same dtype"),
    ({"norm": "batch"}, A.InvalidArgumentError, "norm must be"),
    ({"scale_q": None}, A.InvalidArgumentError, "needs scale_q"),
    ({"scale_q": torch.ones(7)}, A.InvalidArgumentError, "scale_q must have the same number of elements as a head, got 7 and 8"),
    ({"scale_k": torch.ones(8).half()}, TypeError, "float32"),
    ({"offset_q": torch.ones(8)}, A.InvalidArgumentError, "offset_q does not belong to norm='rms'"),
    ({"norm": "none"}, A.InvalidArgumentError, "scale_q does not belong to norm='none'"),
    ({"norm": "layer"}, A.InvalidArgumentError, "needs offset_q"),
    ({"k": None}, A.InvalidArgumentError, "scale_k does not belong"),
    ({"positions": torch.zeros(2, 2, 3)}, TypeError, "int32 or int64"),
    ({"positions": torch.zeros(2, 2, 4, dtype=torch.int64)}, A.InvalidArgumentError, "positions must be"),
    ({"positions": torch.zeros(2, 3, 3, dtype=torch.int64)}, A.InvalidArgumentError, "positions must be"),
    ({"positions": torch.zeros(3, dtype=torch.int64)}, A.InvalidArgumentError, "positions must be"),
    ({"inv_freq": torch.ones(4)}, TypeError, "float64"),
    ({"pair_axis": torch.zeros(4, dtype=torch.int64)}, TypeError, "int32"),
    ({"pair_axis": torch.zeros(3, dtype=torch.int32)}, A.InvalidArgumentError, "of one length"),
    ({"inv_freq": torch.ones(5).double(), "pair_axis": torch.zeros(5, dtype=torch.int32)}, A.InvalidArgumentError,
     "has 5 pairs, a head has only 8 elements"),
    ({"positions": None}, A.InvalidArgumentError, "need positions"),
    ({}, RuntimeError, "no CPU implementation"),
])
def test_refusals(lib, change, error, text):
    with pytest.raises(error, match=text):
        A.fused_head_norm_rotary_op(**args(**change))
    if "offset" not in text:
        a = args(**change)
        q, k = a.pop("q"), a.pop("k")
        with pytest.raises(error, match=text):
            A.fused_head_norm_rotary_grad_op(q, k, q, k, **a)


def test_frequencies(lib):
    for bad in ((), (0, 0), (-1, 3)):
        with pytest.raises(ValueError, match="sections"):
            A.rotary_frequencies(bad)
    f, a = A.rotary_frequencies((0, 4, 0, 2))
    assert a.tolist() == [1, 1, 1, 1, 3, 3] and f.tolist()[0] == 1.0 and f.tolist()[4] == 1.0
    assert torch.equal(A.rotary_frequencies((6,))[0], A.rotary_frequencies((2, 4), shared=True)[0])


class Heads(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p)] + [(n, ctypes.c_int64) for n in ("heads", "sb", "st", "sh")]


class Problem(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_int32) for n in ("dtype", "norm", "interleaved")] + [("epsilon", ctypes.c_float)]
                + [(n, ctypes.c_int64) for n in ("batch", "tokens", "head_dim", "pairs")]
                + [(n, ctypes.c_int32) for n in ("axes", "position_bytes")] + [("positions", ctypes.c_void_p)]
                + [(n, ctypes.c_int64) for n in ("pa", "pb", "pt")]
                + [(n, ctypes.c_void_p) for n in ("inv_freq", "pair_axis")] + [("q", Heads), ("k", Heads)]
                + [(n, ctypes.c_void_p) for n in ("scale_q", "offset_q", "scale_k", "offset_k")])


def test_the_packed_problem_has_the_layout_of_the_header(lib):
    assert R._PROBLEM.size == ctypes.sizeof(Problem) and R._HEADS.size == ctypes.sizeof(Heads)
    raw = R._PROBLEM.pack(1, 2, 3, 0.5, *range(4, 8), 8, 9, *range(10, 14), 14, 15, *range(16, 21), *range(21, 26),
                          *range(26, 30))
    p = Problem.from_buffer_copy(raw)
    assert (p.dtype, p.norm, p.interleaved, p.epsilon, p.batch, p.pairs, p.axes, p.position_bytes) == (1, 2, 3, 0.5, 4, 7, 8, 9)
    assert (p.positions, p.pt, p.inv_freq, p.pair_axis, p.q.data, p.q.sh, p.k.data, p.k.sh) == (10, 13, 14, 15, 16, 20, 21, 25)
    assert (p.scale_q, p.offset_q, p.scale_k, p.offset_k) == (26, 27, 28, 29)


def test_abi_refuses_before_it_touches_cuda(lib):
    buf = (ctypes.c_float * 256)()
    p = ctypes.cast(buf, ctypes.c_void_p).value

    def problem(**kw):
        c = Problem(dtype=0, norm=1, batch=1, tokens=2, head_dim=8, pairs=2, axes=1, position_bytes=8, positions=p,
                    inv_freq=p, pair_axis=p, q=Heads(p, 2, 16, 16, 8), scale_q=p)
        for k, v in kw.items():
            setattr(c, k, v)
        return c

    def fwd(c, q=Heads(p, 2, 16, 16, 8), k=None):
        return lib.nvn_head_norm_rotary_fwd(ctypes.byref(c), ctypes.byref(q) if q else None,
                                            ctypes.byref(k) if k else None, None)
    bad = L.NVN_ERR_INVALID_ARGUMENT
    assert lib.nvn_head_norm_rotary_fwd(None, None, None, None) == bad
    for kw in ({"dtype": 5}, {"norm": 3}, {"norm": -1}, {"batch": -1}, {"head_dim": 0}, {"pairs": 5}, {"pairs": -1},
               {"axes": 0}, {"position_bytes": 2}, {"positions": None}, {"inv_freq": None}, {"pair_axis": None},
               {"scale_q": None}, {"norm": 2}, {"q": Heads(p, 0, 1, 1, 1)}, {"q": Heads(None, 2, 16, 16, 8)},
               {"k": Heads(p, 1, 16, 16, 8)}):
        assert fwd(problem(**kw)) == bad, kw
    assert fwd(problem(), q=None) == bad and fwd(problem(), q=Heads(p, 3, 16, 16, 8)) == bad
    assert fwd(problem(head_dim=520)) == L.NVN_ERR_LIMIT
    assert fwd(problem(batch=1 << 20, tokens=1 << 12)) == L.NVN_ERR_UNSUPPORTED
    assert fwd(problem(q=Heads(p, 70000, 16, 16, 8))) == L.NVN_ERR_UNSUPPORTED
    assert fwd(problem(batch=0)) == L.NVN_OK
    h = Heads(p, 2, 16, 16, 8)

    def bwd(c, dparams=p, ws=None):
        return lib.nvn_head_norm_rotary_bwd(ctypes.byref(c), ctypes.byref(h), None, ctypes.byref(h), None, dparams, ws,
                                            1 << 20, None)
    assert bwd(problem(), dparams=None) == bad
    assert bwd(problem()) == L.NVN_ERR_WORKSPACE
    assert bwd(problem(), ws=(p + 255) // 256 * 256 + 8) == L.NVN_ERR_WORKSPACE
    assert lib.nvn_head_norm_rotary_bwd_workspace_bytes(ctypes.byref(problem(norm=0, scale_q=None))) == 0


def test_layer_interface(lib):
    layer = A.HeadNormRotary((2, 2), norm="layer")
    layer.build(8)
    assert layer.gamma_q.shape == (8,) and layer.beta_k.shape == (8,) and len(list(layer.parameters())) == 4
    assert layer.get_config()["head_norm_rotary"]["sections"] == (2, 2)
    with pytest.raises(A.InvalidArgumentError, match="norm must be"):
        A.HeadNormRotary((2,), norm="x")
    assert layer.half()._rotary[0].dtype == torch.float64
