"""The operators of a transformer block: host-side behaviour at the edges.  No GPU."""
import contextlib
import os
import subprocess

import pytest
import torch

import atex_b200 as A
from atex_b200 import _lib as L
from atex_b200 import rms_norm_ops as M

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ---------------------------------------------------------------------------
# sizes that follow from a device
# ---------------------------------------------------------------------------
def test_workspace_sizes_are_remembered_per_device(monkeypatch):
    """A device with more SMs needs more partial rows."""
    current, asked = [None], []

    @contextlib.contextmanager
    def device(index):
        current[0] = index
        yield

    class Library:
        @staticmethod
        def nvn_rms_bwd_workspace_bytes(code, n, d):
            asked.append(current[0])
            return 256 * (1 + current[0])

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(L, "load", lambda: Library)
    rows = M._Rows(0, 64, 128)
    for _ in range(2):
        assert rows.workspace_bytes("nvn_rms_bwd_workspace_bytes", 0) == 256
        assert rows.workspace_bytes("nvn_rms_bwd_workspace_bytes", 3) == 1024
    assert asked == [0, 3]


def test_residency_is_remembered_per_device(tmp_path):
    """The launchers' cache, compiled for the host."""
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    if not os.path.exists(os.path.join(cuda, "include", "cuda_runtime.h")):
        pytest.skip("needs the CUDA headers")
    src = tmp_path / "cache.cc"
    src.write_text("""
#include "nvn_host.h"
static nvn::ResidencyCache c;
int main() {
  if (c.get(0, 0) != 0 || c.get(1, 4096) != 0) return 1;
  c.put(0, 4096, 296);
  if (c.get(0, 4096) != 296 || c.get(1, 4096) != 0 || c.get(0, 0) != 0) return 2;
  c.put(1, 4096, 264);
  if (c.get(0, 4096) != 296 || c.get(1, 4096) != 264) return 3;
  c.put(0, 0, 148);
  if (c.get(0, 0) != 148 || c.get(0, 4096) != 0 || c.get(1, 4096) != 264) return 4;
  c.put(64, 4096, 7);
  c.put(-1, 4096, 7);
  return c.get(64, 4096) != 0 || c.get(-1, 4096) != 0 ? 5 : 0;
}
""")
    exe = str(tmp_path / "cache")
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "atex_b200", "csrc"), "-I", os.path.join(cuda, "include"),
                    str(src), "-o", exe], check=True, capture_output=True, text=True)
    assert subprocess.run([exe]).returncode == 0


# ---------------------------------------------------------------------------
# layers cast to half precision
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("cast", [lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.to(torch.bfloat16),
                                  lambda m: torch.nn.Sequential(m).half()[0]])
def test_a_cast_keeps_the_layers_parameters(cast):
    """The ops take float32 scales and offsets, also beside 16-bit activations; values, gradients and the
    parameter objects that an optimizer holds stay."""
    for layer, size in ((A.HeadNormRotary((4,), norm="layer"), 8), (A.RMSNormalization(), (2, 8))):
        layer.build(size)
        held = list(layer.parameters())
        with torch.no_grad():
            for i, p in enumerate(held):
                p.uniform_(0.3, 0.7)
                p.grad = torch.full_like(p, 1e-8 * (i + 1))   # below fp16's smallest
        was = [(p.detach().clone(), p.grad.clone()) for p in held]
        layer = cast(layer)
        now = list(layer.parameters())
        assert all(a is b for a, b in zip(held, now))
        for p, (v, g) in zip(now, was):
            assert p.dtype == torch.float32 and torch.equal(p, v) and torch.equal(p.grad, g)
    layer = A.HeadNormRotary((4,))
    layer.build(8)
    assert layer.to("meta").gamma_q.device.type == "meta"


# ---------------------------------------------------------------------------
# scratch of captured calls
# ---------------------------------------------------------------------------
def test_captured_calls_do_not_use_the_streams_scratch(monkeypatch):
    """The gradient behind layer_norm_residual, like every older op, has its partial rows there.  Two graphs
    captured on one stream may run at once, and the stream's scratch is replaced when it has to grow."""
    from atex_b200 import nv_norm_ops as O
    monkeypatch.setattr(O, "_workspaces", {})
    capturing = [False]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    device = torch.device("cpu")
    eager = O._workspace(device, 7, 4096)
    assert O._workspace(device, 7, 8192)[0] == eager[0]       # consecutive calls share it
    capturing[0] = True
    first, second = O._workspace(device, 7, 4096), O._workspace(device, 7, 4096)
    assert len({eager[0], first[0], second[0]}) == 3
    assert all(w[1] >= 4096 and w[2].data_ptr() == w[0] for w in (first, second))
    assert O._workspace(device, 7, 0)[:2] == (0, 0)
    capturing[0] = False
    assert O._workspace(device, 7, 4096)[0] == eager[0] and len(O._workspaces) == 1
