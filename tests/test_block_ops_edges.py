"""Block operators (ops.py) at the edges of what their documentation allows.  Formulas, cases and tolerances: test_block_ops.py."""
import ctypes as C
import subprocess
import sys
from pathlib import Path

from conftest import PKG
from test_block_ops import native

REPO = Path(__file__).resolve().parent.parent

EMPTY_WORKSPACES = """
import ctypes as C, importlib
n = importlib.import_module("%s._native")
lib, P = n.load(), 0x1000
for size in (dict(batch=1, seq=0), dict(batch=0, seq=1), dict(batch=0, seq=0)):
    for more in (dict(), dict(d_scale=P, scale_stride=8), dict(d_scale=P), dict(d_y=P, d_gate=P, gate_stride=8, d_shift=P)):
        d = n.GatedNormDesc(**size, dim=8, post=0, pre=2, residual_scale=1.0, eps=1e-5, d_x=P, d_weight=P, **more)
        for g in (n.GatedNormGrads(d_gx=P), n.GatedNormGrads(d_gx=P, d_gweight=P), n.GatedNormGrads(d_gscale=P if "d_scale" in more else 0)):
            print(lib.cmdi_gated_norm_vjp_workspace(C.byref(d), C.byref(g)), flush=True)
""" % PKG


def test_gated_norm_workspace_without_rows():
    """No rows need no workspace (in a process of its own: a division by zero would end it)."""
    run = subprocess.run([sys.executable, "-c", EMPTY_WORKSPACES], cwd=REPO, capture_output=True, text=True, timeout=100)
    assert run.returncode == 0 and run.stdout.split() == ["0"] * 36, (run.returncode, run.stdout, run.stderr)
    n = native()
    d = n.GatedNormDesc(batch=0, seq=1, dim=0, post=0, pre=2, residual_scale=1.0, eps=1e-5)
    assert n.load().cmdi_gated_norm_vjp_workspace(C.byref(d), C.byref(n.GatedNormGrads())) == -1      # the other checks come first
