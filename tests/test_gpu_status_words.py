"""The words that expired waits are reported in, asked for the first time in the middle of a capture."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]

FIRST = """
import ctypes, sys
sys.path.insert(0, {root!r})
import torch
import __graft_entry__ as entry
pkg = entry.load_package()
x = torch.zeros(4, device="cuda")
torch.cuda.synchronize()
g, status = torch.cuda.CUDAGraph(), ctypes.c_int(-1)
with torch.cuda.graph(g):
    x += 1
    pkg.check(pkg.lib.{name}(ctypes.byref(status), 0))
    x += 2
assert status.value == 0
g.replay()
torch.cuda.synchronize()
assert (x == 3).all()
print("fine")
"""


@pytest.mark.parametrize("name", ["cmlb200_attention8_status", "cmlb200_attention_latent_status"])
def test_asked_for_first_while_a_stream_is_captured(name):
    r = subprocess.run([sys.executable, "-c", FIRST.format(root=str(ROOT), name=name)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]
