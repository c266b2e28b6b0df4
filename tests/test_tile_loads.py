"""The addresses of the tile products' loads (``csrc/kernels/tile_mul.h``), computed on the host by the header's own functions."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = next((c for c in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")) if c and os.path.exists(c)), None)


@pytest.mark.skipif(HIPCC is None, reason="hipcc not found")
def test_no_load_leaves_its_array(tmp_path):
    """Codes whose rows end inside a stage (K = 64, 257, 320, ..), one channel in the last tile, odd numbers of stages for two groups."""
    exe = str(tmp_path / "tile_loads")
    subprocess.run([HIPCC, "--cuda-host-only", "-O2", "-std=c++17", "-I", os.path.join(ROOT, "csrc", "kernels"),
                    os.path.join(ROOT, "tests", "tile_loads.hip"), "-o", exe], check=True, capture_output=True, text=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.startswith("ok"), out.stdout + out.stderr
