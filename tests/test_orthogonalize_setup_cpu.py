"""An optimiser step whose products cannot be set up leaves momentum and weight as they were: nothing is launched."""
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent

# Without any device the set-up of the products fails.  The addresses are never read: the kernels cannot start either.
CHILD = """
import ctypes as C, os
from cuop_b200 import _native as N, muon as M
import torch
assert not torch.cuda.is_available()
lib, A = N.lib(), 1 << 32
k = (C.c_double * 15)(*([3.4445, -4.7750, 2.0315] * 5))
size = lib.cuopx_orthogonalize_workspace_size(1, 40, 60)
if {muon}:
    rc = lib.cuopx_muon_step(M._MUON.pack(N.BF16, N.BF16, N.F32, 5, 1, 0, 1, 40, 60, 1e-7, C.addressof(k), 0.1, 0.9, 0.0, 1.0, 0,
                                          A, 60, 0, 2 * A, 60, 0, 3 * A, 60, 0, 4 * A, size), None)
else:
    rc = lib.cuopx_orthogonalize(M._ORTHO.pack(N.BF16, N.BF16, 5, 0, 1, 40, 60, 1e-7, C.addressof(k), A, 60, 0, 2 * A, 60, 0,
                                               4 * A, size), None)
print(rc, lib.cuopx_launch_count())
"""


@pytest.mark.parametrize("muon", [True, False])
def test_nothing_is_launched(muon):
    import os

    from cuop_b200 import _native as N

    env = dict(os.environ, CUDA_VISIBLE_DEVICES="")
    r = subprocess.run([sys.executable, "-c", CHILD.replace("{muon}", str(muon))], cwd=ROOT, env=env, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr
    assert r.stdout.split() == [str(N.CUDA_ERROR), "0"]
