"""Listed experts' products with any n_expert: the launch is sized by it on the host,
where it must not wrap.  A process of its own that sees no GPU, so that a launch is
refused before it reads anything."""
import os
import subprocess
import sys

import pytest

from conftest import PKG

CALL = """
import sys
sys.path.insert(0, %r)
import q4mi
L, A = q4mi.lib(), 1 << 20
if %r == "f8":
    ok = L.q4mi_f8_mul_sel(A, A, 64, 128, 8192, 4, %d, A, A, q4mi.T_F8, 0, 1, A, %d, A, 0, 64)
else:
    ok = L.q4mi_mx4_mul_sel(A, A, 64, 128, 4096, 256, %d, A, A, q4mi.T_MXFP4, 0, 1, A, %d, A, 0, 64)
print(bool(ok), q4mi.last_error())
"""


@pytest.mark.parametrize("kind", ["f8", "mx4"])
@pytest.mark.parametrize("n", [64, 1000, 65535])
def test_no_wrap(kind, n):
    for ne in {2 ** 32 - n // 16, 2 ** 32 - n // 16 + 1, 2 ** 32 - 1, 2 ** 31}:
        env = dict(os.environ, HIP_VISIBLE_DEVICES="-1")
        r = subprocess.run([sys.executable, "-c", CALL % ((PKG, kind) + (ne, n) * 2)], env=env,
                           capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, (ne, r.returncode, r.stderr)
        assert r.stdout.startswith("False"), (ne, r.stdout)
