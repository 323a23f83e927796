"""GPU: the CUDA error of a refused call is reported by that call and not by the next one."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu


def test_a_refused_call_does_not_fail_the_next():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = (f"import sys; sys.path.insert(0, {root!r})\n"
            "import numpy as np, acfun_b200 as acf\n"
            "x, pos, spec = np.ones((2, 1, 8), np.float32), np.zeros(2, np.int32), acf.Rope(np.ones(4, np.float32))\n"
            "try: acf.rope(x, pos, spec); sys.exit('no such device, but no error')\n"
            "except acf.AcfunError as e: assert 'cudaSetDevice' in str(e), e\n"
            "assert acf.lib().acfun_set_device(0) == 0\n"
            "assert (acf.rope(x, pos, spec) == x).all()\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, ACFUN_DEVICE="40"))
    assert r.returncode == 0, r.stdout + r.stderr
