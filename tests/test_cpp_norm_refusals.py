"""Tables of the ranks' buffers that the C++ front end's norms refuse."""
import os
import subprocess

import pytest

EXE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "test_norm_refusals")


@pytest.mark.gpu
def test_norm_refusals_program():
    assert os.path.exists(EXE), "tests/cpp/test_norm_refusals is not built (make -C tests/cpp)"
    p = subprocess.run([EXE], capture_output=True, text=True, timeout=120)
    print(p.stdout[-3000:], p.stderr[-1000:])
    assert p.returncode == 0, p.stdout[-3000:]
    assert "PASSED" in p.stdout
