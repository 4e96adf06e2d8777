"""The first call of a process to the fixed-rate operators' torch entry points: what it refuses it leaves as it was."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", ["device", "status", "capture", "threads"])
def test_first_call(case):
    at = os.path.join(os.path.dirname(os.path.abspath(__file__)), "native", "first_call.py")
    got = subprocess.run([sys.executable, at, case], capture_output=True, text=True, timeout=100)
    assert got.returncode == 0 and got.stdout.endswith("fine\n"), got.stdout + got.stderr
