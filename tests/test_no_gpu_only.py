"""Tests that hand made-up device addresses to the library run only where no GPU is present."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

RUN = """
import sys
import pytest
from tpt_spark_b200 import _lib
_lib.lib().tptc_device_count = lambda: 1  # as on a machine with a GPU
sys.exit(pytest.main(["tests/test_serve_args.py", "-q", "-p", "no:cacheprovider"]))
"""


def test_made_up_addresses_stay_off_a_gpu():
    r = subprocess.run([sys.executable, "-c", RUN], cwd=ROOT, capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, CUDA_VISIBLE_DEVICES=""))
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    last = r.stdout.strip().splitlines()[-1]
    assert "skipped" in last and "passed" not in last, last
