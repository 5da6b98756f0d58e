"""tests/test_training_edges_emu.py under AddressSanitizer, the threads and blocks of every launch in reverse order and outputs that start
as NaN, as tests/test_training_ops_asan.py does: an access outside a tensor ends the run.  (Without the runs of the attack: minutes.)"""
import os
import subprocess
import sys

import pytest

from test_kernels_asan import RUNTIME, _env
from tests_hipemu import build_emu

HERE = os.path.dirname(os.path.abspath(__file__))

if build_emu.host_compiler() is None or RUNTIME is None:
    pytest.skip("no host clang++ / shared AddressSanitizer runtime", allow_module_level=True)


def test_edges_of_the_training_ops_are_clean_under_address_sanitizer():
    res = subprocess.run([sys.executable, "-m", "pytest", os.path.join(HERE, "test_training_edges_emu.py"), "-q", "-x", "-p", "no:cacheprovider",
                          "-k", "not attack"],
                         env=_env(), cwd=os.path.dirname(HERE), capture_output=True, text=True, timeout=2400)
    tail = (res.stdout + res.stderr)[-3000:]
    assert res.returncode == 0 and "AddressSanitizer" not in res.stdout + res.stderr, tail
    assert " passed" in res.stdout and "failed" not in res.stdout, tail
