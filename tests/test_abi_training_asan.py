"""The argument checks of the training step's operators' entry points
(tests/test_abi_training.py) against the build of the library whose host code
runs under AddressSanitizer.  CPU only: no entry point reaches a kernel launch."""
import os
import shutil
import subprocess
import sys

import pytest

from terra_amd import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _library():
    """The sanitized library, built unless one is there that is newer than its sources."""
    sources = [os.path.join(d, f) for d in (build.CSRC, os.path.join(ROOT, "include")) for f in os.listdir(d)]
    if os.path.exists(build.ASAN_LIB_PATH) and \
            os.path.getmtime(build.ASAN_LIB_PATH) > max(map(os.path.getmtime, [*sources, build.__file__])):
        return build.ASAN_LIB_PATH
    return build.build_library(asan_host=True)


@pytest.mark.skipif(shutil.which("hipcc") is None and not os.path.exists("/opt/rocm/bin/hipcc"),
                    reason="hipcc (ROCm) needed to build the sanitized library")
def test_checks_under_host_address_sanitizer():
    lib = _library()
    env = dict(os.environ, LD_PRELOAD=build.asan_runtime(), TERRA_SWIN_LIB=lib,
               ASAN_OPTIONS="detect_leaks=0:abort_on_error=0:halt_on_error=1:exitcode=66")
    run = subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "no:cacheprovider", "-m", "not gpu",
                          os.path.join(ROOT, "tests", "test_abi_training.py")], cwd=ROOT, env=env,
                         stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=600)
    assert run.returncode == 0, run.stdout[-4000:]
    assert "ERROR: AddressSanitizer" not in run.stdout
    assert " passed" in run.stdout
