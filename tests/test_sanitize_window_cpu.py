"""The windowed planners, and the page lists and tile walks that they and the kernels
share, under AddressSanitizer and UndefinedBehaviorSanitizer (tests/sanitize/window_fuzz.cpp):
against an enumeration of the tokens that are seen, and with malformed metadata, which must
come back as an error status.  CPU only."""

import os
import shutil
import subprocess

import pytest

HERE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "sanitize")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


@pytest.mark.skipif(not os.path.exists(HIPCC) or shutil.which("make") is None,
                    reason="needs hipcc and make")
def test_windows_under_sanitizers():
    subprocess.run(["make", "-C", HERE, "window_fuzz", f"HIPCC={HIPCC}"], check=True,
                   capture_output=True, timeout=600)
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    for seed in (1, 2, 3):
        r = subprocess.run([os.path.join(HERE, "window_fuzz"), "8000", str(seed)], env=env,
                           capture_output=True, text=True, timeout=600)
        report = r.stdout[-2000:] + r.stderr[-6000:]
        assert r.returncode == 0, report
        assert "runtime error" not in r.stderr and "Sanitizer" not in r.stderr, report
        assert "0 failures" in r.stdout, report
