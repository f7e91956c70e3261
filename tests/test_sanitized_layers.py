"""The CPU tests of the norms' and the 4-bit weights' entries with the library's host code under AddressSanitizer and
UndefinedBehaviorSanitizer: argument checks and workspace counting up to the sizes' limits.  Any report fails the run.
"""

from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

from guass_amd import build

ROOT = Path(__file__).resolve().parent.parent
TESTS = ["tests/test_norms.py", "tests/test_quantized.py"]


def _library() -> Path:
    """The sanitized library, built anew unless the one that lies there is younger than every source (tests/test_sanitized_host.py,
    which runs before this, builds it too)."""
    lib = build.SANITIZE_DIR / "libgaussfield.so"
    sources = [*build.CSRC.iterdir(), ROOT / "include" / "gaussfield.h", Path(build.__file__)]
    if not lib.exists() or lib.stat().st_mtime <= max(p.stat().st_mtime for p in sources):
        build.build_sanitized()
    return lib


def test_block_cpu_tests_under_asan_and_ubsan():
    env = dict(os.environ)
    env.update({
        "LD_PRELOAD": str(build.asan_runtime()),
        "ASAN_OPTIONS": "detect_leaks=0:abort_on_error=1:halt_on_error=1:symbolize=1",
        "UBSAN_OPTIONS": "halt_on_error=1:print_stacktrace=1",
        "GUASS_AMD_LIB": str(_library()),
    })
    proc = subprocess.run([sys.executable, "-m", "pytest", "-q", "-m", "not gpu", "-p", "no:cacheprovider", *TESTS], cwd=ROOT, env=env,
                          capture_output=True, text=True, timeout=900)
    out = proc.stdout[-6000:] + "\n" + proc.stderr[-6000:]
    assert proc.returncode == 0, out
    for marker in ("ERROR: AddressSanitizer", "runtime error:", "SUMMARY: UndefinedBehaviorSanitizer"):
        assert marker not in proc.stdout + proc.stderr, out
    assert " passed" in proc.stdout, out
