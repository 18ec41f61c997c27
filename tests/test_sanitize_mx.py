"""CPU: the host side of the microscaled weights (host/mx.c) built with AddressSanitizer and UndefinedBehaviorSanitizer
against a runtime in host memory (tests/sanitize/mx_host.c): the list of chunks and layers, and every failure on the way,
which has to leave nothing behind."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent
ROOT = HERE.parent


def test_weights_under_asan_and_ubsan(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    exe = tmp_path / "mx_host"
    b = subprocess.run(["gcc", "-O1", "-g", "-std=c11", "-D_GNU_SOURCE", "-Wall", "-Werror=implicit-function-declaration",
                        "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-fno-omit-frame-pointer",
                        f"-I{ROOT / 'include'}", f"-I{ROOT / 'cogito_amd' / 'csrc'}", "-o", str(exe),
                        str(HERE / "sanitize" / "mx_host.c"), str(ROOT / "cogito_amd" / "csrc" / "host" / "mx.c")],
                       capture_output=True, text=True)
    assert b.returncode == 0, b.stdout + b.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    out = r.stdout + r.stderr
    assert r.returncode == 0, out
    assert "runtime error" not in out and "Sanitizer" not in out, out
    assert "mx host check: ok" in out
