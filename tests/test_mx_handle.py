"""CPU: the handle of a microscaled weight as tests/test_mx_api.py lays it out is the library's (cgx_internal.h)."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

from test_mx_api import Weight

ROOT = Path(__file__).resolve().parent.parent


def test_layout_of_the_handle(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    names = [n for n, _ in Weight._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "cg_mi355x.h"\n#include "cgx_internal.h"\nint main(void) {\n' +
                   "".join(f'printf("%zu ", offsetof(cgx_mx_weight, {n}));\n' for n in names) +
                   'printf("%zu\\n", sizeof(cgx_mx_weight));\nreturn 0;\n}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", f"-I{ROOT / 'include'}", f"-I{ROOT / 'cogito_amd' / 'csrc'}", "-o", str(exe), str(src)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    import ctypes
    assert got == [getattr(Weight, n).offset for n in names] + [ctypes.sizeof(Weight)]
