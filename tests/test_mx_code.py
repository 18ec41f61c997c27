"""CPU: the machine code of the 32-value conversions.  They write their result over several cycles in which they
still read their operands, so that no register of the result may be one of an operand's; the compiler does not keep
them apart by itself."""
from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

OBJ = Path(__file__).resolve().parent.parent / "cogito_amd" / "_build"
LLVM = Path("/opt/rocm/llvm/bin")
FORM = re.compile(r"(v_cvt_scalef32_(?:2xpk16|pk32)_\w+)\s+([^/\n]*)")


def _regs(text):
    out = []
    for kind, lo, hi, one in re.findall(r"([av])(?:\[(\d+):(\d+)\]|(\d+))", text):
        lo, hi = (int(one), int(one)) if one else (int(lo), int(hi))
        out.append({(kind, i) for i in range(lo, hi + 1)})
    return out


def _device_code(obj: Path, tmp: Path) -> str:
    part = tmp / (obj.name + ".elf")
    subprocess.run([LLVM / "clang-offload-bundler", "--type=o", "--unbundle", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950",
                    f"--input={_bundle(obj, tmp)}", f"--output={part}"], check=True)
    return subprocess.run([LLVM / "llvm-objdump", "-d", "--mcpu=gfx950", part], check=True, capture_output=True, text=True).stdout


def _bundle(obj: Path, tmp: Path) -> Path:
    out = tmp / (obj.name + ".bundle")
    subprocess.run([LLVM / "llvm-objcopy", f"--dump-section=.hip_fatbin={out}", obj, tmp / "copy.o"], check=True)
    return out


@pytest.mark.parametrize("name", ["mx", "mx_loss"])
def test_conversions_keep_their_operands(name, tmp_path):
    obj = OBJ / f"{name}.hip.o"
    if not obj.exists() or not shutil.which(str(LLVM / "llvm-objdump")):
        pytest.skip("no object file of this build")
    found = 0
    for op, args in FORM.findall(_device_code(obj, tmp_path)):
        regs = _regs(args)
        assert len(regs) >= (3 if "2xpk16" in op else 2), (op, args)   # the scale may be a constant
        found += 1
        assert not any(regs[0] & r for r in regs[1:]), f"{op} {args}"
    assert found > 0
