"""Build of the MI355X library (libcogito_mi355x.so) and the CPU checkers.

HIP sources are compiled for gfx950 only with hipcc; the host C that
implements cogito's API is compiled with gcc; everything links into one
shared library under cogito_amd/lib/.  The build always recompiles (it is the
"does it build" check) and runs the compiles in parallel.
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
OBJDIR = PKG / "_build"
LIBDIR = PKG / "lib"
LIBNAME = "libcogito_mi355x.so"
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"

HIP_FLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC",
    # packed fp32 instructions stay off (they have miscomputed on this pool)
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
    f"-I{INCLUDE}", f"-I{CSRC}",
]
# Files whose arithmetic must round exactly where written (no implicit
# contraction of a*b+c into fma).  decoder.hip is among them so that RoPE's
# x0 c - x1 s rounds twice, as the reference's CPU code does, whatever the
# surrounding code looks like (with contraction the backend fuses such pairs,
# in the inlined sin / cos / pow too, depending on the code's layout).  paged.hip
# for its append, whose codes have to be the same bits as the contiguous cache's.
EXACT_FP = {"accept.hip", "int4.hip", "filter.hip", "tree.hip", "decoder.hip",
            "paged.hip"}
C_FLAGS = ["-O2", "-fPIC", "-std=c11", "-Wall", "-Wextra", "-Wno-unused-parameter",
           # a call to an undeclared function (e.g. POSIX strdup under C11)
           # would truncate a returned pointer to int
           "-Werror=implicit-function-declaration",
           f"-I{INCLUDE}", f"-I{CSRC}"]


def _run(cmd: list[str]) -> tuple[list[str], int, str]:
    p = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    return cmd, p.returncode, p.stdout


def _compile_jobs() -> list[tuple[list[str], Path]]:
    jobs = []
    for src in sorted(CSRC.glob("*.hip")):
        obj = OBJDIR / (src.stem + ".hip.o")
        flags = list(HIP_FLAGS)
        if src.name in EXACT_FP:
            flags.append("-ffp-contract=off")
        jobs.append(([HIPCC, *flags, "-c", str(src), "-o", str(obj)], obj))
    for src in sorted((CSRC / "host").glob("*.c")):
        obj = OBJDIR / (src.stem + ".c.o")
        jobs.append((["gcc", *C_FLAGS, "-c", str(src), "-o", str(obj)], obj))
    return jobs


def build_library(verbose: bool = True) -> Path:
    OBJDIR.mkdir(exist_ok=True)
    LIBDIR.mkdir(exist_ok=True)
    jobs = _compile_jobs()
    workers = min(len(jobs), max(1, min(8, os.cpu_count() or 1)))
    failed = []
    with cf.ThreadPoolExecutor(max_workers=workers) as ex:
        for cmd, rc, out in ex.map(lambda j: _run(j[0]), jobs):
            if rc != 0:
                failed.append((cmd, out))
            elif verbose and out.strip():
                # keep compiler warnings visible, minus the known host-pass note
                lines = [l for l in out.splitlines() if "packed-fp32-ops" not in l]
                if lines:
                    print("\n".join(lines), file=sys.stderr)
    if failed:
        msg = "\n\n".join(" ".join(c) + "\n" + o for c, o in failed)
        raise RuntimeError(f"compilation failed:\n{msg}")
    lib = LIBDIR / LIBNAME
    tmp = LIBDIR / (LIBNAME + ".tmp")
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", str(tmp),
           *[str(o) for _, o in jobs]]
    _, rc, out = _run(cmd)
    if rc != 0:
        raise RuntimeError(f"link failed:\n{' '.join(cmd)}\n{out}")
    os.replace(tmp, lib)
    if verbose:
        print(f"built {lib}")
    return lib


def build_checkers(verbose: bool = True) -> None:
    """oracle/_build/liboracle.so, and oracle/_ref/libcgref.so when the
    reference tree is present (test infrastructure, not the product)."""
    cmd = ["make", "-C", str(ROOT / "oracle"), "-j4", "all"]
    _, rc, out = _run(cmd)
    if verbose:
        print(out.strip())
    if rc != 0:
        raise RuntimeError(f"checker build failed:\n{out}")


def build_all(verbose: bool = True) -> Path:
    lib = build_library(verbose)
    build_checkers(verbose)
    return lib


if __name__ == "__main__":
    build_all()
