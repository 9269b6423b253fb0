"""Host-side validation of the cache operators' C ABI under AddressSanitizer and
UndefinedBehaviorSanitizer, as test_host_sanitize.py has it for the other entry
points: ssa_cache_abi.hip (checks and size queries) and the three sources whose
launches it reaches are compiled with host-only sanitizers and linked with the
library's other objects into tests/host_sanitize/validate_cache.c, which runs on the CPU."""

from __future__ import annotations

import os
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "luciole-1b_amd" / "csrc"
BUILD = ROOT / "luciole-1b_amd" / "_build"
SANITIZED = ("ssa_cache_abi", "ssa_cache", "ssa_key_weights", "ssa_tree")
PLAIN = tuple(sorted(f.stem for f in CSRC.glob("*.hip") if f.stem not in SANITIZED))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
CLANG = "/opt/rocm/llvm/bin/clang"
HOST_SAN = ["-Xarch_host", "-fsanitize=address", "-Xarch_host", "-fsanitize=undefined",
            "-Xarch_host", "-fno-sanitize-recover=all"]


@pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="a GPU is visible; the validation program passes fake device pointers")
def test_cache_validation_is_ub_free_under_sanitizers(tmp_path):
    if not (Path(HIPCC).exists() and Path(CLANG).exists()):
        pytest.skip("hipcc / ROCm clang not found")
    missing = [n for n in PLAIN if not (BUILD / f"{n}.o").exists()]
    if missing:
        pytest.skip(f"library objects not built ({missing}); run __graft_entry__.build() first")
    flags = ["--offload-arch=gfx950", "-O1", "-g", "-std=c++20", "-fPIC",
             "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
    procs = [subprocess.Popen([HIPCC, *flags, *HOST_SAN, "-c", str(CSRC / f"{n}.hip"), "-o", f"{n}.o"],
                              cwd=tmp_path, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)
             for n in SANITIZED]
    for n, p in zip(SANITIZED, procs):
        out, err = p.communicate(timeout=900)
        assert p.returncode == 0, f"{n}: {out}\n{err}"
    san = ["-fsanitize=address,undefined", "-fno-sanitize-recover=all"]
    main = str(ROOT / "tests" / "host_sanitize" / "validate_cache.c")
    objs = ["main.o", *(f"{n}.o" for n in SANITIZED), *(str(BUILD / f"{n}.o") for n in PLAIN)]
    for cmd in ([CLANG, "-O1", "-g", "-std=c11", "-Wall", "-Werror", *san, "-c", main, "-o", "main.o"],
                [CLANG + "++", *san, "-o", "validate", *objs, "-L/opt/rocm/lib", "-lamdhip64", "-Wl,-rpath,/opt/rocm/lib"]):
        res = subprocess.run(cmd, cwd=tmp_path, capture_output=True, text=True, timeout=600)
        assert res.returncode == 0, f"{' '.join(cmd)}\n{res.stdout}\n{res.stderr}"
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0", UBSAN_OPTIONS="print_stacktrace=1")
    res = subprocess.run([str(tmp_path / "validate")], capture_output=True, text=True, timeout=300, env=env)
    assert res.returncode == 0, f"sanitizer run failed (rc {res.returncode}):\n{res.stdout}\n{res.stderr[-4000:]}"
    assert "0 failures" in res.stdout, res.stdout
    assert "runtime error" not in res.stderr, res.stderr[-4000:]
