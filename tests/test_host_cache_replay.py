"""The cache operators' address code, replayed on the CPU under AddressSanitizer and
UndefinedBehaviorSanitizer (tests/host_addr/cache_replay.cpp calls
csrc/ssa_cache_plan.hpp as the kernels do), and mistakes planted in a copy of the
headers, each of which the replay has to find."""

from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "luciole-1b_amd" / "csrc"
SRC = ROOT / "tests" / "host_addr" / "cache_replay.cpp"
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
BASE = ["-x", "hip", "--cuda-host-only", "-std=c++20"]
SAN = ["-O1", "-g", "-Xarch_host", "-fsanitize=address", "-Xarch_host", "-fsanitize=undefined",
       "-Xarch_host", "-fno-sanitize-recover=all"]

pytestmark = pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc not found")


def _build(out: Path, include: Path, flags: list[str]) -> None:
    cmd = [HIPCC, *BASE, *flags, "-I", str(include), str(SRC), "-o", str(out)]
    res = subprocess.run(cmd, capture_output=True, text=True, timeout=900)
    assert res.returncode == 0, f"{' '.join(cmd)}\n{res.stdout}\n{res.stderr[-4000:]}"


def _run(exe: Path, *args: str) -> subprocess.CompletedProcess:
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0", UBSAN_OPTIONS="print_stacktrace=1")
    return subprocess.run([str(exe), *args], capture_output=True, text=True, timeout=900, env=env)


def test_cache_replay_under_sanitizers(tmp_path):
    exe = tmp_path / "cache_replay"
    _build(exe, CSRC, ["-Wall", "-Werror", *SAN])
    res = _run(exe)
    assert res.returncode == 0, f"rc {res.returncode}\n{res.stdout[-3000:]}\n{res.stderr[-6000:]}"
    assert " 0 failures" in res.stdout and "FAILED" not in res.stdout, res.stdout[-3000:]
    assert "runtime error" not in res.stderr, res.stderr[-4000:]


# (file, original text, planted mistake, what it breaks)
MUTATIONS = [
    ("ssa_row_tile.hpp", "row = row < nrows ? row : nrows - 1;", "row = row <= nrows ? row : nrows - 1;",
     "the row clamp of partial tiles"),
    ("ssa_row_tile.hpp", "if (row0 + 32 * BLOCKS <= nrows && ", "if (row0 + 32 * BLOCKS <= nrows + 8 && ",
     "a partial tile loaded as a whole one"),
    ("ssa_row_tile.hpp", "return (lane % R::LPR) ^ (4 * R::swz(lane / R::LPR));", "return lane % R::LPR;",
     "the quarters' permutation on the loads' side"),
    ("ssa_row_tile.hpp", "return p * 1024 + (p & 3) * 16 + (p >> 2) * 256;", "return p * 1024 - (p & 3) * 16 + (p >> 2) * 256;",
     "pieces that overlap"),
    ("ssa_row_tile.hpp", "const int s = D == 128 ? i >> 2 : 4 * hh + (i >> 2);", "const int s = D == 128 ? i >> 2 : 4 * hh + (i & 3);",
     "the rows of V's transpose reads"),
    ("ssa_cache_plan.hpp", "const int row0 = u.kbeg + C::KEYS * i;", "const int row0 = u.kbeg + C::KEYS * (i + 1) - 32;",
     "a stage's first key"),
    ("ssa_cache_plan.hpp", "const uint32_t dst = lds0 + (i & 1) * 2 * C::TILE;", "const uint32_t dst = lds0 + (i & 1) * C::TILE;",
     "buffers that overlap"),
    ("ssa_cache_plan.hpp", "kend = beg + p.split_keys < L ? static_cast<int>(beg + p.split_keys) : L;",
     "kend = beg + p.split_keys <= L ? static_cast<int>(beg + p.split_keys) : L + 1;", "a split one key past the sequence"),
    ("ssa_cache_plan.hpp", "(u.G * p.T) + r) * p.splits + u.split;", "(u.G * p.T) + r) * p.splits + (p.splits - 1 - u.split);",
     "the partials' order of splits"),
    ("ssa_cache_plan.hpp", "return static_cast<int>((L + p.split_keys - 1) / p.split_keys);",
     "return static_cast<int>(L / p.split_keys + 1);", "a split without keys joined"),
    ("ssa_cache_ops.hpp", "return static_cast<int>((rows + per - 1) / per);", "return static_cast<int>((rows + per - 1) / per + 1);",
     "a chunk without rows joined"),
    ("ssa_cache_plan.hpp", "return sees / p.chunk_rows;", "return sees / p.chunk_rows - (sees >= p.chunk_rows);",
     "a chunk that no key's sum was written to"),
    ("ssa_cache_plan.hpp", "    if (g >= u.G) {\n      g -= u.G;\n      ++t;\n    }", "    if (g > u.G) {\n      g -= u.G;\n      ++t;\n    }",
     "the walk over a group's heads"),
    ("ssa_cache_plan.hpp", "return Row{in, in ? t : p.T - 1, in ? g : u.G - 1};", "return Row{in, t, in ? g : u.G - 1};",
     "queries past the last"),
    ("ssa_cache_plan.hpp", "rstart = sees > from ? sees : from;", "rstart = sees > from ? sees + ROWS : from;",
     "rows that see a key left out"),
]


def _mutant(tmp_path: Path, k: int, fname: str, old: str, new: str) -> tuple[int, str]:
    inc = tmp_path / f"m{k}" / "csrc"
    shutil.copytree(CSRC, inc, ignore=shutil.ignore_patterns("*.hip", "*.cpp"))
    path = inc / fname
    text = path.read_text()
    assert text.count(old) == 1, f"mutation {k}: the original text is not in {fname} exactly once"
    path.write_text(text.replace(old, new))
    _build(inc / "replay", inc, SAN)
    res = _run(inc / "replay", "--quick")
    return res.returncode, res.stderr


def test_planted_mistakes_are_found(tmp_path):
    with cf.ThreadPoolExecutor(max_workers=min(6, os.cpu_count() or 1)) as ex:
        futs = [ex.submit(_mutant, tmp_path, k, f, o, n) for k, (f, o, n, _) in enumerate(MUTATIONS)]
        results = [f.result() for f in futs]
    missed = [why for (rc, err), (_, _, _, why) in zip(results, MUTATIONS)
              if rc == 0 or not ("FAIL" in err or "AddressSanitizer" in err or "runtime error" in err)]
    assert not missed, f"planted mistakes the replay did not find: {missed}"
