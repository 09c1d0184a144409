"""Prompt attention's kernel, checked without a GPU: the waits in the code that the compiler makes of
it, and the search of its tiles.

No counterpart in the reference (its prefill is the model's own forward pass, engine.py:42-49)."""
import os
import re
import shutil
import subprocess

import pytest

from exactkv_amd import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _hipcc():
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    return hipcc


def test_barriers_wait_for_lds_reads(tmp_path):
    """Tiles are loaded straight to LDS by other wavefronts right behind a barrier, so in front of
    it every wavefront's loads have landed and its reads of the stage have returned."""
    asm = tmp_path / "prompt.s"
    subprocess.run([_hipcc(), *build.HIP_FLAGS, "-w", "--offload-device-only", "-S", "-o", str(asm),
                    os.path.join(build.CSRC, "prompt.hip")], check=True, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    lines = [x.split(";")[0].strip() for x in asm.read_text().splitlines()]
    lines = [x for x in lines if x and (not x.startswith(".") or x.endswith(":"))]
    starts = [i for i, x in enumerate(lines) if re.match(r"_ZN4exkv13prompt_kernel\w*:$", x)]
    assert len(starts) == 4                            # head dims 64, 128 and 256, the last one twice
    at = [i for i, x in enumerate(lines) if x == "s_barrier"]
    for a, b in zip(starts, starts[1:] + [len(lines)]):
        assert any(a < i < b for i in at)
    for i in at:
        wait = lines[i - 1].split()
        assert wait[0] == "s_waitcnt" and "vmcnt(0)" in wait and "lgkmcnt(0)" in wait, lines[i - 4:i + 1]


def test_every_tile_and_part_is_taken_once(tmp_path):
    """The search of a workgroup's row tile and part of its keys (csrc/prompt_tiles.hpp), which the
    addresses of its reads follow from, over random offsets, sound and broken, and every number of
    parts (tests/native/tiles_check.cpp)."""
    exe = tmp_path / "tiles_check"
    subprocess.run([_hipcc(), "-O2", "-o", str(exe), os.path.join(ROOT, "tests", "native", "tiles_check.cpp")],
                   check=True, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    r = subprocess.run([str(exe)], stdout=subprocess.PIPE, text=True)
    assert r.returncode == 0, r.stdout
    assert " 0 failures" in r.stdout
