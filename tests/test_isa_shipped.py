"""CPU: the invariant of tests/test_isa_invariants.py -- no scratch traffic inside a hand-counted LDS-DMA loop -- for the code as it ships: every source that holds such loops,
the row operators' among them, with the Makefile's own flags (packed fp32 arithmetic off) and for both 16-bit builds."""
import os
import re
import shlex
import subprocess
import tempfile
from concurrent.futures import ThreadPoolExecutor

import pytest

from tests.test_isa_invariants import CSRC, HIPCC, ROOT, SOURCES, _dma_loops_with_scratch

ROWS = ["linear.hip", "linear256.hip", "linear_rows.hip", "linear_wgrad256.hip"]


def _flags():
    text = open(os.path.join(CSRC, "Makefile")).read()
    flags = shlex.split(re.search(r"^CXXFLAGS := (.*)$", text, re.M).group(1).replace("$(ARCH)", "gfx950"))
    assert "-packed-fp32-ops" in flags
    return flags


def _asm(job):
    src, half, out_dir = job
    out = os.path.join(out_dir, src.replace(".hip", f"{half}.s"))
    cmd = [HIPCC, *_flags(), *(["-DSH_H16_FP16"] if half == "f16" else []), f"-I{os.path.join(ROOT, 'include')}", "-S", "--cuda-device-only", "-o", out, os.path.join(CSRC, src)]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stderr[-2000:]
    return open(out).read()


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not found")
def test_every_source_with_dma_loops_is_looked_at():
    held = {f for f in os.listdir(CSRC) if f.endswith(".hip") and "global_load_lds" in open(os.path.join(CSRC, f)).read()}
    assert held <= set(SOURCES) | set(ROWS), held - set(SOURCES) - set(ROWS)


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not found")
def test_no_scratch_traffic_inside_the_shipped_dma_loops():
    jobs = [(s, "bf16") for s in SOURCES + ROWS] + [(s, "f16") for s in ROWS]
    with tempfile.TemporaryDirectory() as tmp, ThreadPoolExecutor(max_workers=min(6, os.cpu_count() or 2)) as pool:
        asms = list(pool.map(_asm, [j + (tmp,) for j in jobs]))
    seen, bad = {}, []
    for (src, half), asm in zip(jobs, asms):
        seen[src] = seen.get(src, 0) + len(re.findall(r"global_load_lds", asm))
        bad += [(src, half) + b for b in _dma_loops_with_scratch(asm)]
        assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", asm), f"{src}: packed fp32 arithmetic"
    assert all(seen[s] > 4 for s in ROWS), "the scan found no LDS-DMA kernels: the sources or the pattern moved"
    assert not bad, "scratch traffic inside a hand-counted DMA loop (hipcc waits vmcnt(0) behind it):\n" + "\n".join(map(str, bad))


def test_every_recipe_builds_with_those_flags():
    """Variants and probes are timed and compared against the shipped kernels: their compile lines leave packed fp32 arithmetic out as well."""
    scripts = os.path.join(ROOT, "scripts")
    for d, _, files in os.walk(scripts):
        for f in files:
            if f.endswith((".sh", ".hip", ".py")):
                for line in open(os.path.join(d, f), errors="replace"):
                    if re.search(r"hipcc\b.*(-c|-O3|\$src)\b", line) and "-shared" not in line:
                        assert "-packed-fp32-ops" in line or "$flags" in line, (f, line)
    assert "CXXFLAGS" in open(os.path.join(scripts, "build_variant.sh")).read()
