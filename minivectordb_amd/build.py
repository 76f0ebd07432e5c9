"""Build libmvdb_hip.so (HIP kernels + C ABI) for gfx950 with hipcc, in-tree."""
from __future__ import annotations

import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB_DIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIB_DIR, "libmvdb_hip.so")
SOURCES = ["engine.hip", "mx4.hip", "host_graph.cpp"]


def _stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [os.path.join(ROOT, "include", "mvdb_hip.h")]
    return any(os.path.getmtime(d) > t for d in deps)


def _current(obj: str, src: str) -> bool:
    """Is this object newer than everything it was compiled from?  (mx4.hip and its mx4_*.hip.hpp stand apart from the rest.)"""
    if not os.path.exists(obj) or not os.path.exists(obj + ".txt"):
        return False
    mx4 = src == "mx4.hip"
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)
            if f.endswith(".hpp") and (f == "mx4.hpp" or f.startswith("mx4_") == mx4)]
    deps += [os.path.join(CSRC, src), os.path.join(ROOT, "include", "mvdb_hip.h"), os.path.abspath(__file__)]
    return all(os.path.getmtime(d) <= os.path.getmtime(obj) for d in deps)


def build(force: bool = False, verbose: bool = False, defines=(), out: str | None = None) -> str:
    """Build the library.  `defines`/`out` build a tuning variant (tools/ only) beside it."""
    target = LIB if out is None else os.path.join(LIB_DIR, out)
    if out is None and not force and not _stale():
        return LIB
    os.makedirs(LIB_DIR, exist_ok=True)
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    flags = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-pthread",
             "-fno-fast-math", "-Wall", "-Wno-unused-function",
             # no packed f32 arithmetic: some forms of v_pk_{add,mul,fma}_f32 have given wrong results on this hardware
             # (the host pass does not know the feature and says so: harmless)
             "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
             "-I", os.path.join(ROOT, "include"), "-I", CSRC]
    flags += ["-Rpass-analysis=kernel-resource-usage"]  # -> lib/kernel_resources.txt (see check_resources)
    flags += ["-D" + d for d in defines]
    # one object per source, compiled side by side; an unforced build takes up the objects whose sources did not change
    obj_dir = os.path.join(LIB_DIR, "_build" if out is None else "_build_" + out)
    os.makedirs(obj_dir, exist_ok=True)
    jobs = []
    for src in SOURCES:
        obj = os.path.join(obj_dir, src + ".o")
        if out is None and not force and _current(obj, src):
            jobs.append((obj, None))
            continue
        cmd = [hipcc] + flags + ["-x", "hip", "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            print(" ".join(cmd))
        with open(obj + ".txt", "w") as f:
            jobs.append((obj, subprocess.Popen(cmd, stdout=f, stderr=subprocess.STDOUT)))
    failed = [obj for obj, proc in jobs if proc is not None and proc.wait() != 0]
    notes = []
    for obj, _ in jobs:
        with open(obj + ".txt") as f:
            notes.append(f.read())
        if obj in failed:
            sys.stderr.write(notes[-1])
            os.remove(obj + ".txt")
    if failed:
        raise RuntimeError("hipcc failed building libmvdb_hip.so")
    notes = "".join(notes)
    r = subprocess.run([hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-pthread"] + [o for o, _ in jobs] + ["-o", target],
                       capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("hipcc failed linking libmvdb_hip.so")
    if verbose:
        sys.stderr.write("".join(l for l in notes.splitlines(True) if "warning" in l and "packed-fp32-ops" not in l))
    if out is None:
        with open(RESOURCES, "w") as f:
            f.write(_resource_table(notes))
        check_resources()
    return target


RESOURCES = os.path.join(LIB_DIR, "kernel_resources.txt")


def _resource_table(stderr: str) -> str:
    """hipcc's per-kernel remarks -> one line per kernel: name VGPRs AGPRs scratch occupancy."""
    import re
    rows, cur = [], None
    for line in stderr.splitlines():
        m = re.search(r"remark: +(Function Name|VGPRs|AGPRs|ScratchSize \[bytes/lane\]|Occupancy \[waves/SIMD\]): (\S+)", line)
        if not m:
            continue
        if m.group(1) == "Function Name":
            cur = [m.group(2)]
            rows.append(cur)
        elif cur is not None:
            cur.append(m.group(2))
    return "".join(" ".join(r) + "\n" for r in rows if len(r) == 5)


def check_resources() -> None:
    """The lean traversal is latency-bound: its throughput is waves resident x 1 / chain time.  At 384-512 B rows it
    sits close to 256 VGPRs, where one more live value halves the residency (2 -> 1 waves per SIMD) without any test
    noticing.  Refuse a build in which that happened, or in which the kernel spills."""
    import re
    if not os.path.exists(RESOURCES):
        return
    for line in open(RESOURCES):
        name, vgpr, agpr, scratch, occ = line.split()
        m = re.match(r"_ZN4mvdb20traverse_lean_kernelILi(\d)ELb([01])EEEvNS_12TraverseArgsE", name)
        if not m:
            continue
        j, full = int(m.group(1)), m.group(2) == "1"   # rows of up to j * 128 bytes; full: exactly that many
        # the benchmarked shapes (384- and 512-byte rows) strictly; ragged row sizes may spill a little, and 385..511-byte
        # rows (j = 4, not full) run with one wave per SIMD
        if (j <= 3 and int(occ) < 2) or (full and j <= 4 and int(occ) < 2) or (full and j <= 3 and int(scratch) > 0):
            raise RuntimeError(f"{name}: {vgpr} VGPRs + {agpr} AGPRs, {scratch} B scratch, {occ} wave(s) per SIMD -- "
                               "the lean traversal must keep 2 waves per SIMD and, for full 128/256/384-byte rows, no scratch (see build.py)")


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
