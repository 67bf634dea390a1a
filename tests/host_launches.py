"""Runs tests/host/launches.cpp: the library's host code over a runtime that writes launches down."""
from __future__ import annotations

import os
import subprocess

from syntropy_amd import _lib

CLANG = "/opt/rocm/llvm/bin/clang++"
HERE = os.path.dirname(os.path.abspath(__file__))
MISSING = not (os.path.exists(CLANG) and os.path.exists(_lib.LIB_PATH))
F32, F16, BF16 = 0, 1, 30


def build(out_dir, where=os.path.dirname(_lib.LIB_PATH), flags=()) -> str:
    """The program over the library in `where`, into out_dir."""
    exe = os.path.join(str(out_dir), "launches")
    subprocess.run([CLANG, "-std=c++17", "-O1", "-Wall", *flags, os.path.join(HERE, "host", "launches.cpp"), "-o", exe, f"-L{where}",
                    "-l:libsyntropy_hip.so", f"-Wl,-rpath,{where}", "-Wl,--allow-shlib-undefined", "-rdynamic"], check=True, capture_output=True,
                   text=True)
    return exe


def run(exe: str, commands, env=None) -> list[list[str]]:
    """The answers' lines of each command, its "rc" last."""
    r = subprocess.run([exe], input="\n".join(commands) + "\n", capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and "runtime error" not in r.stderr and "Sanitizer" not in r.stderr, r.stderr[-6000:]
    out, at = [], []
    for line in r.stdout.splitlines():
        at.append(line)
        if line.startswith("rc "):
            out.append(at)
            at = []
    assert len(out) == len(commands) and not at
    return out


def launches(answer) -> list[tuple[int, int, int, str]]:
    """(device, dynamic LDS, the limit said for that device, kernel) of each launch."""
    return [(int(d), int(lds), int(limit), name)
            for d, lds, limit, name in (line.split(" ", 4)[1:] for line in answer if line.startswith("launch "))]
