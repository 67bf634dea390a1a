"""How the calls of the half-precision product, the norms between blocks and the sampling are launched, on the CPU
(host/block_launches.cpp): limits of LDS, shapes of grids, every kernel by the device tests' cases, the ends of every
size and type."""
import itertools
import os
import subprocess

import pytest

import host_launches as H
from host_launches import BF16, F16, F32
from syntropy_amd import _lib

NONE = 9
TYPES = (F32, F16, BF16)


def program(out_dir, where=os.path.dirname(_lib.LIB_PATH), flags=()) -> str:
    exe = os.path.join(str(out_dir), "block_launches")
    subprocess.run([H.CLANG, "-std=c++17", "-O1", "-Wall", *flags, os.path.join(H.HERE, "host", "block_launches.cpp"), "-o", exe, f"-L{where}",
                    "-l:libsyntropy_hip.so", f"-Wl,-rpath,{where}", "-Wl,--allow-shlib-undefined", "-rdynamic"], check=True, capture_output=True,
                   text=True)
    return exe


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    if H.MISSING:
        pytest.skip("needs the built library and ROCm's clang++")
    return program(tmp_path_factory.mktemp("block_launches"))


def test_lds_is_allowed_on_every_device(exe):
    shapes = ((4096, 4096, 20), (4096, 512, 100), (4096, 4096, 512), (14336, 4096, 128), (14336, 4096, 2048), (300, 14336, 40), (64, 64, 3))
    calls = []
    for device in (0, 1, 7, 0, 200):
        calls += [f"device {device}"] + [f"half {w} {n} {k} {rows} 0 {k} {y} {NONE} {F32}" for w in (F16, BF16) for n, k, rows in shapes
                                         for y in (F32, F16)]
    seen = set()
    for c, answer in zip(calls, H.run(exe, calls)):
        assert answer[-1] == "rc 0", c
        for device, lds, limit, name in H.launches(answer):
            if lds > 65536:
                seen.add((device, name))
                assert limit >= lds, f"{c}: {name} asks for {lds} bytes of LDS on device {device}, allowed {limit}"
    assert {d for d, _ in seen} == {0, 1, 7, 200} and len(seen) >= 4 * 12


def test_the_cases_of_the_device_tests_reach_every_kernel(exe):
    """Those of test_gpu_half.py, test_gpu_block_norm.py and test_gpu_sample.py."""
    from test_gpu_block_norm import WIDTHS
    from test_gpu_half import SHAPES
    kernels = {line[len("kernel "):] for line in H.run(exe, ["kernels"])[0]
               if any(f"syn::k_{k}" in line for k in ("half_", "block_norm", "sample"))}
    assert sum("k_half_gemm" in k for k in kernels) == 36 and len(kernels) >= 36 + 2 + 8 + 7 * 9 + 5 * 3
    calls = [f"half {w} {n} {k} {rows} 0 {k} {y} {NONE} {NONE}" for w in (F16, BF16) for n, k, rows in SHAPES for y in (F32, w)]
    # (the device test of widths has two of the types, that of types all of them at three widths)
    calls += [f"norm {x} {b} {F32} 20 {n} 17" for x, b in itertools.product(TYPES, TYPES) for n in WIDTHS]
    calls += [f"sample {t} {rows} {vocab} {k} {each}" for t in TYPES for rows, vocab, k, each in ((6, 1000, 0, 0), (14, 100003, 9, 1))]
    run = {name for answer in H.run(exe, calls) for *_, name in H.launches(answer)}
    assert kernels <= run, "not launched: " + ", ".join(sorted(kernels - run))


def test_no_estimate_raises_an_invalid_operation(exe):
    for n, k, rows in itertools.product((0, 1, 4096, (1 << 24) - 1), (1, 1000, 1 << 20), (0, 1, 9, 2097120)):
        (need,) = H.run(exe, [f"halfneed {n} {k} {rows} 0"])
        assert need[-1] == "rc 0" and need[0].split()[2] == "0", (n, k, rows)
        if not n or not rows:
            assert need[0].split()[1] == "0"


NS = (0, 1, 63, 4096, 1 << 20, (1 << 24) - 1, 1 << 24, (1 << 32) - 1)
KS = (0, 1, 128, 4095, 14336, 1 << 20, (1 << 20) + 1, (1 << 32) - 1)
ROWS = (0, 1, 8, 9, 333, 2097120, 2097121, (1 << 24) - 1, 1 << 24, (1 << 32) - 1)


def at_their_ends(exe, env=None):
    calls = [f"half {(F16, BF16, F32)[i % 7 % 3]} {n} {k} {r} {i % 3} {k + 8 * (i % 2)} {TYPES[i % 3]} {(*TYPES, NONE)[i % 4]} {(*TYPES, NONE)[i // 4 % 4]}"
             for i, (n, k, r) in enumerate(itertools.product(NS, KS, ROWS))]
    # (y of what no memory holds is not asked for: its grid is none)
    calls = [c for c in calls if int(c.split()[2]) * int(c.split()[4]) < 1 << 40 or int(c.split()[2]) >= 1 << 24 or int(c.split()[4]) > 2097120]
    calls += [f"half {F16} {n} {k} {r} 0 {s} {F32} {NONE} {NONE}" for n, k, r, s in itertools.product((9, 5000), (64, 640), (9, 70000), (1 << 24, 1 << 29))]
    calls += [f"norm {x} {b} {y} {r} {n} {w}" for (x, b, y), r, n, w in itertools.product(
        ((F32, F16, BF16), (BF16, BF16, BF16), (F16, F32, 2)), ROWS, (0, 1, 512, 513, 4096, 4097, 8193, 32768, 32769, (1 << 32) - 1), (0, 1, 16, 17, 23, 27, 2))]
    calls += [f"sample {t} {r} {n} {k} {e}" for t, r, n, k, e in itertools.product(
        (*TYPES, 2), (0, 1, 128, 129, (1 << 20) + 1, (1 << 24) - 1, 1 << 24, (1 << 32) - 1), (0, 1, 32768, 32769, 65537, 128256, 1 << 24, (1 << 24) + 1, (1 << 32) - 1),
        (0, 64, 65, (1 << 31) - 1), (0, 1))]
    answers = H.run(exe, calls, env)
    for c, a in zip(calls, answers):
        what, *v = c.split()
        v = [int(t) for t in v]
        launched, ok = bool(H.launches(a)), a[-1] == "rc 0"
        if what == "half":
            w, n, k, r, _, stride = v[:6]
            fits, some = w != F32 and 1 <= k <= 1 << 20 and n < 1 << 24 and r <= 2097120, n > 0 and r > 0
        elif what == "norm":
            x, b, y, r, n, w = v
            fits = 1 <= n <= 32768 and r < 1 << 24
            if r:
                fits = fits and (bool(w & 1) or (w & 16 and not w & 14)) and not (w & 16 and y not in TYPES)
            some = r > 0
        else:
            t, r, n, k, e = v
            fits, some = t in TYPES and 1 <= n <= 1 << 24 and r < 1 << 24, r > 0
        assert ok == bool(fits), f"{c}: {a[-1]}"
        assert launched == bool(fits and some), c


def test_sizes_at_their_ends(exe):
    at_their_ends(exe)
