"""That the device tests' own cases reach every form of the half-precision product's epilogue and of the norms between
blocks, on the CPU (host/block_launches.cpp): the lists that those tests run over are what is launched here."""
import re

import host_launches as H
from host_launches import BF16, F16, F32
from test_block_launches import exe  # noqa: F401

CODE = {"torch.float32": F32, "torch.float16": F16, "torch.bfloat16": BF16}


def test_each_epilogue_case_is_another_tile(exe):  # noqa: F811
    from test_gpu_half_tiles import CASES
    seen, tiles = set(), {}
    for w in (F16, BF16):
        for out in (F32, F16, BF16):
            calls = [f"half {w} {n} {k} {rows} 0 {k} {out} {F16} {F32}" for n, k, rows in CASES]
            for case, answer in zip(CASES, H.run(exe, calls)):
                names = [name for *_, name in H.launches(answer) if "k_half_gemm" in name]
                assert len(names) == 1, case
                tile, kind = re.search(r"HalfTile<([^>]*)>, \d+, (\d)>", names[0]).groups()
                assert tiles.setdefault(case, tile) == tile, case
                seen.add(names[0])
    assert len(set(tiles.values())) == len(CASES)
    every = {line[len("kernel "):] for line in H.run(exe, ["kernels"])[0] if "k_half_gemm" in line}
    left = {k for k in every if ", 0>(" not in k} - seen  # (0: a part's sums, no epilogue)
    assert len(seen) == 24 and not left, "not launched: " + ", ".join(sorted(left))


def test_each_norm_case_is_another_form(exe):  # noqa: F811
    from test_gpu_block_norm_types import CASES
    every = {line[len("kernel "):] for line in H.run(exe, ["kernels"])[0] if "k_block_norm" in line}
    calls = [f"norm {CODE[str(x)]} {CODE[str(b)]} {F32} 7 {n} 23" for x, b, n in CASES]
    names = [name for answer in H.run(exe, calls) for *_, name in H.launches(answer)]
    assert len(names) == len(CASES) == len(every) == 63
    assert set(names) == every, "not launched: " + ", ".join(sorted(every - set(names)))
