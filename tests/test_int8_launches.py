"""How the int8 products' calls are launched, on the CPU (host_launches.py)."""
import pytest

import host_launches as H

pytestmark = pytest.mark.skipif(H.MISSING, reason="needs the built library and ROCm's clang++")


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    return H.build(tmp_path_factory.mktemp("launches"))


def test_lds_is_allowed_on_every_device(exe):
    """A kernel's limit of dynamic LDS is its device's: said on each device before the first launch there."""
    calls = [f"i8 {gated} {n} {k} {rows} {H.BF16} {H.F32} 0" for gated in (0, 1)
             for n, k, rows in ((512, 512, 1), (512, 512, 6), (512, 16384, 1), (512, 512, 12), (4096, 4096, 20), (4096, 4096, 100),
                                (14336, 1024, 2048), (1000, 8192, 100))]
    for device in (0, 1, 7, 0, 200):
        calls += [f"device {device}"] + calls[:16]
    seen = set()
    for c, answer in zip(calls, H.run(exe, calls)):
        assert answer[-1] == "rc 0", c
        for device, lds, limit, name in H.launches(answer):
            if lds > 65536:
                seen.add((device, name))
                assert limit >= lds, f"{c}: {name} asks for {lds} bytes of LDS on device {device}, allowed {limit}"
    assert {d for d, _ in seen} == {0, 1, 7, 200} and len(seen) >= 4 * 4


@pytest.mark.parametrize("rows", [0, 1, 17, 2097120])
@pytest.mark.parametrize("k", [1, 1000, 131072])
def test_a_matrix_without_rows_needs_its_tokens_alone(exe, k, rows):
    """No estimate is made of no weights (0 / 0), and nothing is launched."""
    need, call = H.run(exe, [f"need 0 {k} {rows}", f"i8q 0 {k} {rows} {H.F32}"])
    bytes_, invalid = need[0].split()[1:]
    assert need[-1] == call[-1] == "rc 0" and not H.launches(call)
    assert int(bytes_) >= rows * (k + 4) and (int(bytes_) == 0) == (rows == 0)
    assert invalid == "0", "the host's arithmetic raised the invalid-operation flag"


def test_the_cases_of_the_device_tests_reach_every_kernel(exe):
    """test_gpu_int8_tiles.py's: each form of each kernel, in each output type, is launched by one of them."""
    from test_gpu_int8_tiles import CASES
    kernels = {line[len("kernel "):] for line in H.run(exe, ["kernels"])[0] if "syn::k_i8_" in line}
    assert sum("k_i8_gemm" in k for k in kernels) >= 64
    calls = [f"i8 {gated} {n} {k} {rows} {t} {t} {int(t == H.BF16)}" for gated, n, k, rows in CASES for t in (H.F32, H.F16, H.BF16)]
    calls += [f"i8quantize {k} {rows} {t}" for rows, k in ((257, 5001), (301, 9001)) for t in (H.F32, H.F16, H.BF16)]
    run = {name for answer in H.run(exe, calls) for *_, name in H.launches(answer)}
    assert kernels <= run, "not launched: " + ", ".join(sorted(kernels - run))
