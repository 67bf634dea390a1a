"""The host code of the int8 products and of token_logprobs under AddressSanitizer and UndefinedBehaviorSanitizer
(CPU only): workspace sizes, the choice of a kernel and its launch over the ends of every size and type, each call
through to the launches that it makes, which host_launches.py's runtime writes down.  A report aborts the run."""
import itertools
import os
import shutil

import pytest

import host_launches as H
from syntropy_amd import build as B
from test_host_sanitizers import CLANG, ENV, SAN

pytestmark = pytest.mark.skipif(not (os.path.exists(B.HIPCC) and os.path.exists(CLANG)),
                                reason="needs hipcc and ROCm's clang++ with its sanitizer runtimes")

NS = (0, 1, 63, 5120, 14336, 1 << 23, (1 << 24) - 1, 1 << 24, (1 << 32) - 1)
KS = (0, 1, 4096, 16385, 131072, 131073, (1 << 32) - 1)
ROWS = (0, 1, 8, 9, 16, 17, 333, 2097120, 2097121, (1 << 32) - 1)


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("sanitized_int8"))
    B.build_host_sanitized(out)
    yield H.build(out, out, SAN)
    shutil.rmtree(out, ignore_errors=True)


def test_sizes_at_their_ends(exe):
    types = (H.F32, H.F16, H.BF16)
    calls = [f"i8 {g} {n} {k} {r} {types[i % 3]} {types[(i + g) % 3]} {i % 2}"
             for i, (n, k, r) in enumerate(itertools.product(NS, KS, ROWS)) for g in (0, 1)]
    calls += [f"{what} {n} {k} {r} {H.F32}" for what in ("i8q", "i8logits") for n, k, r in itertools.product(NS, KS, ROWS)]
    calls += [f"need {n} {k} {r}" for n, k, r in itertools.product(NS, KS, ROWS)]
    calls += [f"{what} {k} {r} {t}" for what in ("i8quantize", "i8act") for k, r, t in itertools.product(KS, ROWS, (*types, 2, 8))]
    calls += [f"logprobs {t} {r} {v} {top} {b}" for t, r, v, top, b in itertools.product(
        (*types, 2), (0, 1, 110, 111, 160, 161, 256, 257, 1025, (1 << 24) - 1, 1 << 24, (1 << 32) - 1),
        (0, 1, 64, 4097, 32769, 65537, 128256, 163841, 1 << 30, (1 << 30) + 1, (1 << 32) - 1), (0, 1, 64, 65), (4, 8, 2))]
    answers = H.run(exe, calls, dict(os.environ, **ENV))
    # what is within the header's limits is launched, and nothing else is
    for c, a in zip(calls, answers):
        what, *v = c.split()
        v = [int(t) for t in v]
        launched, ok = bool(H.launches(a)), a[-1] == "rc 0"
        assert ok or not launched, c
        if what == "i8":
            g, n, k, r = v[:4]
            fits = 1 <= k <= 131072 and n * (1 + g) < 1 << 24 and r <= 2097120
        elif what in ("i8q", "i8logits", "need"):
            n, k, r = v[:3]
            fits = 1 <= k <= (16384 if what == "i8logits" else 131072) and n < 1 << 24 and r <= 2097120
        elif what == "i8quantize":
            n, k, r = 1, v[0], v[1]
            fits = 1 <= k <= 131072 and r < 1 << 24 and (r == 0 or v[2] in types)
        elif what == "i8act":
            n, k, r = 1, v[0], v[1]
            fits = 1 <= k <= 131072 and r <= 2097120 and (r == 0 or v[2] in types)
        else:
            t, r, vocab, top, b = v
            n, fits = 1, t in types and r < 1 << 24 and 1 <= vocab <= 1 << 30 and top <= min(64, vocab) and b in (4, 8)
        assert ok == fits, f"{c}: {a[-1]}"
        assert launched == (fits and what != "need" and n > 0 and r > 0), c
