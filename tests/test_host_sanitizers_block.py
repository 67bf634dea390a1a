"""The host code of the half-precision product, the norms between blocks and the sampling under AddressSanitizer and
UndefinedBehaviorSanitizer (CPU only): test_block_launches.py's calls at the ends of every size and type, each through
to the launches that it makes.  A report aborts the run."""
import os
import shutil

import pytest

from syntropy_amd import build as B
from test_block_launches import at_their_ends, program
from test_host_sanitizers import CLANG, ENV, SAN

pytestmark = pytest.mark.skipif(not (os.path.exists(B.HIPCC) and os.path.exists(CLANG)),
                                reason="needs hipcc and ROCm's clang++ with its sanitizer runtimes")


def test_sizes_at_their_ends(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("sanitized_block"))
    try:
        B.build_host_sanitized(out)
        at_their_ends(program(out, out, SAN), dict(os.environ, **ENV))
    finally:
        shutil.rmtree(out, ignore_errors=True)
