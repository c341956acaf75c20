"""The largest and smallest arguments of the serving operators, on the host (no GPU): what the kernels' arithmetic
holds is taken, the next value is refused."""
import ctypes

import pytest

from lucid_amd import _lib


@pytest.fixture(scope="module")
def lib():
    from lucid_amd import build
    import os
    if not all(os.path.exists(_lib.lib_path(n)) for n in build.TARGETS):
        build.build()
    return _lib.load()


def test_temperatures_whose_exponents_overflow(lib):
    """exp(x / t) is taken as exp2(x log2 e / t): at 1 / t = 2.5e38 the factor is 3.6e38, which fp32 does not hold, and
    0 times it made every maximum NaN."""
    p = ctypes.c_void_p(1 << 20)
    for rows in (0, 4):
        for fwd in (True, False):
            rc = (lib.lucid_token_logprobs_fwd(p, 0, 8, p, rows, 4, 8, 0, 4e-39, 2, p, p, p, p, p, p, None) if fwd else
                  lib.lucid_token_logprobs_bwd(p, 0, 8, p, rows, 4, 8, 0, 4e-39, 2, p, p, p, p, p, p, None))
            assert rc == _lib.LUCID_EINVAL and b"temperature" in lib.lucid_last_error()
        if rows == 0:
            assert lib.lucid_token_logprobs_fwd(p, 0, 8, p, rows, 4, 8, 0, 4.3e-39, 2, p, p, p, p, p, p, None) == 0
