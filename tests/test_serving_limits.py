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


def test_places_of_the_line_of_sequences(lib):
    """A sequence of c rows takes ceil(c / 128) + 1 places of a line that 512 workgroups share; its length, rounded up to
    equal shares, has to stay below 2^31.  512 sequences of 2^22 - 2 units, 2^31 - 512 places, do not; 2^31 - 1536
    do.  (Past 2^31 the shares came out as one place each, and nearly all rows were left out.)"""
    ws = lib.lucid_decode_paged_workspace_bytes
    for units, ok in ((2 ** 22 - 2, False), (2 ** 22 - 3, False), (2 ** 22 - 4, True), (2 ** 21, True)):
        assert (ws(512, 2, 2, 1, 128, units, 64) > 0) == ok, units
    p, s, pool = ctypes.c_void_p(1 << 20), (ctypes.c_int64 * 3)(256, 64, 64), (ctypes.c_int64 * 3)(8192, 4096, 64)
    rc = lib.lucid_decode_paged(p, s, p, s, p, s, p, pool, p, pool, p, 8, p, p, s, p, p, 512, 2, 2, 1, 8, 128, 2 ** 22 - 2, 64,
                                0.125, 1e-5, None)
    assert rc == _lib.LUCID_EINVAL and b"2^38" in lib.lucid_last_error()
