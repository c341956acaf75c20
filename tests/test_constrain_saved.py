"""The backward of constraints without a history takes no logits: what the C entry point asks for (no GPU)."""
import ctypes

import pytest

from test_prompt_args import PTR, _err, lib  # noqa: F401


def _bwd(lib, x, N, **kw):
    a = dict(hist=PTR if N else None, out=None, dtype=0, sb=0, st=100)
    a.update(kw)
    return lib.lucid_constrain_logits_bwd(x, a["sb"], a["st"], 2, 1, 100, a["dtype"], a["hist"], 8, N, None, 1.2, PTR, 4, PTR, a["out"], None)


def test_logits_are_asked_for_behind_a_history_alone(lib):  # noqa: F811
    _err(lib, _bwd(lib, None, 8), b"logits are null")
    _err(lib, _bwd(lib, None, 0), b"null argument")  # the missing output: what is checked behind the logits
    odd = ctypes.c_void_p((1 << 20) + 1)
    for N in (0, 8):
        _err(lib, _bwd(lib, odd, N), b"misaligned")


def test_the_forward_always_takes_logits(lib):  # noqa: F811
    rc = lib.lucid_constrain_logits(None, 0, 100, 2, 1, 100, 0, None, 0, 0, None, None, 1.0, None, 0.0, None, 0.0, None, 0, PTR, 4, PTR, None)
    _err(lib, rc, b"logits are null")


@pytest.mark.parametrize("sb,st", [(-1, 100), (0, -1)])
def test_strides_are_checked_without_logits_too(lib, sb, st):  # noqa: F811
    _err(lib, _bwd(lib, None, 0, sb=sb, st=st), b"negative strides")
