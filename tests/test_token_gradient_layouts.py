"""Which layouts of the logits' gradient the token log-probability entry points refuse, on the CPU: rows that share
addresses, along one leading axis or between several, and rows that leave their last workgroup no 31-bit numbers."""
from __future__ import annotations

import ctypes as C

import pytest

from plast_amd.abi import INT32, KernelParams
from plast_amd.runtime import LIB_PATH, Library, PlastHipError
from test_operator_refusals import T

pytestmark = pytest.mark.skipif(not LIB_PATH.exists(), reason="the library is not built")


@pytest.mark.parametrize("strides", [
    (10, 10, 1),      # both axes step a row: (0, 1) and (1, 0) are the same rows
    (20, 10, 1),      # three rows of 10, every 20
    (0, 10, 1),
    (29, 10, 1),      # a row's last logit is the next group's first
    (10, 15, 1),
    (-10 % 2 ** 64, 10, 1),
], ids=str)
def test_rows_that_share_addresses(strides):
    lib = Library()
    lib.plast_hip_clear_error()
    x = T((2, 3, 10), grad=T((2, 3, 10), strides=strides))
    vec, logp = [T((6,), INT32), T((6, 2)), T((6,))], T((6,))
    ins = (C.c_void_p * 4)(*[C.addressof(t) for t in [x, *vec]])
    lib.by_address["backward", "token_logprob"](ins, C.addressof(logp), KernelParams(0, 1, 1.0))
    with pytest.raises(PlastHipError, match="overlap"):
        lib.check()
    step = [x, vec[0], None, None, logp, vec[2], x.grad.contents]
    lib.token_logprob_step_hip(*[C.addressof(t) if t is not None else None for t in step], 1.0)
    with pytest.raises(PlastHipError, match="overlap"):
        lib.check()


@pytest.mark.parametrize("vocab", [2 ** 31 - 64, 2 ** 31 - 8191])
def test_rows_that_are_too_long(vocab):
    lib = Library()
    lib.plast_hip_clear_error()
    x, vec = T((1, vocab), grad=T((1, vocab))), [T((1,), INT32), T((1, 2)), T((1,))]
    logp = T((1,))
    ins = (C.c_void_p * 4)(*[C.addressof(t) for t in [x, *vec]])
    lib.by_address["backward", "token_logprob"](ins, C.addressof(logp), KernelParams(0, 1, 1.0))
    with pytest.raises(PlastHipError, match="logits are not supported"):
        lib.check()
