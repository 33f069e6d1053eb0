"""A Newton-Schulz rule's range is worked out once, also where calls with several rules take turns. On the CPU: rules
are checked before anything else."""
from __future__ import annotations

import ctypes as C
import time

import pytest

from plast_amd import abi
from plast_amd.runtime import LIB_PATH, Library, PlastHipError

pytestmark = pytest.mark.skipif(not LIB_PATH.exists(), reason="the library is not built")


def test_rules_that_take_turns():
    lib = Library()
    lib.plast_hip_clear_error()

    def call(rule):
        begin = time.perf_counter()
        lib.newton_schulz_hip(None, None, C.byref(rule))
        took = time.perf_counter() - begin
        with pytest.raises(PlastHipError, match="g must be"):
            lib.check()
        return took

    rules = [abi.NewtonSchulz(1.5 + 0.01 * k, -0.5 - 0.01 * k, 0.0, 1e-7, 1000) for k in range(6)]
    first = min(call(r) for r in rules)              # 1000 steps from 4097 values: milliseconds
    again = [call(r) for _ in range(5) for r in rules]
    assert sorted(again)[len(again) // 2] < first / 5, (first, again)
