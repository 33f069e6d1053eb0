"""The policy-table example runs the log-probability step, Muon and the scoring form together, and learns."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


def test_policy_table_learns():
    from plast_amd.examples.policy_table import STATES, train
    (lp0, hit0), (lp1, hit1) = train()
    assert lp1 > lp0 + 1.0 and hit1 > max(2 * hit0, STATES // 2), (lp0, hit0, lp1, hit1)
