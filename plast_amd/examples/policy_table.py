"""Policy gradient with an entropy bonus on a table of logits: the token log-probability step gives the
table's gradient in one pass, Muon updates the table, and the scoring form reports what it has learnt.

    python -m plast_amd.examples.policy_table [steps]

Each of the table's rows is a state, each column an action, and one action of a state is rewarded. A step
draws an action in every state, takes the advantage A over the mean reward, and descends
-(A log p[action] + bonus H) / states.
"""
from __future__ import annotations

import ctypes as C
import sys

import numpy as np

from plast_amd import abi, ops
from plast_amd.runtime import DeviceTensor, lib

STATES, ACTIONS, BONUS = 512, 24, 0.01


def _upload(t: DeviceTensor, values: np.ndarray) -> None:
    values = np.ascontiguousarray(values)
    lib().arena_memcpy_h2d_hip(t.ptr, values.ctypes.data, values.nbytes)
    lib().check("upload")


def train(steps: int = 150, seed: int = 0):
    """The mean log-probability of the rewarded actions before and after, and how many states have theirs
    first among the alternatives."""
    L = lib()
    rng = np.random.RandomState(seed)
    best = rng.randint(0, ACTIONS, STATES).astype(np.int32)
    table = DeviceTensor.from_numpy((0.01 * rng.randn(STATES, ACTIONS)).astype(np.float32), requires_grad=True)
    goal = DeviceTensor.from_numpy(best)
    tokens = DeviceTensor((STATES,), abi.INT32)
    dlogp, dentropy = DeviceTensor((STATES,)), DeviceTensor((STATES,))
    logp, entropy = DeviceTensor((STATES,)), DeviceTensor((STATES,))
    _upload(dentropy, np.full(STATES, -BONUS / STATES, np.float32))
    params, keep = abi.tensor_array(table.t)
    muon = abi.Muon(lr=0.4, momentum=0.9, weight_decay=0.0, nesterov=1,
                    rule=abi.NewtonSchulz(3.4445, -4.7750, 2.0315, 1e-7, 5), m=None)

    def score():
        inputs, lp, _ = ops.token_logprob(table, goal, top=1)
        return float(lp.numpy().mean()), int((inputs[5].numpy()[:, 0] == best).sum())

    before = score()
    step = [C.byref(t.t) for t in (table, tokens, dlogp, dentropy, logp, entropy, table.grad)]
    for _ in range(steps):
        # the largest logit plus Gumbel noise is a draw from the softmax
        drawn = (table.numpy() + rng.gumbel(size=(STATES, ACTIONS))).argmax(1).astype(np.int32)
        reward = (drawn == best).astype(np.float32)
        _upload(tokens, drawn)
        _upload(dlogp, -(reward - reward.mean()) / STATES)
        L.token_logprob_step_hip(*step, 1.0)
        L.check("token_logprob_step")
        L.muon_step_hip(C.byref(muon), params, 1)
        L.check("muon_step")
    after = score()
    L.plast_hip_muon_release(C.byref(muon), 1)
    return before, after


if __name__ == "__main__":
    (lp0, hit0), (lp1, hit1) = train(int(sys.argv[1]) if len(sys.argv) > 1 else 150)
    print(f"log p of the rewarded action: {lp0:.3f} -> {lp1:.3f}; first among the alternatives in {hit0} -> "
          f"{hit1} of {STATES} states")
