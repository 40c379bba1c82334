"""What a vocabulary loss call plans before the device is touched: runs anywhere."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

FIRST_SIZES = """
from caffecontroll_amd import _lib
from caffecontroll_amd.driver import BF16, HIPDriver, vocab_loss_args
d = HIPDriver.__new__(HIPDriver)
d.lib = _lib.load()
args = vocab_loss_args(1023, 1000, 50021, BF16)
sizes = lambda: (d.vocab_loss_workspace_bytes(args, training=False), d.vocab_loss_workspace_bytes(args))
print(*sizes())
d.lib.cct_hip_set_tuning(b"%s", %d)
print(*sizes())
d.lib.cct_hip_set_tuning(b"%s", 0)
print(*sizes())
"""


@pytest.mark.parametrize("knob, value", [("vocab_tile", 3), ("vocab_keep", 1)])
def test_the_environment_s_knobs_count_from_the_first_workspace_size_on(knob, value):
    """A program asks for the workspace before its first call selects a device: the size has to be the one that the call
    then finds necessary."""
    env = dict(os.environ, **{"CCT_HIP_" + knob.upper(): str(value)})
    out = subprocess.run([sys.executable, "-c", FIRST_SIZES % (knob, value, knob)], cwd=ROOT, env=env, check=True,
                         capture_output=True, text=True, timeout=120).stdout.split("\n")
    first, pinned, free = out[:3]
    assert first == pinned != free
