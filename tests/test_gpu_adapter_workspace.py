"""The workspace of q4k_linear_lora, each case in a process of its own
(adapter_child.py): a call that is refused for want of it has done nothing, gated
calls of few rows are captured after any first call, a slow rise of their rows
allocates seldom, and a call refused by the runtime does not fail the next."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.parametrize("case", ["refused", "captured", "growth", "errors"])
def test_adapter_workspace(case, gpu):
    env = {k: v for k, v in os.environ.items() if not k.startswith(("Q4K_", "Q6K_"))}
    r = subprocess.run([sys.executable, "-u", os.path.join(HERE, "adapter_child.py"), case], env=env, capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), f"{case} failed ({r.returncode}):\n{r.stdout[-1500:]}\n{r.stderr[-2000:]}"
