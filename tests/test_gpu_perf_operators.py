"""The measured cases of perf/operators.py make their calls as a program has to."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent

# torch brings a HIP runtime of its own, which has to be a process's first
PROGRAM = """
import importlib.util
import torch
spec = importlib.util.spec_from_file_location("perf_operators", "perf/operators.py")
cases = importlib.util.module_from_spec(spec)
spec.loader.exec_module(cases)
cases.own = True
assert torch.cuda.is_available()
for case in cases.listed():
    for seed in (1, 2):
        cases.prepare(case, seed)
        assert torch.cuda.current_stream().query(), case["name"]
    torch.cuda.synchronize()
    print("ready", case["name"], flush=True)
"""


def test_inputs_are_there_before_the_first_call():
    """The library's stream is not torch's: nothing that torch computes for a call is pending
    when prepare() returns."""
    p = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True,
                       timeout=110)
    assert p.returncode == 0, p.stdout[-500:] + p.stderr[-1500:]
    assert p.stdout.count("ready") == 12
