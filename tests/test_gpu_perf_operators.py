"""The measured cases of perf/operators.py make their calls as a program has to."""
import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cases():
    path = Path(__file__).resolve().parent.parent / "perf" / "operators.py"
    spec = importlib.util.spec_from_file_location("perf_operators", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.own = True
    return m


def test_inputs_are_there_before_the_first_call(cases):
    """The library's stream is not torch's: nothing that torch computes for a call is pending
    when prepare() returns."""
    for case in cases.listed():
        for seed in (1, 2):
            cases.prepare(case, seed)
            assert torch.cuda.current_stream().query(), case["name"]
        torch.cuda.synchronize()
