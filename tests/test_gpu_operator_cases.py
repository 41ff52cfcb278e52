"""The performance cases of the operators for a served batch (perf/operators.py), as a program would use them."""

import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["attention-8b-32", "adapter-8b-prompts", "verify-8b-32"])
def test_buffers_hold_their_values_before_a_pass(native_libs, name):
    """The package's stream is not ordered behind the one that fills them: nothing may be under way on it when a state is handed out."""
    import torch
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py")
    spec = importlib.util.spec_from_file_location("operators", path)
    operators = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(operators)
    operators.own = True
    case = next(c for c in operators.listed() if c["name"] == name)
    for seed in range(3):  # (the first one's work is mostly on the host)
        state = operators.prepare(case, seed)
        assert torch.cuda.current_stream().query()
        del state
    operators._backend.close()
