import os
import sys

import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")


# Tests whose expectation is wrong, and what takes their place. They stay as they are and are expected to fail.
_WRONG_EXPECTATIONS = {
    "test_gpu_lm_training.py::test_host_training_steps_with_muon":
        "scales a Linear's update by sqrt(max(1, in / out)): its weight is [in, out], and the factor is sqrt(max(1, out / in)); "
        "test_gpu_lm_training_edges.py::test_training_steps_with_muon holds the same run to that",
}


def pytest_collection_modifyitems(items):
    for item in items:
        for name, reason in _WRONG_EXPECTATIONS.items():
            if item.nodeid.endswith(name):
                item.add_marker(pytest.mark.xfail(reason=reason, strict=True))
