import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")


# Tests whose expected values are known to be wrong, with the reason; they still run, and have to fail.
WRONG_VALUES = {
    "test_gpu_orthogonalize.py::test_training_steps_under_every_evaluator":
        "its computation by hand multiplies muon's step by the root of inputs / outputs; the published factor is that of "
        "outputs / inputs, which test_gpu_muon.py expects of the same training",
}


def pytest_collection_modifyitems(items):
    for item in items:
        for name, reason in WRONG_VALUES.items():
            if item.nodeid.split("[")[0].endswith(name):
                item.add_marker(pytest.mark.xfail(reason=reason, strict=True))


@pytest.fixture(scope="session")
def oracle():
    from oracle import oracle as orc
    orc.build()
    return orc
