import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "tests")):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (run with -m gpu on a B200)")


# Cases that hold a wrong value and are kept as they were: they want outputs of zero for rows of positive weight outside every
# sequence, where the policy loss's definition (include/whirl_b200.h, perf/operators.py) has the row's own values.
# tests/test_gpu_losses_rows.py has the same calls with the right ones.
WRONG_VALUES = {f"test_policy[{shape}-2-{dtype}]" for dtype in ("f32", "bf16")
                for shape in ("17-1003-1-0", "40-4096-0-0", "24-33001-0-1", "9-151936-0-0", "5-262144-64-0")}


def pytest_collection_modifyitems(items):
    for item in items:
        if item.name in WRONG_VALUES and item.path.name == "test_gpu_losses.py":
            item.add_marker(pytest.mark.xfail(reason="wants zeros for rows outside every sequence", strict=True))


@pytest.fixture(scope="session")
def oracle():
    from oracle import oracle as orc
    return orc.Oracle()


@pytest.fixture(scope="session")
def reference():
    """The reference's own code (oracle/_ref); built when a reference checkout is present, else the test is skipped."""
    from oracle import oracle as orc
    try:
        path = orc.build_reference()
    except Exception:  # a checkout that does not build is reported by test_oracle_ref.py, not here
        path = None
    if not path:
        pytest.skip("oracle/_ref not built (no reference checkout on this machine)")
    return orc.Reference(path)


@pytest.fixture(scope="session")
def golden():
    import json
    import numpy as np
    g = os.path.join(ROOT, "tests", "golden")

    class G:
        def npz(self, name):
            return np.load(os.path.join(g, name + ".npz"))

        def json(self, name):
            with open(os.path.join(g, name + ".json")) as f:
                return json.load(f)
    return G()
