import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "xor-net_amd"), os.path.join(ROOT, "oracle")):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (runs libxtern kernels)")


# Tests that hold a wrong value, kept as they are: they have to fail.
WRONG = {
    "test_gpu_cache.py::test_evict_scores":
        "its plain form drops kept rows whose position 0..budget-1 has no page, and leaves evicted ones "
        "where a kept one has none; test_gpu_evict_holes.py::test_scores has these inputs and the definition",
}


def pytest_collection_modifyitems(items):
    for item in items:
        for name, why in WRONG.items():
            if item.nodeid.endswith(name):
                item.add_marker(pytest.mark.xfail(reason=why, strict=True))
