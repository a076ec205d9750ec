import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

# Some tests pin a plan (tile rows, K slices, exact scaling) through the
# library's PW4_* plan overrides; the library reads them only when this is set
# before its first GEMM call in the process.
os.environ["PW4_PLAN_OVERRIDES"] = "1"


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (runs the HIP kernels)")


# Cases that hold a value which an operator's definition excludes, and where the right one is tested.
HOLDS_A_WRONG_VALUE = {
    "test_paged_append.py::test_blocks_of_every_kind[dtype1]":
        "bf16's greatest value, 1.99 * 2^127, is expected back as infinity; a finite block is held as something finite: "
        "test_fp4_magnitudes.py, which has this test's other blocks too",
}


def pytest_collection_modifyitems(config, items):
    import torch

    for item in items:
        reason = HOLDS_A_WRONG_VALUE.get(item.nodeid.split("/")[-1])
        if reason:
            item.add_marker(pytest.mark.xfail(reason=reason, strict=True))
    if torch.cuda.is_available():
        return
    skip = pytest.mark.skip(reason="needs a GPU")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)


@pytest.fixture(scope="session")
def orc():
    from oracle import oracle

    oracle.lib()
    return oracle
