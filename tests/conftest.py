import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (runs through the HIP C-ABI)")


@pytest.fixture(scope="session")
def oracle():
    from oracle import oracle as o
    o.lib()
    return o


# Their reference takes x - (m + log sum exp(x - m)), where m + log is m alone from |m| = 2^53 log on: of V equal logits of
# 1e30, or of the type's lowest value, each then has a log-probability of 0, not of -log V (V probabilities of 1).
# tests/test_beam_far_logits.py has the same rows with the values that log-softmax gives.
WRONG_VALUES = ("test_encoder_decoder.py::test_selection_of_extreme_logits",
                "test_encoder_decoder.py::test_selection_under_masks_of_the_lowest_value")


def pytest_collection_modifyitems(items):
    for item in items:
        if item.nodeid.split("[")[0].endswith(WRONG_VALUES):
            item.add_marker(pytest.mark.xfail(strict=True, raises=AssertionError,
                                              reason="expects a log-probability of 0 for each of several equal logits"))
