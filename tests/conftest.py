import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")


# Files whose tests hand made-up pointers to entry points that have to refuse the call: where there is a GPU, a refusal that got
# lost would launch a kernel on them
MADE_UP_POINTERS = {"test_operator_refusals.py"}


def pytest_runtest_setup(item):
    if os.path.basename(str(item.fspath)) in MADE_UP_POINTERS:
        import torch
        if torch.cuda.device_count() > 0:
            pytest.skip("made-up pointers: only on a machine without a GPU")
