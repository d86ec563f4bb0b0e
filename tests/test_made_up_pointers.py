"""CPU: tests that pass made-up pointers to the library do not run where a kernel could follow them."""
import os

import pytest
import torch

import conftest


class Item:
    def __init__(self, name):
        self.fspath = os.path.join("tests", name)


@pytest.mark.parametrize("gpus", [0, 1])
def test_made_up_pointers_stay_off_the_gpu(monkeypatch, gpus):
    monkeypatch.setattr(torch.cuda, "device_count", lambda: gpus)
    conftest.pytest_runtest_setup(Item("test_gpu_fp8.py"))
    for name in conftest.MADE_UP_POINTERS:
        assert os.path.exists(os.path.join(os.path.dirname(__file__), name))
        if gpus:
            with pytest.raises(pytest.skip.Exception):
                conftest.pytest_runtest_setup(Item(name))
        else:
            conftest.pytest_runtest_setup(Item(name))
