"""A GPU test starts without garbage of the test before it (tests/conftest.py).  CPU only."""
from __future__ import annotations

import gc
import weakref

import pytest

import conftest


class Local:
    """Stands for a graph in a test's local."""


class Item:
    def __init__(self, gpu):
        self.gpu = gpu

    def get_closest_marker(self, name):
        return self.gpu if name == "gpu" else None


def leave_garbage():
    """A caught exception's traceback holds this frame, and the frame the exception."""
    held = Local()
    with pytest.raises(ValueError) as e:
        raise ValueError
    assert e.value is not None
    return weakref.ref(held)


@pytest.mark.parametrize("gpu", [True, False])
def test_garbage_of_the_last_test(gpu):
    gc.disable()
    try:
        ref = leave_garbage()
        assert ref() is not None  # only the collector can free it
        conftest.pytest_runtest_setup(Item(gpu))
        assert (ref() is None) == gpu
    finally:
        gc.enable()
        gc.collect()
