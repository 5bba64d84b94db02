"""pytest configuration: the `gpu` marker and import paths.

Tests marked `gpu` need a visible HIP device and the built library
(diffuse-rs_amd/lib/libdr_attn.so); everything else runs on the CPU.
"""
import gc
import pathlib
import sys

ROOT = pathlib.Path(__file__).resolve().parent.parent
for p in (ROOT, ROOT / "diffuse-rs_amd", ROOT / "oracle", ROOT / "tests"):
    if str(p) not in sys.path:
        sys.path.insert(0, str(p))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a HIP GPU (MI355X) and the built library")


def pytest_collection_finish(session):
    """What the imports made stays for good: later collections pass over it."""
    gc.collect()
    gc.freeze()


def pytest_runtest_setup(item):
    """No test inherits garbage from the one before.  A torch.cuda.CUDAGraph that a
    reference cycle holds (a function's local, by way of a caught exception's
    traceback) is destroyed whenever the collector runs, and its destructor waits
    for the device: inside another test's stream capture that is an error, thrown
    in a destructor, and ends the process."""
    if item.get_closest_marker("gpu"):
        gc.collect()
