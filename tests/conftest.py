import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")


def pytest_collection_modifyitems(config, items):
    import torch

    if torch.cuda.is_available():
        return
    skip = pytest.mark.skip(reason="no GPU in this container")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)


@pytest.fixture(autouse=True)
def _reload_library_env_after_the_test():
    """a test that flips a PGNN_* knob restores os.environ through monkeypatch; the library caches the values per call site, so it
    is told to look again AFTER monkeypatch's teardown (this fixture is set up first, hence torn down last) -- also when the test
    failed half way, so that one failure does not cascade into the tests behind it"""
    yield
    mod = sys.modules.get("pretrain_gnns_amd._lib")
    lib = getattr(mod, "_lib", None) if mod is not None else None
    if lib is not None:
        lib.pgnn_reload_env()


# Host results of the GPU tests: how torch cuts a sum into parts, and so its last bits, depends on the number of host threads.  With 6, 10, 12
# or 16 of them one fp32 BatchNorm pre-activation of those that are compared (3.8e-8 in 64 bits) falls on the other side of zero, and its
# ReLU's gradient with it; with 1 or 4 a sum over 5 000 rows is further from the 64-bit one than the GPU's may be from it.  With 8 every
# reference has the signs of 64 bits and is within two thirds of the tolerance (test_cpu_host_reference.py)
HOST_THREADS = 8


@pytest.fixture(autouse=True)
def _host_threads_of_gpu_tests(request):
    if "gpu" not in request.keywords:
        yield
        return
    import torch

    before = torch.get_num_threads()
    torch.set_num_threads(HOST_THREADS)
    yield
    torch.set_num_threads(before)
