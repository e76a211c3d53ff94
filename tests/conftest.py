import gc
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a B200 (run with -m gpu on the GPU box)")


_by_exception = set()


@pytest.hookimpl(hookwrapper=True)
def pytest_runtest_makereport(item, call):
    """A test that ends by an exception (a skip in its body, a failure) leaves its frames, and the device memory of what they hold, in reference
    cycles: they go at once, not in the middle of a later test that compares the free device memory."""
    yield
    if call.excinfo is not None:
        _by_exception.add(item.nodeid)


@pytest.hookimpl(trylast=True)
def pytest_runtest_logfinish(nodeid, location):
    if nodeid in _by_exception:
        _by_exception.remove(nodeid)
        gc.collect()


@pytest.fixture(scope="session")
def pkg():
    import __graft_entry__ as entry
    return entry.load_package()


@pytest.fixture(scope="session", autouse=True)
def _oracle_built():
    from oracle import build_oracle
    build_oracle.build_restatements()
