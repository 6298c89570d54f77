import os
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

GOLDEN = os.path.join(ROOT, "tests", "golden")


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")


# Tests that hold a value shown to be wrong, kept as they were written: (file, test, the cases, why).  Strict: one that passes fails.
HELD_WRONG = [
    ("test_catalogue_paths_gpu.py", "test_engine_softmax_xent", ("both-50", "both-100"),
     "expects logits loss_gamma * <u, v> + cb; the engine's score is <u, v> + ub + cb (predict_scores) and loss_gamma scales all of it "
     "(log-loss): test_engine_head_gpu.py holds the head to predict_scores itself"),
]


def pytest_collection_modifyitems(items):
    for item in items:
        for path, name, cases, why in HELD_WRONG:
            if item.path.name == path and getattr(item, "originalname", None) == name and item.callspec.id in cases:
                item.add_marker(pytest.mark.xfail(reason=why, strict=True, raises=AssertionError))


@pytest.fixture(scope="session")
def sampler_golden():
    return np.load(os.path.join(GOLDEN, "sampler_golden.npz"))


@pytest.fixture(scope="session", autouse=True)
def _built():
    """Make sure libnncf_hip.so and the C oracle exist (hipcc cross-compiles without a GPU)."""
    import __graft_entry__ as g
    g.build(quiet=True)


def gpu_available():
    try:
        import torch
        return torch.cuda.is_available()
    except Exception:
        return False
