import os
import sys

import pytest

# no MANO files in any test environment: HandNet(mano_root="misc/mano") falls back to the seeded synthetic model here only
os.environ.setdefault("OBMAN_MANO_SYNTHETIC", "1")
REPO = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
if REPO not in sys.path:
    sys.path.insert(0, REPO)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")


def pytest_collection_modifyitems(config, items):
    """GPU tests must FAIL (not skip) on a GPU box whose HIP library is missing; on a
    CPU-only box they are deselected by ``-m "not gpu"`` and skipped if selected anyway."""
    import torch

    # A pre-activation of this case is -1.2e-6 in 64 bits, a tenth of fp32's error there: its fp32 oracle takes the kernels' side of that ReLU on
    # some hosts and the other side on others.  tests/test_decoder_ties_gpu.py holds the kernels to the same bound with the tie taken care of.
    for item in items:
        if item.nodeid.endswith("test_decoder_gpu.py::test_decoder_forward_backward_matches_oracle[515-2-1-True-25]"):
            item.add_marker(pytest.mark.xfail(reason="the fp32 oracle meets a tie whose side depends on the host", raises=AssertionError, strict=False))
    if torch.cuda.is_available():
        return
    skip = pytest.mark.skip(reason="no GPU visible")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)


@pytest.fixture(scope="session")
def golden():
    import numpy as np

    from tests.golden.common import GOLDEN_DIR

    def _load(name):
        return np.load(os.path.join(GOLDEN_DIR, name + ".npz"), allow_pickle=False)

    return _load


def record_measurement(name, values):
    """Append measured parity errors to gpurun_out/parity_measured.jsonl (scratch; copied to profiles/ by hand) so that a
    tolerance can be frozen at a small multiple of what the hardware actually produced.  Never fails a test."""
    import json

    try:
        out = os.path.join(REPO, "gpurun_out")
        os.makedirs(out, exist_ok=True)
        with open(os.path.join(out, "parity_measured.jsonl"), "a") as fh:
            fh.write(json.dumps({"test": name, **values}) + "\n")
    except OSError:
        pass
