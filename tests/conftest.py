import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
import pta_bootstrap  # noqa: E402

pta_bootstrap.load()
GOLDEN = os.path.join(ROOT, "tests", "golden")


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")


@pytest.fixture(scope="session")
def golden_dir():
    return GOLDEN


# The oracle's fp32 form depends on the host: on some CPUs its convolutions sum in an order in which an arg-max of the warp layer flips, and
# single gradients then lie up to 6.4e-2 of a tensor's largest value from the oracle's own 64-bit form (the device: 7e-5).  Tests of
# gradients through the warp layer that take the oracle's value as the reference get it evaluated in 64 bits, rounded once.
ORACLE_IN_64_BITS = {"test_generator_backward_vs_oracle"}


@pytest.fixture(autouse=True)
def _oracle_in_64_bits(request, monkeypatch):
    if request.node.name not in ORACLE_IN_64_BITS or not hasattr(request.module, "R"):
        return
    oracle = request.module.R
    forward = oracle.generator_forward

    def forward64(inp, warps, masks, params, pose_dim, enc, dec, size, drops=None, **kw):
        params = {k: v.double() for k, v in params.items()}
        drops = None if drops is None else [d.double() for d in drops]
        return forward(inp.double(), warps.double(), masks.double(), params, pose_dim, enc, dec, size, drops, **kw).float()

    monkeypatch.setattr(oracle, "generator_forward", forward64)


# PG_FORCE_REDUCER=1 (+ RANK/WORLD_SIZE/MASTER_* in the environment) runs the GPU suite with the data-parallel
# gradient reducer active at world size 1, so the bucketed RCCL all-reduce path is exercised on a single GPU.
if os.environ.get("PG_FORCE_REDUCER") == "1" and "RANK" in os.environ:
    from pose_transfer_amd.runtime import dp as _dp
    _dp.init_from_env()
