"""Shared fixtures.  GPU tests are marked ``gpu``; everything else runs on CPU."""
from __future__ import annotations

import os
import sys
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a B200 (runs the CUDA library)")
    config.addinivalue_line("markers", "slow: long-running")


def pytest_collection_modifyitems(items):
    """test_evict's reference ranks protected rows by their row alone.  The header, and the
    operator's plain form, rank them by weight, then row: of five protected rows with
    weights 5, 1, 9, 2, 7 the two that stay are 2 and 4, not 0 and 1.  Where more rows are
    protected than stay and their weights differ, its expected rows are wrong;
    test_evict_in_documented_order has the same cases with the documented order."""
    for item in items:
        if getattr(item, "originalname", "") == "test_evict":
            p = item.callspec.params
            if p["kind"] != "equal" and p["n"] > max(2, p["keep"]):
                item.add_marker(pytest.mark.xfail(strict=True, reason="expects protected rows ranked by row, not by weight"))


@pytest.fixture(scope="session")
def oracle():
    from oracle.oracle import Oracle
    return Oracle()


@pytest.fixture(scope="session")
def ref_strict():
    from oracle.oracle import REF_STRICT_SO, RefLib
    if not REF_STRICT_SO.exists():
        pytest.skip("reference library not built here (oracle/_ref)")
    return RefLib(REF_STRICT_SO)


@pytest.fixture(scope="session")
def ref_native():
    from oracle.oracle import REF_NATIVE_SO, RefLib
    if not REF_NATIVE_SO.exists():
        pytest.skip("reference library not built here (oracle/_ref)")
    return RefLib(REF_NATIVE_SO)


@pytest.fixture(scope="session")
def gpu():
    """The CUDA library bound to torch's current stream (fails loudly without it)."""
    import torch
    if not torch.cuda.is_available():
        pytest.fail("GPU test selected but no CUDA device is visible")
    from gncx_b200 import core
    lib = core.load()
    torch.cuda.init()
    lib.gncx_set_synchronous(1)
    core.bind_torch_stream(lib)
    return lib


def golden(name: str) -> dict:
    with np.load(ROOT / "tests" / "golden" / name, allow_pickle=False) as z:
        return {k: z[k] for k in z.files}
