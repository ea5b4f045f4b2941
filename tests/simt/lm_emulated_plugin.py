"""Fixtures of the emulated runs (test_lm_operators_emulated.py)."""
import numpy as np
import pytest

@pytest.fixture(scope="session")
def api():
    from libgpuarray_b200 import api as a
    return a


@pytest.fixture(scope="session")
def ctx(api):
    return api.Context(0)


@pytest.fixture()
def rng():
    return np.random.default_rng(12345)
