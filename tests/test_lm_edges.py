"""The C++ layer's language-model operators (include/nn_hip_modules.hpp) where something changes between two calls."""
import ctypes as C
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
HARNESS = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "lib", "liblm_edges_harness.so")


@pytest.fixture(scope="module")
def harness(gpu):
    if not os.path.exists(HARNESS):
        pytest.fail(f"{HARNESS} missing: build it with `make -C tests/cpp` (or __graft_entry__.build())")
    lib = C.CDLL(HARNESS)
    lib.edges_last_error.restype = C.c_char_p
    return lib


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("change,code", [(0, 0), (1, 1), (2, 2), (3, 2)])
def test_adamw_refuses_what_its_moments_do_not_fit(harness, bits, change, code):
    """The moments keep the kind and sizes they were made with: a step after a change of either is refused, nothing written."""
    n = 200
    p, steps = np.zeros(n, np.float32), C.c_size_t(0)
    rc = harness.edges_adamw_changed(C.c_size_t(n), bits, change, p.ctypes.data_as(C.c_void_p), C.byref(steps))
    assert rc == code, harness.edges_last_error().decode()
    assert steps.value == (2 if change == 0 else 1)
    # a constant gradient's steps are lr each, m / sqrt(v) being 1 after the corrections. p near 1 rounds by 2^-24 a step, 1.2e-4
    # of the step; in 8 bits the second step takes a moment and a root each off by 2^-4 at most: (17/16) / (15/16) - 1 of half
    size = 1.0 - (1 - 1e-3 * 0.01) ** steps.value + 1e-3 * steps.value
    np.testing.assert_allclose(1.0 - p, size, rtol=1e-3 if bits == 32 else 0.07)
