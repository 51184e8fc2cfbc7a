"""The C++ layer's language-model operators (include/nn_hip_modules.hpp) where something changes between two calls."""
import ctypes as C
import os

import numpy as np
import pytest
import torch

from lm_reference import assert_within, linear_cross_entropy

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


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("add", [0, 1])
def test_one_node_given_twice_to_the_loss(harness, which, add):
    """x that is the weight or the bias too gets the sum of both gradients, in one buffer."""
    V, D = (30, 24) if which != 1 else (24, 24)
    rng = np.random.default_rng(which)
    rows = 1 if which == 1 else V
    x = rng.standard_normal((rows, D)).astype(np.float32)
    w = x if which == 0 else rng.standard_normal((V, D)).astype(np.float32)
    b = x[0] if which == 1 else rng.standard_normal(V).astype(np.float32)
    y = rng.integers(0, V, rows).astype(np.int32)
    loss, dx, dw, db = np.zeros(1, np.float32), np.zeros_like(x), np.zeros_like(w), np.zeros_like(b)
    at = lambda a: a.ctypes.data_as(C.c_void_p)  # noqa: E731
    rc = harness.edges_loss_shared(which, add, C.c_size_t(V), C.c_size_t(D), at(x), at(w), at(b), at(y), at(loss), at(dx), at(dw), at(db))
    assert rc == 0, harness.edges_last_error().decode()
    want = linear_cross_entropy(*(torch.from_numpy(a) for a in (x, w, y, b)))
    u = 2.0 ** -24
    both = lambda *names: tuple(sum(want[n][i].view_as(want[names[0]][i]) for n in names) for i in (0, 1))  # noqa: E731
    pairs = [(dx, both("dx", "dw") if which == 0 else both("dx", "db") if which == 1 else want["dx"])]
    pairs += [(dw, want["dw"])] * (which != 0) + [(db, want["db"])] * (which != 1)
    for got, (value, bound) in pairs:
        value = value + add
        # the additions to what a buffer holds: two at most, half a step each
        assert_within(torch.from_numpy(got), (value, bound + 3 * u * (value.abs() + 1 + bound)), which)
    assert_within(torch.from_numpy(loss)[0], want["loss"], "loss")
