"""The language-model entry points without a GPU: what they refuse, under the host sanitizers, and what their workspace
queries answer."""
import os

import pytest

import nnh
from test_sanitize import _check, _run, built  # noqa: F401


def test_validation_under_address_and_ub_sanitizers(built):  # noqa: F811
    r = _run(os.path.join(built, "lm_sanitize"))
    if r.returncode == 77 or r.stdout.startswith("skipped"):
        pytest.skip(r.stdout.strip())
    _check(r, "every code as expected")


def test_workspace_queries():
    size = nnh.workspace_size
    # attention: a range of 12 bytes for each 64 tokens of either side (256-byte pieces); delta of the backward pass
    assert size("masked_attention", 1, 100, 100, 2, 2, 64, 0, 0) == 0
    assert size("masked_attention", 1, 100, 100, 2, 2, 64, 1, 0) == 512
    assert size("masked_attention", 2, 512, 512, 4, 4, 64, 0, 1) >= 2 * 4 * 512 * 4
    assert size("masked_attention", 0, 100, 100, 2, 2, 64, 1, 1) == 0
    # the split form's parts: 8192 keys in 32 of 256 at most, 64 rows of 130 floats
    assert size("masked_attention", 1, 1, 8192, 64, 8, 128, 0, 0) == 32 * 64 * 130 * 4
    # cross entropy: the forward keeps statistics, not scores; the one call keeps the scores where they fit
    rows, D, V = 8192, 4096, 128000
    scores = rows * V * 2
    assert size("linear_cross_entropy", nnh.BF16, rows, D, V, 0, 1) < scores // 20
    assert size("linear_cross_entropy", nnh.BF16, rows, D, V, 1, 1) < (1 << 30) + rows * D * 4 * 2
    assert scores < size("linear_cross_entropy", nnh.BF16, rows, D, V, 2, 1) < scores * 1.1
    assert size("linear_cross_entropy", nnh.BF16, 65536, D, V, 2, 1) < 5 << 30
    # rows that need a copy of the weight
    assert size("linear_cross_entropy", nnh.BF16, 64, 33, 5000, 0, 1) >= 5000 * 40 * 2


def test_options_are_checked_by_the_binding():
    torch = pytest.importorskip("torch")
    rule = nnh.AttentionRule(window=-1)
    with pytest.raises(nnh.NnhError):
        rule._struct(1, 1, 1, 1, 0)
    with pytest.raises(nnh.NnhError, match="device"):
        nnh._on(torch.zeros(3), 0)
    assert nnh._REDUCTIONS == {"none": 0, "mean": 1, "sum": 2}
