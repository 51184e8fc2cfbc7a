"""Host programs over the language-model entry points (tests/cpp), without a GPU."""
import os

import pytest

from test_sanitize import _check, _run, built  # noqa: F401


@pytest.mark.parametrize("program,says", [("lm_empty_sanitize", "empty sides: "), ("lm_nomem", "without memory: "), ("lm_align_sanitize", "alignment: ")])
def test_program(built, program, says):  # noqa: F811
    r = _run(os.path.join(built, program))
    if r.returncode == 77:
        pytest.skip(r.stdout.strip())
    _check(r, says)
