"""The serving entry points without a GPU: what they refuse, under the host sanitizers and without memory, what their workspace queries
answer, and what the binding refuses itself."""
import os

import pytest

import nnh
from test_sanitize import _check, _run, built  # noqa: F401


@pytest.mark.parametrize("program,says", [("serving_sanitize", "every code as expected"), ("serving_nomem", "without memory: ")])
def test_program(built, program, says):  # noqa: F811
    r = _run(os.path.join(built, program))
    if r.returncode == 77:
        pytest.skip(r.stdout.strip())
    _check(r, says)


def test_workspace_queries():
    size = nnh.workspace_size
    # 8-bit linears: few rows are quantised where they are multiplied; else codes (a pitch of 64) and scales
    assert size("linear_int8", 1, 4096, 4096) == 0 and size("linear_int8", 16, 900, 4096) == 0
    assert size("linear_int8", 32, 4096, 16384) == 32 * 4096 + 256
    assert size("linear_int8", 0, 64, 64) == 0
    # sampling: a vocabulary that one workgroup holds needs none
    assert size("sample", nnh.F32, 300, 8192) == 0 and size("sample", nnh.BF16, 1, 1) == 0
    assert 0 < size("sample", nnh.F32, 1, 50257) < 1 << 20
    # attention: parts only where keys are divided
    assert size("paged_attention", 0, 0, 1, 4096, 8, 2, 64) == 0
    assert size("paged_attention", 1, 1, 1, 16, 8, 2, 64) == 0 or size("paged_attention", 1, 1, 1, 16, 8, 2, 64) < 1 << 20
    few, more = (size("paged_attention", 1, 1, 1, keys, 32, 8, 128) for keys in (4096, 32768))
    assert 0 < few <= more


def test_options_are_checked_by_the_binding(monkeypatch):
    torch = pytest.importorskip("torch")
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    z, i, u = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32), torch.zeros(2)
    starts, pages = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 4, 2, 8)
    codes, scale, cache = torch.zeros(3, 8, dtype=torch.int8), torch.zeros(3), nnh.PagedCache(pages, pages.clone(), i.view(2, 1))
    rule = nnh.AttentionRule(k_lens=i)
    for call in (lambda: nnh.sample(z, u), lambda: nnh.linear_int8(z, codes, scale), lambda: nnh.quantize_rows(z),
                 lambda: nnh.paged_append(cache, pages[0], pages[1], starts, i), lambda: nnh.paged_attention(pages[0], cache, starts, 1, rule)):
        with pytest.raises(nnh.NnhError, match="device"):
            call()
    for call in (lambda: nnh.sample(u, u), lambda: nnh.linear_int8(z[:, :5], codes, scale), lambda: nnh.quantize_rows(u),
                 lambda: nnh.paged_append(cache, z, z, starts, i), lambda: nnh.paged_attention(z, cache, starts, 1, rule),
                 lambda: nnh.PagedCache(pages, pages[:2], i.view(2, 1))._struct(0), lambda: nnh.PagedCache(pages, pages, i)._struct(0)):
        with pytest.raises(nnh.ShapeError):
            call()
    with pytest.raises(nnh.NnhError, match="consecutive"):
        nnh.sample(z.t().contiguous().t(), u)
    with pytest.raises(nnh.NnhError, match="strides"):
        nnh.PagedCache(pages, pages.transpose(1, 2).contiguous().transpose(1, 2), i.view(2, 1))._struct(0)
    with pytest.raises(nnh.NnhError, match="negative"):
        nnh.paged_attention(pages[0], cache, starts, -1, rule)
