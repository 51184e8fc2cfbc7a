"""What nnh.masked_attention_forward and _backward hand to the library's calls, without a GPU: the calls are replaced by ones that
record their arguments (nothing is run, so host tensors stand in for device ones)."""
import pytest

import nnh

torch = pytest.importorskip("torch")
N, T, H, D = 2, 5, 2, 16


class Recorder:
    def __init__(self):
        self.refuse = False
        self.rest = []

    def _call(self, rest):
        if self.refuse:
            return nnh.ERR_ALIAS
        self.rest.append(None if rest is None else rest._obj.data)
        return nnh.OK

    def nnh_masked_attention_forward(self, *a):
        return self._call(a[12])

    def nnh_masked_attention_backward(self, *a):
        return self._call(a[12])

    def nnh_last_error(self):
        return b"refused"


@pytest.fixture
def library(monkeypatch):
    rec = Recorder()
    monkeypatch.setattr(nnh, "lib", lambda: rec)
    monkeypatch.setattr(nnh, "_stream", lambda stream: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)  # what a host tensor's get_device() says
    return rec


def inputs():
    return [torch.zeros(N, T, H, D, dtype=torch.bfloat16) for _ in range(4)]


def test_a_refused_call_leaves_the_rest(library):
    """lse still holds the last call's values, and so does its rest."""
    q, k, v, _ = inputs()
    out, lse = nnh.masked_attention_forward(q, k, v, nnh.AttentionRule())
    kept = lse.rest
    assert library.rest == [kept.data_ptr()]
    library.refuse = True
    for rest in (True, False):
        with pytest.raises(nnh.NnhError):
            nnh.masked_attention_forward(q, k, v, nnh.AttentionRule(), out=out, lse=lse, rest=rest)
        assert lse.rest is kept
    with pytest.raises(nnh.NnhError):  # refused before the library's call
        nnh.masked_attention_forward(q, k, v, nnh.AttentionRule(window=-1), out=out, lse=lse)
    assert lse.rest is kept
    library.refuse = False
    nnh.masked_attention_forward(q, k, v, nnh.AttentionRule(), out=out, lse=lse, rest=False)
    assert lse.rest is None


def test_the_rest_beside_a_copy_of_lse(library):
    """A copy, a view or a saved tensor has no attribute: the rest is then an argument of its own."""
    q, k, v, g = inputs()
    out, lse = nnh.masked_attention_forward(q, k, v, nnh.AttentionRule())
    other = torch.zeros_like(out)
    for given, rest, want in ((lse, None, lse.rest.data_ptr()), (lse.clone(), None, None), (lse.clone(), lse.rest, lse.rest.data_ptr()),
                              (lse.view(-1).view(N, H, T), other, other.data_ptr()), (lse, other, other.data_ptr()), (lse, False, None)):
        nnh.masked_attention_backward(g, q, k, v, out, given, nnh.AttentionRule(), rest=rest)
        assert library.rest[-1] == want
    with pytest.raises(nnh.ShapeError):
        nnh.masked_attention_backward(g, q, k, v, out, lse, nnh.AttentionRule(), rest=other[:1])
