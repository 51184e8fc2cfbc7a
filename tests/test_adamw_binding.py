"""What nnh.AdamW hands to nnh_adamw_step when the caller's tensors change between steps, without a GPU: the library's call is
replaced by one that records its arguments (nothing is run, so host tensors stand in for device ones)."""
import pytest

import nnh

torch = pytest.importorskip("torch")


class Recorder:
    def __init__(self):
        self.calls = []

    def nnh_adamw_step(self, options, tensors, n, stream):
        o = options._obj
        self.calls.append((o.bits, [{k: getattr(tensors[i], k) for k, _ in tensors[i]._fields_} for i in range(n)]))
        return nnh.OK


@pytest.fixture
def calls(monkeypatch):
    rec = Recorder()
    monkeypatch.setattr(nnh, "lib", lambda: rec)
    monkeypatch.setattr(nnh, "_stream", lambda stream: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)  # what a host tensor's get_device() says
    return rec.calls


def made(bits=32, copies=False, sizes=(5, 130), **more):
    p, g = [torch.zeros(n) for n in sizes], [torch.ones(n) for n in sizes]
    c = [torch.zeros(n).bfloat16() for n in sizes] if copies else None
    return nnh.AdamW(p, g, bits=bits, copies=c, **more), p, g, c


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_uses_the_tensors_of_the_lists(calls, bits):
    opt, p, g, c = made(bits, copies=True)
    opt.step()
    _, rows = calls[-1]
    for i, row in enumerate(rows):
        want = {"p": p[i], "g": g[i], "m": opt.m[i], "v": opt.v[i], "copy": c[i], "m_scale": opt.m_scale[i], "v_scale": opt.v_scale[i]}
        assert row == {**{k: None if t is None else t.data_ptr() for k, t in want.items()}, "count": p[i].numel()}


@pytest.mark.parametrize("what", ["p", "g", "copy"])
@pytest.mark.parametrize("how", ["data", "item", "list"])
def test_a_step_follows_moved_tensors(calls, what, how):
    """New memory behind a tensor, another tensor in a list, another list: the next step has the new addresses."""
    opt, p, g, c = made(copies=True)
    opt.step()
    name = {"p": "params", "g": "grads", "copy": "copies"}[what]
    old = getattr(opt, name)
    new = torch.full_like(old[1], 3.0)
    if how == "data":
        old[1].data = new
    elif how == "item":
        old[1] = new
    else:
        setattr(opt, name, [old[0], new])
    opt.step()
    before, after = (call[1] for call in calls)
    assert after[1][what] == new.data_ptr() != before[1][what]
    assert {k: v for k, v in after[1].items() if k != what} == {k: v for k, v in before[1].items() if k != what}
    assert after[0] == before[0]
    assert opt.steps == 2


@pytest.mark.parametrize("change,error", [
    ("longer parameter", nnh.ShapeError), ("shorter parameter", nnh.ShapeError), ("shorter gradient", nnh.ShapeError),
    ("no gradient", nnh.NnhError), ("another type", nnh.NnhError), ("strided", nnh.NnhError),
    ("another device", nnh.NnhError), ("one more", nnh.ShapeError)])
def test_a_step_refuses_what_the_moments_are_not_for(calls, monkeypatch, change, error):
    opt, p, g, _ = made()
    opt.step()
    if change == "longer parameter":
        p[0].data, g[0].data = torch.zeros(9), torch.zeros(9)
    elif change == "shorter parameter":
        p[1].data, g[1].data = torch.zeros(64), torch.zeros(64)
    elif change == "shorter gradient":
        opt.grads[1] = torch.zeros(64)
    elif change == "no gradient":
        opt.grads[0] = None
    elif change == "another type":
        p[0].data = p[0].data.half()
    elif change == "strided":
        opt.grads[0] = torch.zeros(10)[::2]
    elif change == "another device":
        monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    else:
        opt.params.append(torch.zeros(3))
        opt.grads.append(torch.zeros(3))
    with pytest.raises(error):
        opt.step()
    assert len(calls) == 1 and opt.steps == 1


def test_the_moments_are_not_replaced_unnoticed(calls):
    opt, *_ = made(8)
    for name in ("m", "v", "m_scale", "v_scale", "bits"):
        with pytest.raises(AttributeError):
            setattr(opt, name, getattr(opt, name))
    with pytest.raises(TypeError):
        opt.m[0] = torch.zeros(5, dtype=torch.uint8)
    opt.step()
    assert calls[-1][0] == 8


def test_an_address_is_not_given_out_again_between_steps(calls):
    """The memory that the last step's table names is held: what else a tensor is given cannot lie there, or begin there and end
    sooner."""
    import weakref
    opt, p, g, _ = made()
    opt.step()
    before = [t.untyped_storage().data_ptr() for t in (p[0], g[0])]
    p[0].data, g[0].data = torch.zeros(9), torch.zeros(9)
    held = [t for t in opt._held if t.data_ptr() in before]
    assert len(held) == 2 and all(t.numel() == 5 for t in held)
    seen = [weakref.ref(t) for t in held]
    p[0].data, g[0].data = torch.zeros(5), torch.zeros(5)
    del held
    opt.step()
    assert all(r() is None for r in seen)  # and no longer


def test_tensors_from_iterators(calls):
    """model.parameters() and the like may be read once."""
    p, g = [torch.zeros(5), torch.zeros(70)], [torch.ones(5), torch.ones(70)]
    m, v = [torch.zeros(5), torch.zeros(70)], [torch.zeros(5), torch.zeros(70)]
    opt = nnh.AdamW(iter(p), (x for x in g), m=iter(m), v=iter(v))
    opt.step()
    assert [(r["p"], r["g"], r["m"], r["v"]) for r in calls[-1][1]] == [tuple(t.data_ptr() for t in row) for row in zip(p, g, m, v)]


def test_the_moments_memory_is_held(calls):
    """A step writes where the moments were made: that memory lives as long as the optimizer, whatever becomes of the tensors."""
    opt, *_ = made(8)
    opt.step()
    row = dict(calls[-1][1][1])
    for name in ("m", "v", "m_scale", "v_scale"):
        t = getattr(opt, name)[1]
        t.data = torch.zeros_like(t)
        assert row[name] != t.data_ptr() and row[name] in [x.data_ptr() for x in opt._kept]
    opt.step()
    assert calls[-1][1][1] == row
