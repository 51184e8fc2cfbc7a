"""Masked attention (nnh_masked_attention_*) on the GPU against the formula in 64 bits, within the bounds of its roundings."""
import math

import pytest
import torch

from lm_reference import assert_within, masked_attention

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "bf16": torch.bfloat16}


def draw(seed, *shape, dtype=torch.float32, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * scale).to(dtype)


def documents(N, length, seed):
    """Runs of tokens of one document, some that belong to none."""
    gen = torch.Generator().manual_seed(seed)
    cuts = (torch.rand(N, length, generator=gen) < 4.0 / max(4, length)).int().cumsum(1)
    return torch.where(torch.rand(N, length, generator=gen) < 0.05, -1, cuts).int()


def run(q, k, v, g=None, **opts):
    import nnh
    dev = lambda x: x.cuda() if isinstance(x, torch.Tensor) else x  # noqa: E731
    rule = nnh.AttentionRule(**{n: dev(x) for n, x in opts.items()})
    q, k, v = q.cuda(), k.cuda(), v.cuda()
    out, lse = nnh.masked_attention_forward(q, k, v, rule)
    got = {"out": out, "lse": lse}
    if g is not None:
        got.update(zip(("dq", "dk", "dv"), nnh.masked_attention_backward(g.cuda(), q, k, v, out, lse, rule)))
    torch.cuda.synchronize()
    return got


def check(dtype, N, Tq, Tk, H, Hkv, D, train=True, seed=0, scale_q=1.0, **opts):
    t = T[dtype]
    print(dtype, N, Tq, Tk, H, Hkv, D, train, {n: x if not isinstance(x, torch.Tensor) else "given" for n, x in opts.items()}, flush=True)
    q, k, v = draw(seed, N, Tq, H, D, dtype=t, scale=scale_q), draw(seed + 1, N, Tk, Hkv, D, dtype=t), draw(seed + 2, N, Tk, Hkv, D, dtype=t)
    g = draw(seed + 3, N, Tq, H, D, dtype=t) if train else None
    want = masked_attention(q, k, v, g, **opts)
    got = run(q, k, v, g, **opts)
    assert set(got) == set(want)
    for name in want:
        assert_within(got[name], want[name], name)


SHAPES = [(1, 1, 1, 1, 1, 8), (2, 33, 33, 4, 2, 64), (1, 64, 64, 2, 2, 128), (2, 40, 70, 4, 1, 80), (1, 129, 257, 2, 1, 96), (3, 100, 31, 3, 3, 40),
          (1, 200, 200, 6, 2, 20), (1, 65, 130, 2, 2, 13), (1, 130, 65, 1, 1, 1), (1, 300, 300, 1, 1, 128)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("causal", [False, True])
def test_shapes(gpu, dtype, shape, causal):
    check(dtype, *shape, causal=causal)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["cap", "slopes", "window", "window_only", "prefix", "lens", "docs", "all", "scale"])
def test_rules(gpu, dtype, kind):
    N, L, H, Hkv, D = 3, 190, 4, 2, 64
    o = {"causal": kind != "window_only"}
    every = kind == "all"
    if kind == "cap" or every:
        o["cap"] = 5.0
    if kind == "slopes" or every:
        o["slopes"] = torch.exp2(-torch.arange(1.0, H + 1))
    if kind in ("window", "window_only") or every:
        o["window"] = 37
    if kind == "prefix" or every:
        o["prefix"] = torch.tensor([0, 70, 500], dtype=torch.int32)
    if kind == "lens" or every:
        o["k_lens"] = torch.tensor([190, 0, 65], dtype=torch.int32)
    if kind == "docs" or every:
        o["q_docs"] = o["k_docs"] = documents(N, L, 5)
    if kind == "scale":
        o["scale"] = 0.37
    check(dtype, N, L, L, H, Hkv, D, scale_q=2.0, **o)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_documents_of_their_own(gpu, dtype):
    """Queries and keys of different lengths and unsorted documents, some of one side alone; a document of one token; no
    token of any document."""
    gen = torch.Generator().manual_seed(3)
    qd, kd = torch.randint(-1, 4, (2, 150), generator=gen).int(), torch.randint(-1, 5, (2, 210), generator=gen).int()
    check(dtype, 2, 150, 210, 2, 1, 64, q_docs=qd, k_docs=kd)
    check(dtype, 2, 150, 210, 2, 1, 64, q_docs=torch.full_like(qd, -1), k_docs=kd)
    one = torch.arange(150).int().repeat(2, 1)
    check(dtype, 2, 150, 150, 2, 1, 64, q_docs=one, k_docs=one, causal=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tq", [1, 2, 5, 31, 32])
@pytest.mark.parametrize("heads", [(1, 1), (8, 8), (8, 2), (40, 1)])
def test_single_tokens(gpu, dtype, tq, heads):
    """Queries at the end of a cache; the cache's unused rows hold NaN."""
    import nnh
    N, Tk, D = 3, 777, 64
    lens = torch.tensor([777, tq, 130], dtype=torch.int32)
    t = T[dtype]
    q, k, v = draw(1, N, tq, heads[0], D, dtype=t), draw(2, N, Tk, heads[1], D, dtype=t), draw(3, N, Tk, heads[1], D, dtype=t)
    for n in range(N):
        k[n, lens[n]:] = math.nan
        v[n, lens[n]:] = math.nan
    o = dict(causal=True, k_lens=lens, q_start=lens - tq, cap=20.0)
    want = masked_attention(q, k, v, **o)
    got = run(q, k, v, **o)
    for name in want:
        assert_within(got[name], want[name], name)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tk", [0, 1, 255, 256, 511, 4096, 20000])
@pytest.mark.parametrize("D", [32, 80, 128, 30])
def test_cache_lengths(gpu, dtype, tk, D):
    check(dtype, 2, 1, tk, 4, 2, D, train=False, k_lens=torch.tensor([tk, max(0, tk - 300)], dtype=torch.int32))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_window_in_a_cache(gpu, dtype):
    lens = torch.tensor([3000, 700], dtype=torch.int32)
    check(dtype, 2, 3, 3000, 4, 2, 64, train=False, causal=True, window=100, k_lens=lens, q_start=lens - 3, slopes=torch.tensor([0.5, 0.1, 0.01, 0.0]))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_seen_does_not_matter(gpu, dtype, bad):
    """Two documents in one tile; values of one that are not finite stay out of the other's results and gradients, and
    masked rows (no document) may hold anything."""
    t = T[dtype]
    N, L, H, D = 1, 150, 2, 64
    docs = torch.zeros(N, L, dtype=torch.int32)
    docs[:, 70:120] = 1
    docs[:, 120:] = -1
    q, k, v, g = (draw(s, N, L, H, D, dtype=t) for s in range(4))
    o = dict(causal=True, q_docs=docs, k_docs=docs)
    clean = masked_attention(q, k, v, g, **o)
    for x in (q, k, v, g):
        x[:, 120:] = bad
        x[:, 75, :, 5] = bad
    got = run(q, k, v, g, **o)
    for name, (value, bound) in clean.items():
        cut = (slice(None), slice(None), slice(0, 70)) if name == "lse" else (slice(None), slice(0, 70))
        assert_within(got[name][cut], (value[cut], bound[cut]), name)
        tail = got[name][:, :, 120:] if name == "lse" else got[name][:, 120:]
        assert bool((tail == (-math.inf if name == "lse" else 0.0)).all()), name
    # a value that is not finite makes exactly the queries that see it so
    fine = torch.isfinite(got["out"].float()[0, 70:120, 0, 5]).cpu()
    assert bool(fine[:5].all()) and not bool(fine[5:].any())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_accumulation(gpu, dtype):
    """q, k and v beside each other in one buffer, their gradients in another; heads before tokens; rows of odd strides; one
    key sequence shared by the batch (stride 0); gradients added to what is there."""
    import nnh
    t = T[dtype]
    N, L, H, Hkv, D = 2, 90, 4, 2, 32
    rule = nnh.AttentionRule(causal=True)
    qkv = draw(0, N, L, (H + 2 * Hkv), D, dtype=t).cuda()
    cut = lambda x: (x[:, :, :H], x[:, :, H:H + Hkv], x[:, :, H + Hkv:])  # noqa: E731
    q, k, v = cut(qkv)
    g = draw(1, N, L, H, D, dtype=t).cuda()
    want = masked_attention(q, k, v, g, causal=True)
    out, lse = nnh.masked_attention_forward(q, k, v, rule)
    grads = torch.full_like(qkv, math.nan)
    nnh.masked_attention_backward(g, q, k, v, out, lse, rule, *(x for part in cut(grads) for x in (part, True)))
    for name, part in zip(("dq", "dk", "dv"), cut(grads)):
        assert_within(part, want[name], name)
    old = draw(2, *grads.shape, dtype=t).cuda()
    total = old.clone()
    nnh.masked_attention_backward(g, q, k, v, out, lse, rule, *(x for part in cut(total) for x in (part, False)))
    for name, part, was in zip(("dq", "dk", "dv"), cut(total), cut(old)):
        value, bound = want[name]
        was = was.double().cpu()
        u = torch.finfo(t).eps / 2
        assert_within(part, (value + was, bound + u * (value + was).abs() + u * bound), name)
    # heads before tokens, and rows of an odd stride (elements loaded one by one)
    for pad in (0, 1):
        wide = [torch.zeros(N, x.shape[2], L, D + pad, dtype=t, device="cuda") for x in (q, k, v)]
        views = [w[..., :D].transpose(1, 2) for w in wide]
        for view, x in zip(views, (q, k, v)):
            view.copy_(x)
        out2, lse2 = nnh.masked_attention_forward(*views, rule)
        assert_within(out2, want["out"], "out")
        for name, x in zip(("dq", "dk", "dv"), nnh.masked_attention_backward(g, *views, out2, lse2, rule)):
            assert_within(x, want[name], name)
    shared = [x[:1].expand(N, -1, -1, -1) for x in (k, v)]
    want = masked_attention(q, *shared, causal=True)
    assert_within(nnh.masked_attention_forward(q, *shared, rule)[0], want["out"], "shared")
    with pytest.raises(nnh.NnhError, match="overlap"):
        one = torch.empty(1, L, Hkv, D, dtype=t, device="cuda").expand(N, -1, -1, -1)
        nnh.masked_attention_backward(g, q, k, v, out, lse, rule, dk=one)


def test_gradient_against_differences(gpu):
    """The gradient of sum(g out) along random directions against central differences of the 64-bit form."""
    o = dict(causal=True, cap=3.0, slopes=torch.tensor([0.3, 0.05]))
    q, k, v, g = (draw(s, 1, 20, 2, 16) for s in range(4))
    got = run(q, k, v, g, **o)
    f = lambda a, b, c: float((masked_attention(a, b, c, **o)["out"][0] * g.double()).sum())  # noqa: E731
    h = 1e-4
    for n, name in enumerate(("dq", "dk", "dv")):
        d = draw(10 + n, 1, 20, 2, 16).double()
        x = [q.double(), k.double(), v.double()]
        up, down = list(x), list(x)
        up[n], down[n] = x[n] + h * d, x[n] - h * d
        slope = (f(*up) - f(*down)) / (2 * h)
        mine = float((got[name].double().cpu() * d).sum())
        # differences: h^2 times a third derivative of order the sum of |d|^3-weighted terms, far under 1e-5 of the norm
        norm = float(got[name].double().cpu().norm() * d.norm())
        assert abs(slope - mine) <= 1e-5 * norm, (name, slope, mine)


def test_repeats_and_offsets_past_32_bits(gpu):
    """A key cache of more than 2^31 elements, its last sample in use; and the same call twice gives the same bits."""
    import nnh
    D = 128
    strided = torch.as_strided(torch.zeros(2 ** 31 + 2 ** 28, dtype=torch.bfloat16, device="cuda"), (2, 300, 2, D), (2 ** 31 - 2 ** 20, 4096, D, 1))
    vals = draw(7, 2, 300, 2, D, dtype=torch.bfloat16).cuda()
    strided.copy_(vals)
    q = draw(8, 2, 200, 4, D, dtype=torch.bfloat16).cuda()
    rule = nnh.AttentionRule(causal=False)
    want = masked_attention(q, vals, vals)
    for n_q in (200, 1):
        out, lse = nnh.masked_attention_forward(q[:, :n_q], strided, strided, rule)
        assert_within(out, (want["out"][0][:, :n_q], want["out"][1][:, :n_q]), n_q)
        again, _ = nnh.masked_attention_forward(q[:, :n_q], strided, strided, rule)
        assert torch.equal(out, again)


@pytest.mark.parametrize("n_q", [512, 12])
@pytest.mark.parametrize("strided", [False, True])
def test_rest_of_out(gpu, n_q, strided):
    """Peaked rows of short documents, where out's rounding weighs most in the queries' gradients. With the rest two roundings
    of half a step are left (dS and the result), of 2^-8 / sqrt(3) of the values' norm each at most: sqrt(2) 2^-8 / sqrt(3)
    together. Both forms of the forward call (12 queries are split), rows that are not 16-byte aligned too."""
    import nnh
    gen = torch.Generator().manual_seed(n_q)
    q, k, v, g = (torch.randn(1, n_q, 1, 64, generator=gen).bfloat16() for _ in range(4))
    q *= 3
    d = (torch.arange(n_q) // 16).int()[None]
    o = dict(causal=True, cap=30.0, q_docs=d, k_docs=d)
    want = masked_attention(q, k, v, g, **o)
    rule = nnh.AttentionRule(causal=True, cap=30.0, q_docs=d.cuda(), k_docs=d.cuda())
    q, k, v, g = (x.cuda() for x in (q, k, v, g))
    rest = torch.full((1, n_q, 1, 65), 7.0).bfloat16().cuda()[..., :64] if strided else True
    out, lse = nnh.masked_attention_forward(q, k, v, rule, rest=rest)
    exact = want["out"][0]
    lost = exact - out.double().cpu()
    assert float((lse.rest.double().cpu() - lost).abs().max()) <= 2.0 ** -9 * float(exact.abs().max()) * 2.0 ** -2 + float(want["out"][1].max())
    dq, dk, dv = nnh.masked_attention_backward(g, q, k, v, out, lse, rule)
    for name, x in (("dq", dq), ("dk", dk), ("dv", dv)):
        assert_within(x, want[name], name)
        exact = want[name][0]
        assert float((x.double().cpu() - exact).norm() / exact.norm()) <= (2.0 / 3.0) ** 0.5 * 2.0 ** -8
    # a copy has none: the same out and lse, the bounds without it
    copy = nnh.masked_attention_forward(q, k, v, rule, rest=False)
    assert torch.equal(copy[0], out) and torch.equal(copy[1], lse) and copy[1].rest is None
    for name, x in zip(("dq", "dk", "dv"), nnh.masked_attention_backward(g, q, k, v, *copy, rule)):
        assert_within(x, want[name], name)


@pytest.mark.parametrize("dtype,Tq", [("bf16", 200), ("f32", 130), ("bf16", 1)])
def test_capture(gpu, dtype, Tq):
    """Both passes captured once with a workspace of their own (documents' ranges, key tiles shared by workgroups, the split form) and
    replayed on new inputs, with eager calls between; refused without one."""
    import nnh
    t, N, H, Hkv, D, Tk = T[dtype], 2, 4, 2, 64, max(Tq, 150)
    code = nnh.BF16 if dtype == "bf16" else nnh.F32
    assert code in (0, 1)
    q, g = (draw(s, N, Tq, H, D, dtype=t).cuda() for s in (0, 1))
    k, v = (draw(s, N, Tk, Hkv, D, dtype=t).cuda() for s in (2, 3))
    docs = documents(N, Tk, 4).cuda()
    starts = torch.full((N,), Tk - Tq).int().cuda()
    rule = nnh.AttentionRule(causal=True, cap=20.0, q_start=starts, q_docs=docs[:, Tk - Tq:].contiguous(), k_docs=docs)
    size = max(nnh.workspace_size("masked_attention", N, Tq, Tk, H, Hkv, D, 1, b) for b in (0, 1))
    room = torch.empty(size, dtype=torch.uint8, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()

    def both():
        out, lse = nnh.masked_attention_forward(q, k, v, rule)
        return (out, lse) + nnh.masked_attention_backward(g, q, k, v, out, lse, rule)

    nnh.set_workspace(room, side)
    try:
        with torch.cuda.graph(graph, stream=side):
            got = both()
        for seed in range(3):
            for i, x in enumerate((q, k, v, g)):
                x.copy_(draw(10 * seed + i, *x.shape, dtype=t))
            want = both()
            graph.replay()
            torch.cuda.synchronize()
            for x, y in zip(got, want):
                assert torch.equal(x, y)
    finally:
        nnh.set_workspace(None, side)
    other = torch.cuda.CUDAGraph()
    with pytest.raises(nnh.NnhError, match="registered workspace"):
        with torch.cuda.graph(other, stream=side):
            both()


def test_two_streams_at_once(gpu):
    """Calls that need scratch on two streams with no order between them."""
    import nnh
    N, Tq, H, D = 1, 400, 2, 64
    q, k, v, g = ([draw(4 * s + i, N, Tq, H, D, dtype=torch.bfloat16).cuda() for s in range(2)] for i in range(4))
    docs = [documents(N, Tq, s).cuda() for s in range(2)]
    rules = [nnh.AttentionRule(causal=True, q_docs=d, k_docs=d) for d in docs]

    def both(s):
        out, lse = nnh.masked_attention_forward(q[s], k[s], v[s], rules[s])
        return (out, lse) + nnh.masked_attention_backward(g[s], q[s], k[s], v[s], out, lse, rules[s])

    want = [both(s) for s in range(2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(4):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                got[s].append(both(s))
    torch.cuda.synchronize()
    for s in range(2):
        for one in got[s]:
            for x, y in zip(one, want[s]):
                assert torch.equal(x, y)


@pytest.mark.parametrize("n_q", [1, 40])
@pytest.mark.parametrize("far", ["rows", "samples"])
def test_offsets_past_32_bits(gpu, n_q, far):
    """Keys and values whose rows lie 2^22 elements apart (the last ones past 2^31 elements), or whose samples do 2^31."""
    N, Tk, D = (1, 600, 64) if far == "rows" else (2, 70, 64)
    strides = (0, 1 << 22, D, 1) if far == "rows" else ((1 << 31) + 64, D, D, 1)
    q, k, v = draw(0, N, n_q, 1, D, dtype=torch.bfloat16), draw(1, N, Tk, 1, D, dtype=torch.bfloat16), draw(2, N, Tk, 1, D, dtype=torch.bfloat16)
    room = [torch.empty((N - 1) * strides[0] + (Tk - 1) * strides[1] + D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    kk, vv = (r.as_strided((N, Tk, 1, D), strides) for r in room)
    kk.copy_(k)
    vv.copy_(v)
    g = draw(3, N, n_q, 1, D, dtype=torch.bfloat16)
    want = masked_attention(q, k, v, g)
    got = run(q, kk, vv, g)
    for name, x in got.items():
        assert_within(x, want[name], name)
