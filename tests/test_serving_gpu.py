"""Serving as a whole: generation from the C++ layer's Transformer (Decoder over a paged cache, with 32-bit and with 8-bit linears)
against the same model in 64-bit torch, and one captured step of the binding's operators (append, attention, 8-bit linear, choice of a
token), replayed as sequences grow.

The bound on logits in 32 bits: a block passes about 10 operations, each with roundings of up to 2^-24 times the root of its sum's
terms (random signs; 256 at most) of the values' size, and a layer norm before each branch keeps sizes near 1: 2^-24 * 16 * 10 * 2
blocks = 2e-5 of the largest logit; 5 times that is allowed, as the worst of many.

With 8-bit linears the same roundings move some of an activation's codes by one where it lies next to a tie between two: by scale =
max / 127 of the row, in one of 64 to 256 terms. A code is next to a tie by 2e-5 * 127 of its steps, one in 200; the 1,100 codes behind a
logit (2 blocks of 64 + 64 + 64 + 256, the head's 64) have 6 such, and earlier tokens' as many, through the attention's mean. One changes
an output by max / 127 times a weight, 3 / 127 * 0.06 = 1.5e-3 beside values near 1; sqrt(6 + 6) of these are 5e-3, and 2e-2 of the largest
logit is allowed. A wrong scale, page or column changes them by their whole size, and quantisation itself by 2 to 5 times that bound."""
import ctypes as C
import math
import os

import numpy as np
import pytest
import torch

from serving_reference import T, codes_of, draw, ints
from test_sample_gpu import check

pytestmark = pytest.mark.gpu
HARNESS = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "lib", "libserving_harness.so")
V, D, H, L, LONGEST = 61, 64, 4, 2, 90


@pytest.fixture(scope="module")
def harness(gpu):
    if not os.path.exists(HARNESS):
        pytest.fail(f"{HARNESS} missing: build it with `make -C tests/cpp` (or __graft_entry__.build())")
    lib = C.CDLL(HARNESS)
    lib.serving_last_error.restype = C.c_char_p
    return lib


def ok(harness, rc):
    assert rc == 0, harness.serving_last_error().decode()


def sizes(*values):
    return [C.c_size_t(v) for v in values]


def at(a):
    return None if a is None else C.c_void_p(a.ctypes.data)


def parameters(flat, learned):
    block = [(D,), (D,)] + [(D, D), (D,)] * 4 + [(D,), (D,), (4 * D, D), (4 * D,), (D, 4 * D), (D,)]
    out, k = [], 0
    for s in [(V, D)] + [(LONGEST, D)] * learned + block * L + [(D,), (D,), (V, D), (V,)]:
        out.append(torch.tensor(flat[k:k + math.prod(s)].astype(np.float64)).view(s))
        k += math.prod(s)
    assert k == flat.size
    if not learned:
        pos, c = torch.arange(LONGEST, dtype=torch.float64)[:, None], torch.arange(D)
        angle = pos / 10000.0 ** ((c - c % 2).double() / D)
        out.insert(1, torch.where(c % 2 == 0, angle.sin(), angle.cos()))
    return out


def logits_of(params, ids, int8):
    """The logits after the last of ids, in 64 bits; int8: linears of 8-bit codes."""
    def linear(x, w, b):
        if int8:
            (x, s), (w, t) = codes_of(x), codes_of(w)
            return (x @ w.t()) * s[:, None] * t.double() + b
        return x @ w.t() + b
    p = iter(params)
    take = lambda n: [next(p) for _ in range(n)]  # noqa: E731
    emb, pos = take(2)
    norm = lambda x, g, b: torch.nn.functional.layer_norm(x, (D,), g, b, 1e-5)  # noqa: E731
    n = len(ids)
    h = emb[torch.tensor(ids)] + pos[:n]
    heads = lambda x: x.view(n, H, D // H).transpose(0, 1)  # noqa: E731
    see = torch.ones(n, n, dtype=torch.bool).tril()
    for _ in range(L):
        g1, b1, wq, bq, wk, bk, wv, bv, wo, bo, g2, b2, w1, c1, w2, c2 = take(16)
        x = norm(h, g1, b1)
        q, k, v = (heads(linear(x, w, b)) for w, b in ((wq, bq), (wk, bk), (wv, bv)))
        z = (q @ k.transpose(1, 2) / math.sqrt(D // H)).masked_fill(~see, -math.inf)
        h = h + linear((torch.softmax(z, 2) @ v).transpose(0, 1).reshape(n, D), wo, bo)
        f = linear(norm(h, g2, b2), w1, c1)
        h = h + linear(0.5 * f * (1 + torch.tanh(0.7978845608028654 * (f + 0.044715 * f ** 3))), w2, c2)
    g, b, w, c = take(4)
    return linear(norm(h[-1:], g, b), w, c)[0]


# (steps of (sequence, new tokens; 0: dropped) turns): chunks, single tokens, both, a sequence that starts over in others' pages
RUNS = {
    "single": [[(0, 1)]] * 5,
    "chunk then single": [[(0, 33)]] + [[(0, 1)]] * 4 + [[(0, 47)]],
    "many": [[(0, 5), (1, 40)], [(0, 1), (1, 1), (2, 17)], [(2, 1), (0, 1), (1, 1), (3, 64)], [(1, 0), (0, 20), (3, 1)], [(1, 29), (3, 1), (0, 1)]],
}


@pytest.mark.parametrize("page,pages", [(16, 0), (7, 26), (64, 5), (1, 180)])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("run", RUNS)
def test_steps(harness, run, int8, page, pages):
    steps, rng, learned = RUNS[run], np.random.default_rng(3), page != 7
    turns = np.array([len(s) for s in steps], np.int32)
    flat = [t for s in steps for t in s]
    sequence, count = (np.array([t[i] for t in flat], np.int32) for i in (0, 1))
    tokens = rng.integers(0, V, int(count.sum())).astype(np.int32)
    room, n = np.zeros(1 << 18, np.float32), int((count > 0).sum())
    logits, whole = np.zeros((n, V), np.float32), np.zeros((n, V), np.float32)
    elements, left = C.c_size_t(), C.c_size_t()
    ok(harness, harness.serving_steps(*sizes(V, D, H, L, LONGEST), int(learned), *sizes(4, page, pages), int(int8), C.c_size_t(len(steps)), at(turns),
                                      at(sequence), at(count), at(tokens), at(room), C.byref(elements), at(logits), at(whole), C.byref(left)))
    params = parameters(room[:elements.value], learned)
    held, k, i = {}, 0, 0
    for s, c in flat:
        if c == 0:
            held.pop(s)
            continue
        held.setdefault(s, []).extend(int(t) for t in tokens[k:k + c])
        k += c
        want = logits_of(params, held[s], int8)
        size, far = float(want.abs().max()), float((torch.tensor(logits[i].astype(np.float64)) - want).abs().max())
        assert far <= (2e-2 if int8 else 1e-4) * size, (i, s, c, far, size)
        if not int8:
            assert float(np.abs(logits[i] - whole[i]).max()) <= 2e-4 * size
        i += 1
    total = pages or 4 * -(-LONGEST // page)
    assert left.value == total - sum(-(-len(x) // page) for x in held.values())


@pytest.mark.parametrize("int8", [False, True])
def test_generate(harness, int8):
    n, length, count = 3, 21, 30
    tokens = np.random.default_rng(8).integers(0, V, (n, length)).astype(np.int32)

    def run(temperature, top_k):
        out = np.zeros((n, count), np.int32)
        ok(harness, harness.serving_generate(*sizes(V, D, H, L, LONGEST), int(int8), *sizes(n, length), at(tokens), C.c_size_t(count),
                                             C.c_float(temperature), top_k, at(out)))
        return out
    room, logits = np.zeros(1 << 18, np.float32), np.zeros((2, V), np.float32)
    one, elements, left = np.array([1], np.int32), C.c_size_t(), C.c_size_t()
    ok(harness, harness.serving_steps(*sizes(V, D, H, L, LONGEST), 1, *sizes(1, 16, 0), 0, C.c_size_t(1), at(one), at(np.zeros(1, np.int32)), at(one),
                                      at(one), at(room), C.byref(elements), at(logits[0]), at(logits[1]), C.byref(left)))
    params = parameters(room[:elements.value], True)
    first = run(0.0, 0)
    for a, b in zip(tokens, first):
        for i in (0, 1, 11, count - 1):
            z = logits_of(params, [int(t) for t in a] + [int(t) for t in b[:i]], int8)
            assert float(z.max() - z[b[i]]) <= 2 * (2e-2 if int8 else 1e-4) * float(z.abs().max())
    assert np.array_equal(run(5.0, 1), first)  # (one token to choose from)
    drawn = run(1.0, 0)
    assert np.array_equal(run(1.0, 0), drawn) and not np.array_equal(drawn, first) and drawn.min() >= 0 and drawn.max() < V


@pytest.mark.parametrize("rows,size", [(1, 1), (3, 61), (5, 9000)])
@pytest.mark.parametrize("rule", [(), ("temperature",), ("temperature", "top_k", "top_p", "min_p")])
def test_sample(harness, rows, size, rule):
    rng = np.random.default_rng(rows)
    logits = (4 * rng.standard_normal((rows, size))).astype(np.float32)
    given = {"temperature": rng.uniform(0.5, 2, rows).astype(np.float32), "top_k": rng.integers(1, 40, rows).astype(np.int32),
             "top_p": rng.uniform(0.5, 1, rows).astype(np.float32), "min_p": rng.uniform(0, 0.1, rows).astype(np.float32)}
    u = rng.random(rows).astype(np.float32)
    tokens, logprob = np.zeros(rows, np.int32), np.zeros(rows, np.float32)
    r = {k: given[k] if k in rule else None for k in given}
    ok(harness, harness.serving_sample(*sizes(rows, size), at(logits), at(u), *(at(r[k]) for k in ("temperature", "top_k", "top_p", "min_p")),
                                       at(tokens), at(logprob)))
    check(torch.tensor(logits), torch.tensor(u), got=(torch.tensor(tokens), torch.tensor(logprob)), **{k: torch.tensor(v) for k, v in r.items() if v is not None})


REFUSED = {2: [11, 12, 13, 15, 16, 17, 18, 19, 21], 3: [0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 14, 20, 22, 23, 24]}


@pytest.mark.parametrize("code,which", [(c, w) for c in REFUSED for w in REFUSED[c]])
def test_refused(harness, code, which):
    assert harness.serving_refused(which) == code, harness.serving_last_error().decode()


def test_after_a_refused_step(harness):
    a, b = np.zeros((2, 31), np.float32), np.ones((2, 31), np.float32)
    ok(harness, harness.serving_after_refusal(at(a), at(b)))
    assert np.array_equal(a, b)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [3, 40])
def test_captured_step(gpu, dtype, rows):
    """Hidden rows to tokens: a joint projection in 8 bits, its keys and values (columns of its rows) into the cache, attention, the
    projection to the vocabulary in 8 bits, the choice of tokens. One graph, one workspace of the largest call's size for all of them."""
    import nnh
    t, heads, groups, width, depth, size, page, most, N = T[dtype], 4, 2, 32, 200, 9000, 8, 32, 3
    wide, code = (heads + 2 * groups) * width, {"f32": nnh.F32, "bf16": nnh.BF16}[dtype]
    w, ws = nnh.quantize_rows(draw(1, wide, depth, dtype=t, scale=0.1).cuda())
    v, vs = nnh.quantize_rows(draw(2, size, heads * width, dtype=t, scale=0.1).cuda())
    table = torch.randperm(N * 20).int().view(N, 20).cuda()
    pools = [[torch.zeros(N * 20, page, groups, width, dtype=t, device="cuda") for _ in range(2)] for _ in range(2)]
    caches = [nnh.PagedCache(*p, table) for p in pools]
    x, u = torch.zeros(rows, depth, dtype=t, device="cuda"), torch.zeros(rows, device="cuda")
    starts, lens = ints(*[0] * (N + 1)).cuda(), ints(*[0] * N).cuda()
    temperature, top_k = torch.full((rows,), 0.8, device="cuda"), torch.full((rows,), 50, dtype=torch.int32, device="cuda")
    rule = nnh.AttentionRule(causal=True, k_lens=lens)

    def buffers():
        e = lambda *s, dtype=t: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
        return (e(rows, wide), e(rows, heads, width), e(rows, heads, dtype=torch.float32), e(rows, size), e(rows, dtype=torch.int32),
                e(rows, dtype=torch.float32))

    def step(cache, b):
        joint, out, lse, logits, tokens, logprob = b
        nnh.linear_int8(x, w, ws, out=joint)
        q, k, val = joint.view(rows, heads + 2 * groups, width).split([heads, groups, groups], 1)
        nnh.paged_append(cache, k, val, starts, lens)
        nnh.paged_attention(q, cache, starts, most, rule, out=out, lse=lse)
        nnh.linear_int8(out.view(rows, heads * width), v, vs, out=logits)
        nnh.sample(logits, u, temperature=temperature, top_k=top_k, tokens=tokens, logprob=logprob)

    need = max(nnh.workspace_size("linear_int8", rows, depth, wide), nnh.workspace_size("linear_int8", rows, heads * width, size),
               nnh.workspace_size("paged_attention", N, rows, most, 20 * page, heads, groups, width), nnh.workspace_size("sample", code, rows, size))
    room = torch.full((need + 4096,), 7, dtype=torch.uint8, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    one, two = buffers(), buffers()
    torch.cuda.synchronize()
    nnh.set_workspace(room[:need], side)
    try:
        with torch.cuda.graph(graph, stream=side):
            step(caches[0], one)
        held = [0] * N
        for seed, new in enumerate([[rows - 2, 1, 1], [1, 1, 1], [0, 1, 2], [1, rows - 1, 0], [1, 1, 1]]):
            new = [min(n, most) for n in new]
            held = [a + b for a, b in zip(held, new)]
            x.copy_(draw(10 * seed, rows, depth, dtype=t))
            u.copy_(torch.rand(rows, generator=torch.Generator().manual_seed(seed)))
            starts.copy_(ints(0, new[0], new[0] + new[1], sum(new)))
            lens.copy_(ints(*held))
            step(caches[1], two)
            graph.replay()
            torch.cuda.synchronize()
            live = sum(new)
            for i, (a, b) in enumerate(zip(one, two)):
                assert torch.equal(a[:live], b[:live]), (seed, i)
            assert all(torch.equal(a, b) for a, b in zip(*pools))
            # the same through torch, in 64 bits: the rows' own tokens, each a choice of the logits that the kernels made
            check(two[3][:live].cpu(), u[:live].cpu(), got=(two[4][:live], two[5][:live]), temperature=temperature[:live].cpu(), top_k=top_k[:live].cpu())
        assert bool((room[need:] == 7).all())
    finally:
        nnh.set_workspace(None, side)
