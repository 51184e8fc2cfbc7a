"""Masked attention on the GPU where its kernels take another path than at small sizes, against the formula in 64 bits: key tiles that
workgroups share, more than 64 tiles to a row, key heads dealt out over the chip's parts, wide heads under every mask, the form for
few queries under documents."""
import ctypes as C
import math

import pytest
import torch

from lm_reference import assert_within, masked_attention
from test_masked_attention_gpu import T, check, documents, draw, run

pytestmark = pytest.mark.gpu


def parts(N, Tq, Tk, H, Hkv, D):
    """Workgroups to a key tile in the backward pass, by its scratch: delta and lse beside it are N H Tq floats each."""
    import nnh
    rows = -(-N * H * Tq * 4 // 256) * 256
    left = nnh.workspace_size("masked_attention", N, Tq, Tk, H, Hkv, D, 0, 1) - 2 * rows
    return max(1, left // (2 * N * Hkv * Tk * (-(-D // 4) * 4) * 4))


SHARED = [(1, 1030, 1030, 1, 1, 64, 2), (1, 300, 300, 4, 1, 128, 2), (1, 300, 420, 4, 1, 30, 2), (1, 700, 130, 8, 2, 80, 5), (1, 2100, 200, 2, 1, 96, 8),
          (2, 530, 530, 6, 2, 13, 3)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHARED)
@pytest.mark.parametrize("causal", [False, True])
def test_shared_key_tiles(gpu, dtype, shape, causal):
    *shape, n = shape
    assert parts(*shape) == n
    check(dtype, *shape, causal=causal, cap=8.0 if causal else 0.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["docs", "window", "prefix", "lens"])
def test_shared_key_tiles_under_masks(gpu, dtype, kind):
    N, L = 2, 560
    assert parts(N, L, L, 4, 2, 64) == 2
    o = {"causal": True}
    if kind == "docs":
        o["q_docs"] = o["k_docs"] = documents(N, L, 9)
    if kind == "window":
        o["window"] = 90
    if kind == "prefix":
        o["prefix"] = torch.tensor([300, 17], dtype=torch.int32)
    if kind == "lens":
        o["k_lens"] = torch.tensor([401, 0], dtype=torch.int32)
    check(dtype, N, L, L, 4, 2, 64, **o)


def one_by_one(g, q, k, v, out, lse, rule, grads, first):
    """The C call with the gradients that are given (None: not wanted)."""
    import nnh
    N, Tq, H, D = q.shape
    Tk, Hkv = k.shape[1:3]
    dev = torch.cuda.current_device()
    ref = lambda t: None if t is None else C.byref(nnh.HeadTensor(t.data_ptr(), *t.stride()[:3]))  # noqa: E731
    r = rule._struct(N, Tq, Tk, H, dev)
    nnh.check(nnh.lib().nnh_masked_attention_backward(nnh._type(q), N, Tq, Tk, H, Hkv, D, *map(ref, (g, q, k, v, out, getattr(lse, "rest", None))),
                                                      lse.data_ptr(), C.byref(r), ref(grads[0]), first, ref(grads[1]), first, ref(grads[2]),
                                                      first, nnh._stream(None)))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 30])
@pytest.mark.parametrize("n_q", [300, 100])
def test_gradients_in_part_and_added(gpu, dtype, D, n_q):
    """Each of the gradients alone, each left out, all; stored and added to what is there. Key tiles shared (300 queries) or not."""
    import nnh
    N, Tk, H, Hkv = 1, 200, 4, 1
    assert parts(N, n_q, Tk, H, Hkv, D) == (2 if n_q == 300 else 1)
    t = T[dtype]
    q, g = (draw(s, N, n_q, H, D, dtype=t).cuda() for s in (0, 1))
    k, v = (draw(s, N, Tk, Hkv, D, dtype=t).cuda() for s in (2, 3))
    rule = nnh.AttentionRule(causal=True, q_start=torch.full((N,), 20, dtype=torch.int32, device="cuda"))
    out, lse = nnh.masked_attention_forward(q, k, v, rule)
    want = masked_attention(q, k, v, g, causal=True, q_start=torch.full((N,), 20))
    u = torch.finfo(t).eps / 2
    for wanted in [(1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, 1)]:
        for first in (1, 0):
            old = [draw(20 + i, *x.shape, dtype=t).cuda() for i, x in enumerate((q, k, v))]
            grads = [x.clone() if w else None for w, x in zip(wanted, old)]
            one_by_one(g, q, k, v, out, lse, rule, grads, first)
            for name, x, was in zip(("dq", "dk", "dv"), grads, old):
                if x is None:
                    continue
                value, bound = want[name]
                was = 0.0 if first else was.double().cpu()
                total = value + was
                assert_within(x, (total, bound + u * total.abs() + u * bound), (name, wanted, first))


@pytest.mark.parametrize("dtype,D", [("bf16", 64), ("f32", 64), ("f32", 128), ("bf16", 20)])
@pytest.mark.parametrize("kind", ["causal", "docs", "window"])
def test_more_than_64_tiles(gpu, dtype, D, kind):
    """4200 keys (66 tiles of 64 or 132 of 32) and 2100 queries (66 of 32): the tiles that some query sees are found 64 at a time, whole
    runs of them unseen."""
    N, Tq, Tk = 1, 2100, 4200
    o = {"causal": True, "q_start": torch.tensor([Tk - Tq], dtype=torch.int32)}
    if kind == "docs":
        at = lambda n: (torch.arange(n) // 700).int()[None]  # noqa: E731
        o["k_docs"], o["q_docs"] = at(Tk), at(Tk)[:, Tk - Tq:].contiguous()
        o["k_docs"][:, 4100:] = o["q_docs"][:, 2000:] = -1
        o["window"] = 500
    if kind == "window":
        o["window"] = 33
        o["prefix"] = torch.tensor([40], dtype=torch.int32)
    check(dtype, N, Tq, Tk, 1, 1, D, **o)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads", [(2, 8, 4), (8, 1, 1), (1, 16, 16)])
def test_heads_over_the_chip(gpu, dtype, heads):
    """Pairs of a sample and a key head in eights (each eighth is one XCD's), several tiles of queries and keys, each pair its own length."""
    N, H, Hkv = heads
    L = 290
    o = {"causal": True, "k_lens": torch.tensor([L - 31 * n for n in range(N)], dtype=torch.int32),
         "slopes": torch.exp2(-8.0 * torch.arange(1.0, H + 1) / H)}
    check(dtype, N, L, L, H, Hkv, 64, **o)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [96, 128, 40, 17])
@pytest.mark.parametrize("kind", ["cap", "slopes", "window", "prefix", "lens", "docs", "all"])
def test_masks_at_other_head_widths(gpu, dtype, D, kind):
    N, L, H, Hkv = 3, 190, 4, 2
    every = kind == "all"
    o = {"causal": kind != "docs"}
    if kind == "cap" or every:
        o["cap"] = 5.0
    if kind == "slopes" or every:
        o["slopes"] = torch.exp2(-torch.arange(1.0, H + 1))
    if kind == "window" or every:
        o["window"] = 37
    if kind == "prefix" or every:
        o["prefix"] = torch.tensor([0, 70, 500], dtype=torch.int32)
    if kind == "lens" or every:
        o["k_lens"] = torch.tensor([190, 0, 65], dtype=torch.int32)
    if kind == "docs" or every:
        o["q_docs"] = o["k_docs"] = documents(N, L, 5)
    check(dtype, N, L, L, H, Hkv, D, scale_q=2.0, **o)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [96, 128, 17])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_not_finite_at_other_head_widths(gpu, dtype, D, bad):
    """Values of one document, and of rows of none, that are not finite stay out of another document's results and gradients."""
    t, N, L, H = T[dtype], 1, 150, 2
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


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 96, 30])
@pytest.mark.parametrize("tq", [1, 5, 32])
def test_few_queries_under_documents(gpu, dtype, D, tq):
    """The form that divides the keys: documents whose tiles are skipped, a prefix, a window, lengths of its own for each sample; the
    backward pass of so few queries too."""
    N, Tk, H, Hkv = 3, 1500, 8, 2
    lens = torch.tensor([1500, 901, 64], dtype=torch.int32)
    k_docs = (torch.arange(Tk) // 210).int().repeat(N, 1)
    k_docs[:, 400:420] = -1
    q_docs = torch.stack([k_docs[n, int(lens[n]) - tq:int(lens[n])] for n in range(N)]).contiguous()
    o = dict(causal=True, k_lens=lens, q_start=lens - tq, q_docs=q_docs, k_docs=k_docs)
    check(dtype, N, tq, Tk, H, Hkv, D, **o)
    check(dtype, N, tq, Tk, H, Hkv, D, train=False, window=100, prefix=torch.tensor([3, 0, 2000], dtype=torch.int32), cap=10.0, **o)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_shared_key_tiles_captured(gpu, dtype):
    """Captured with a workspace of exactly the size asked for, replayed on new inputs with eager calls between."""
    import nnh
    N, L, H, Hkv, D, t = 1, 530, 4, 2, 64, T[dtype]
    assert parts(N, L, L, H, Hkv, D) > 1
    q, g = (draw(s, N, L, H, D, dtype=t).cuda() for s in (0, 1))
    k, v = (draw(s, N, L, Hkv, D, dtype=t).cuda() for s in (2, 3))
    rule = nnh.AttentionRule(causal=True)
    size = nnh.workspace_size("masked_attention", N, L, L, H, Hkv, D, 0, 1)
    room = torch.full((size + 4096,), 7, dtype=torch.uint8, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()

    def both():
        out, lse = nnh.masked_attention_forward(q, k, v, rule)
        return (out, lse) + nnh.masked_attention_backward(g, q, k, v, out, lse, rule)

    nnh.set_workspace(room[:size], side)
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
        assert bool((room[size:] == 7).all())
    finally:
        nnh.set_workspace(None, side)
