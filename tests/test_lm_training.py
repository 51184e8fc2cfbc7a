"""A language model's training step through the C++ layer (include/nn_hip_modules.hpp): Transformer::loss over packed documents
(masked attention in every block, the head's cross entropy), its gradients, and AdamW's step on them, against the same model in
64-bit torch.

The bound on a gradient: it passes about 20 operations a block, each of which adds roundings of up to (terms of its sums) u32
of the values' sizes, 64 to 256 terms here; 2^-24 * 40 operations * 256 terms = 6e-4 of the gradient's norm would be the
sum of all at their worst; roundings of random sign grow with the root of their number, and 1e-4 is four times that."""
import ctypes as C
import math
import os

import numpy as np
import pytest
import torch

from lm_reference import visible

pytestmark = pytest.mark.gpu
HARNESS = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "lib", "liblm_harness.so")
V, D, H, L, N, T = 61, 64, 4, 2, 3, 50


@pytest.fixture(scope="module")
def harness(gpu):
    if not os.path.exists(HARNESS):
        pytest.fail(f"{HARNESS} missing: build it with `make -C tests/cpp` (or __graft_entry__.build())")
    lib = C.CDLL(HARNESS)
    lib.lm_last_error.restype = C.c_char_p
    return lib


def fp(a):
    return None if a is None else a.ctypes.data_as(C.POINTER(C.c_float))


def ip(a):
    return None if a is None else a.ctypes.data_as(C.POINTER(C.c_int))


def batch(docs):
    rng = np.random.default_rng(5)
    ids = rng.integers(0, V, (N, T)).astype(np.float32)
    targets = rng.integers(0, V, (N, T)).astype(np.int32)
    targets[rng.random((N, T)) < 0.1] = -1
    d = None
    if docs:
        d = np.cumsum(rng.random((N, T)) < 0.08, axis=1).astype(np.int32)
        d[:, -4:] = -1
        targets[:, -4:] = -1
    return ids, targets, d


def train(harness, docs, cap, slopes, bits, steps, lr=1e-3):
    ids, targets, d = batch(docs)
    losses = np.zeros(steps, np.float32)
    room = [np.zeros(1 << 18, np.float32) for _ in range(3)]
    count = C.c_size_t(0)
    harness.lm_train.argtypes = [C.c_size_t] * 6 + [C.c_void_p] * 3 + [C.c_float, C.c_void_p, C.c_int, C.c_double, C.c_size_t] + [C.c_void_p] * 5
    rc = harness.lm_train(V, D, H, L, N, T, ids.ctypes.data, targets.ctypes.data, None if d is None else d.ctypes.data, cap,
                          None if slopes is None else slopes.ctypes.data, bits, lr, steps, losses.ctypes.data, *(r.ctypes.data for r in room),
                          C.addressof(count))
    assert rc == 0, harness.lm_last_error().decode()
    return losses, [r[:count.value] for r in room], (ids, targets, d)


def shapes():
    block = [(D,), (D,)] + [(D, D), (D,)] * 4 + [(D,), (D,), (4 * D, D), (4 * D,), (D, 4 * D), (D,)]
    return [(V, D), (T, D)] + block * L + [(D,), (D,), (V, D), (V,)]


def cut(flat):
    out, at = [], 0
    for s in shapes():
        n = math.prod(s)
        out.append(torch.tensor(flat[at:at + n].astype(np.float64)).view(s))
        at += n
    assert at == flat.size
    return out


def model(params, ids, targets, docs, cap, slopes):
    """The mean loss in 64 bits."""
    p = iter(params)
    take = lambda n: [next(p) for _ in range(n)]  # noqa: E731
    emb, pos = take(2)
    norm = lambda x, g, b: torch.nn.functional.layer_norm(x, (D,), g, b, 1e-5)  # noqa: E731
    h = emb[torch.tensor(ids.astype(np.int64))] + pos
    d = None if docs is None else torch.tensor(docs)
    see, far = visible(N, T, T, causal=True, q_docs=d, k_docs=d)
    some = see.any(2)
    heads = lambda x: x.view(N, T, H, D // H).transpose(1, 2)  # noqa: E731
    for _ in range(L):
        g1, b1, wq, bq, wk, bk, wv, bv, wo, bo, g2, b2, w1, c1, w2, c2 = take(16)
        x = norm(h, g1, b1)
        q, k, v = (heads(x @ w.t() + b) for w, b in ((wq, bq), (wk, bk), (wv, bv)))
        z = q @ k.transpose(2, 3) / math.sqrt(D // H)
        z = cap * torch.tanh(z / cap) if cap else z
        if slopes is not None:
            z = z - torch.tensor(slopes.astype(np.float64))[None, :, None, None] * far[:, None]
        z = z.masked_fill(~see[:, None] & some[:, None, :, None], -math.inf)
        a = (torch.softmax(z, 3) @ v * some[:, None, :, None]).transpose(1, 2).reshape(N, T, D)
        h = h + a @ wo.t() + bo
        f = norm(h, g2, b2) @ w1.t() + c1
        f = 0.5 * f * (1 + torch.tanh(0.7978845608028654 * (f + 0.044715 * f ** 3)))
        h = h + f @ w2.t() + c2
    g, b, w, c = take(4)
    logits = norm(h, g, b) @ w.t() + c
    return torch.nn.functional.cross_entropy(logits.view(-1, V), torch.tensor(targets.astype(np.int64)).view(-1), ignore_index=-1)


@pytest.mark.parametrize("docs,cap,slopes", [(False, 0.0, False), (True, 0.0, False), (True, 2.0, True)])
@pytest.mark.parametrize("bits", [32, 8])
def test_training_step(harness, docs, cap, slopes, bits):
    s = np.exp2(-np.arange(1, H + 1)).astype(np.float32) if slopes else None
    losses, (before, grads, after), (ids, targets, d) = train(harness, docs, cap, s, bits, 1)
    params = [x.requires_grad_() for x in cut(before)]
    loss = model(params, ids, targets, d, cap, s)
    want = torch.autograd.grad(loss, params)
    loss = loss.detach()
    assert abs(float(loss) - float(losses[0])) <= 1e-5 * float(loss)
    for i, (x, y, shape) in enumerate(zip(cut(grads), want, shapes())):
        # a gradient that cancels (a key bias moves all of a row's scores alike) is rounding alone: against the largest one's size
        size = max(float(y.norm()), 1e-3 * max(float(z.norm()) for z in want) * math.sqrt(y.numel() / max(z.numel() for z in want)))
        assert float((x - y).norm()) <= 1e-4 * size, (i, shape, float((x - y).norm()), float(y.norm()))
    # AdamW's first step from zero moments, on the gradients that the step itself made
    for x, g, new in zip(cut(before), cut(grads), cut(after)):
        exact = x * (1 - 1e-3 * 0.01) - 1e-3 * g / (g.abs() + 1e-8)
        tiny = 1e-3 * (g.abs() < 1e-18)  # (squares below fp32's range)
        assert bool(((new - exact).abs() <= 4 * 2.0 ** -24 * x.abs() + 1e-3 * 16 * 2.0 ** -24 + tiny).all())


def test_steps_run(harness):
    """Several steps in a row, both moments' forms: finite, and the same again."""
    for bits in (32, 8):
        one = train(harness, True, 5.0, None, bits, 6)
        two = train(harness, True, 5.0, None, bits, 6)
        assert np.isfinite(one[0]).all() and np.isfinite(one[1][2]).all()
        assert np.array_equal(one[0], two[0]) and np.array_equal(one[1][2], two[1][2])


def test_one_node_as_query_key_and_value(harness):
    rng = np.random.default_rng(2)
    n, t, heads, dim, vocab = 2, 33, 2, 24, 40
    x, w = rng.standard_normal((n, t, dim)).astype(np.float32), rng.standard_normal((vocab, dim)).astype(np.float32)
    y = rng.integers(0, vocab, (n, t)).astype(np.int32)
    loss, dx, dw = np.zeros(1, np.float32), np.zeros_like(x), np.zeros_like(w)
    rc = harness.lm_shared(*(C.c_size_t(v) for v in (n, t, heads, dim)), fp(x), C.c_size_t(vocab), fp(w), ip(y), fp(loss), fp(dx), fp(dw))
    assert rc == 0, harness.lm_last_error().decode()
    a, b = (torch.tensor(v.astype(np.float64)).requires_grad_() for v in (x, w))
    h = a.view(n, t, heads, dim // heads).transpose(1, 2)
    z = (h @ h.transpose(2, 3) / math.sqrt(dim // heads)).masked_fill(~torch.ones(t, t, dtype=torch.bool).tril(), -math.inf)
    out = (torch.softmax(z, 3) @ h).transpose(1, 2).reshape(n, t, dim)
    want = torch.nn.functional.cross_entropy((out @ b.t()).view(-1, vocab), torch.tensor(y.astype(np.int64)).view(-1))
    ga, gb = torch.autograd.grad(want, (a, b))
    assert abs(want.item() - float(loss[0])) <= 1e-5 * want.item()
    for got, v in ((dx, ga), (dw, gb)):
        assert float((torch.tensor(got.astype(np.float64)) - v).norm()) <= 1e-4 * float(v.norm())


@pytest.mark.parametrize("which,code", [(0, 2), (1, 2), (2, 2), (3, 1)])
def test_refusals(harness, which, code):
    assert harness.lm_refused(which) == code


def test_operators_in_a_row_in_16_bits(gpu):
    """Attention, the head's loss, their gradients and an AdamW step on the head and the queries, in bf16, as a training loop
    calls them, on another stream than the default one."""
    import nnh
    from lm_reference import assert_within, linear_cross_entropy, masked_attention
    gen = torch.Generator().manual_seed(1)
    n, t, h, kv, d, vocab = 2, 70, 4, 2, 32, 300
    q, k, v = (torch.randn(n, t, x, d, generator=gen).bfloat16() for x in (h, kv, kv))
    w = (torch.randn(vocab, h * d, generator=gen) * 0.1).bfloat16()
    y = torch.randint(-1, vocab, (n, t), generator=gen).int()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        Q, K, W, X, Y = q.cuda(), k.cuda(), w.cuda(), v.cuda(), y.cuda()
        rule = nnh.AttentionRule(causal=True, cap=10.0)
        out, lse = nnh.masked_attention_forward(Q, K, X, rule)
        loss, dout, dw, _ = nnh.linear_cross_entropy_train(out.view(n, t, h * d), W, Y)
        dq, dk, dv = nnh.masked_attention_backward(dout.view(n, t, h, d), Q, K, X, out, lse, rule)
        params, masters = [Q, W], [Q.float(), W.float()]
        opt = nnh.AdamW(masters, [dq, dw], bits=8, copies=params, lr=1e-2)
        opt.step()
    s.synchronize()
    assert_within(out, masked_attention(q, k, v, causal=True, cap=10.0)["out"], "out")
    want = linear_cross_entropy(out.cpu().view(n * t, h * d), w, y.view(-1), kept=True)
    assert_within(loss, want["loss"], "loss")
    assert_within(dout.view(n * t, h * d), want["dx"], "dout")
    assert_within(dw, want["dw"], "dw")
    want = masked_attention(q, k, v, dout.view(n, t, h, d), causal=True, cap=10.0)
    for name, x in (("dq", dq), ("dk", dk), ("dv", dv)):
        assert_within(x, want[name], name)
    for low, high in zip(params, masters):
        assert torch.equal(low, high.bfloat16()) and not torch.equal(high, torch.zeros_like(high))
