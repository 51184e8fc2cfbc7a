"""Masked attention (nnh_masked_attention_*) on the GPU: calls at the edges of what its documentation allows."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("N,Tq,Tk", [(2, 40, 0), (2, 1, 0), (2, 0, 70), (0, 5, 7), (2, 0, 0)])
def test_documents_of_an_empty_side(gpu, dtype, N, Tq, Tk):
    """Document arrays beside no keys, no queries or no samples (an empty tensor has no address): rows of zeros, an lse of
    -infinity and gradients of zeros, as without documents."""
    import nnh
    H, Hkv, D, t = 4, 2, 64, T[dtype]
    q, g = (torch.randn(N, Tq, H, D, device="cuda").to(t) for _ in range(2))
    k, v = (torch.randn(N, Tk, Hkv, D, device="cuda").to(t) for _ in range(2))
    docs = [torch.zeros(N, x, dtype=torch.int32, device="cuda") for x in (Tq, Tk)]
    rule = nnh.AttentionRule(causal=True, q_docs=docs[0], k_docs=docs[1])
    out, lse = nnh.masked_attention_forward(q, k, v, rule)
    assert not bool(out.any()) and bool((lse == -math.inf).all())
    grads = [torch.full_like(x, 7.0) for x in (q, k, v)]
    nnh.masked_attention_backward(g, q, k, v, out, lse, rule, *(y for x in grads for y in (x, True)))
    assert not any(bool(x.any()) for x in grads)
    grads = [torch.full_like(x, 7.0) for x in (q, k, v)]
    nnh.masked_attention_backward(g, q, k, v, out, lse, rule, *(y for x in grads for y in (x, False)))
    assert all(bool((x == 7.0).all()) for x in grads)


@pytest.mark.parametrize("which", ["forward", "backward"])
def test_the_rest_is_kept_for_another_stream(gpu, which):
    """A call on a stream given to it: what the call has made and lse carries is not given to others while that stream may use it."""
    import nnh
    q, k, v = (torch.randn(1, 300, 2, 64, device="cuda").bfloat16() for _ in range(3))
    side = torch.cuda.Stream()
    rule = nnh.AttentionRule()
    if which == "backward":
        out, lse = nnh.masked_attention_forward(q, k, v, rule)
    torch.cuda.synchronize()
    nnh.bench_delay(100000, side)
    if which == "backward":
        grads = nnh.masked_attention_backward(q, q, k, v, out, lse, rule, stream=side)
    else:
        out, lse = nnh.masked_attention_forward(q, k, v, rule, stream=side)
        grads = ()
    for x in (q, k, v, out, lse) + grads:
        x.record_stream(side)  # the caller's own
    at, like = lse.rest.data_ptr(), torch.empty_like(lse.rest, device="cpu")
    del lse
    others = [torch.empty(like.shape, dtype=like.dtype, device="cuda") for _ in range(4)]
    busy = not side.query()
    torch.cuda.synchronize()
    assert busy and at not in [x.data_ptr() for x in others]
