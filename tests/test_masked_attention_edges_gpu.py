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
