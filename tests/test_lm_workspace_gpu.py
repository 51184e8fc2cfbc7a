"""The language-model operators' scratch in a caller's buffer (nnh_set_workspace)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def calls(nnh):
    """{name: (bytes, call)} of calls that need scratch."""
    t = torch.bfloat16
    q, k, v = (torch.randn(1, n, 2, 64, device="cuda").to(t) for n in (1, 700, 700))
    long = [torch.randn(1, 100, 2, 64, device="cuda").to(t) for _ in range(4)]
    docs = torch.zeros(1, 100, dtype=torch.int32, device="cuda")
    plain, rule = nnh.AttentionRule(), nnh.AttentionRule(q_docs=docs, k_docs=docs)
    x, w = torch.randn(40, 64, device="cuda").to(t), torch.randn(90, 64, device="cuda").to(t)
    y = torch.randint(0, 90, (40,), device="cuda", dtype=torch.int32)
    size = nnh.workspace_size

    def attend():
        out, lse = nnh.masked_attention_forward(*long[:3], rule)
        return (out, lse) + nnh.masked_attention_backward(long[3], *long[:3], out, lse, rule)

    return {
        "split": (size("masked_attention", 1, 1, 700, 2, 2, 64, 0, 0), lambda: nnh.masked_attention_forward(q, k, v, plain)),
        "attention": (max(size("masked_attention", 1, 100, 100, 2, 2, 64, 1, b) for b in (0, 1)), attend),
        "loss": (size("linear_cross_entropy", nnh.BF16, 40, 64, 90, 2, 1), lambda: nnh.linear_cross_entropy_train(x, w, y)[:3]),
        "loss in 32 bits": (size("linear_cross_entropy", nnh.F32, 40, 64, 90, 2, 1), lambda: nnh.linear_cross_entropy_train(x.float(), w.float(), y)[:3]),
    }


@pytest.mark.parametrize("name", ["split", "attention", "loss", "loss in 32 bits"])
def test_a_buffer_at_any_address(gpu, name):
    """Scratch is read and written in words of 16 bytes: a buffer that begins at a multiple of that gives the results of the library's
    own, another is refused, captured or not."""
    import nnh
    size, call = calls(nnh)[name]
    want = call()
    torch.cuda.synchronize()
    room = torch.empty(size + 16, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream()
    side = torch.cuda.Stream()
    try:
        for at in (0, 16):
            nnh.set_workspace(room[at:at + size], stream)
            for x, y in zip(want, call()):
                assert torch.equal(x, y)
        for at in (1, 4, 8):
            nnh.set_workspace(room[at:at + size], stream)
            with pytest.raises(nnh.NnhError, match="16 bytes"):
                call()
            nnh.set_workspace(room[at:at + size], side)
            with pytest.raises(nnh.NnhError, match="16 bytes"):
                with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                    call()
    finally:
        torch.cuda.synchronize()
        nnh.set_workspace(None, stream)
        nnh.set_workspace(None, side)
    for x, y in zip(want, call()):
        assert torch.equal(x, y)
