"""The AdamW step (nnh_adamw_step) on the GPU against the formula in 64 bits.

Bounds: an fp32 moment takes three roundings of terms that may be larger than their sum (the products and the sum, 4 u32 of
the terms' absolute values); the parameter the roundings of its own product and difference and, on the update, of the two
moments, the root, the quotient and its factors (12 u32); a bf16 store adds half a step of bf16. 8-bit codes and scales are
those of the 64-bit values exactly: the inputs are random, so no value lies within 2^-50 of a border."""
import math

import pytest
import torch

from lm_reference import U32, adamw, assert_within, block_codes, unit

pytestmark = pytest.mark.gpu
HYPER = dict(lr=3e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1)
SIZES = [1, 3, 63, 64, 65, 0, 255, 4096, 4097, 20001]


def tensors(sizes, seed, p_type, g_type, offset=0):
    gen = torch.Generator().manual_seed(seed)

    def cut(scale, dtype):
        rows = []
        for n in sizes:
            whole = torch.zeros(n + offset, dtype=dtype, device="cuda")
            whole[offset:] = (torch.randn(n, generator=gen) * scale).to(dtype)
            rows.append(whole[offset:])
        return rows

    return cut(0.5, p_type), cut(0.01, g_type)


def check_32(sizes, p_type=torch.float32, g_type=torch.float32, copies=False, offset=0, steps=3):
    import nnh
    print(len(sizes), p_type, g_type, copies, offset, flush=True)
    p, g = tensors(sizes, 1, p_type, g_type, offset)
    extra = [torch.zeros(n + offset, dtype=torch.bfloat16, device="cuda")[offset:] for n in sizes] if copies else None
    opt = nnh.AdamW(p, g, copies=extra, **HYPER)
    scale = torch.tensor([0.7312], device="cuda")
    for step in range(1, steps + 1):
        old = [[x.double().cpu() for x in row] for row in (p, opt.m, opt.v)]
        opt.step(grad_scale=scale)
        torch.cuda.synchronize()
        for i, n in enumerate(sizes):
            s, gd = float(scale), g[i].double().cpu() * float(scale)
            want = adamw(old[0][i], g[i].double().cpu(), old[1][i], old[2][i], step, scale=s, **HYPER)
            em = 4 * U32 * (0.9 * old[1][i].abs() + 0.1 * gd.abs())
            ev = 6 * U32 * want[2]
            assert_within(opt.m[i], (want[1], em), f"m {n}")
            assert_within(opt.v[i], (want[2], ev + 1e-44), f"v {n}")
            up = (want[0] - old[0][i] * (1 - HYPER["lr"] * HYPER["weight_decay"])).abs()
            rel_m = em / want[1].abs().clamp(min=1e-300)
            ep = up * (12 * U32 + rel_m) + 4 * U32 * old[0][i].abs()
            stored = unit(p_type) * (want[0].abs() + ep)
            assert_within(p[i], (want[0], ep + stored), f"p {n}")
            if copies:
                assert torch.equal(extra[i], p[i].to(torch.bfloat16))


@pytest.mark.parametrize("p_type", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("g_type", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 1])
def test_32_bits(gpu, p_type, g_type, offset):
    check_32(SIZES, p_type, g_type, copies=p_type == torch.float32, offset=offset)


def test_more_tensors_than_a_launch_takes(gpu):
    check_32([1 + 37 * i for i in range(131)], steps=1)


def test_no_tensors(gpu):
    import nnh
    nnh.AdamW([], [], **HYPER).step()
    check_32([0, 0])


@pytest.mark.parametrize("p_type", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("g_type", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 1])
def test_8_bits(gpu, p_type, g_type, offset):
    import nnh
    p, g = tensors(SIZES, 2, p_type, g_type, offset)
    for x in g:  # gradients over many orders of magnitude, within a block and between blocks, and zeros
        if x.numel() > 100:
            x *= torch.exp2(torch.arange(x.numel(), device="cuda") % 50 - 40.0).to(g_type)
            x[70:75] = 0
    m = [torch.zeros(x.numel() + offset, dtype=torch.uint8, device="cuda")[offset:] for x in p]
    v = [torch.zeros_like(x) for x in m]
    opt = nnh.AdamW(p, g, m=m, v=v, m_scale=[torch.zeros((x.numel() + 63) // 64, dtype=torch.uint8, device="cuda") for x in p],
                    v_scale=[torch.zeros((x.numel() + 63) // 64, dtype=torch.uint8, device="cuda") for x in p], **HYPER)
    vals = [[torch.zeros(x.numel(), dtype=torch.float64) for x in p] for _ in range(2)]
    scale = torch.tensor([0.7312], device="cuda")
    for step in range(1, 5):
        old = [x.double().cpu() for x in p]
        opt.step(grad_scale=scale)
        torch.cuda.synchronize()
        for i, n in enumerate(SIZES):
            new, dm, dv = adamw(old[i], g[i].double().cpu(), vals[0][i], vals[1][i], step, scale=float(scale), **HYPER)
            for name, x, root, codes, scales, k in (("m", dm, False, opt.m, opt.m_scale, 0), ("v", dv, True, opt.v, opt.v_scale, 1)):
                want, e, value = block_codes(x, root)
                assert torch.equal(codes[i].cpu().view(torch.float8_e4m3fn).double(), want), (name, n, step)
                assert torch.equal(scales[i].cpu(), e), (name, n, step)
                vals[k][i] = value * value if root else value
            up = (new - old[i] * (1 - HYPER["lr"] * HYPER["weight_decay"])).abs()
            ep = up * 12 * U32 + 4 * U32 * old[i].abs()
            # far below fp32's normal numbers the root of v, itself below them, is 0 or off: eps is what counts there
            tiny = HYPER["lr"] / (1 - 0.9 ** step) * dm.abs() / HYPER["eps"] * (dv < 1e-37)
            assert_within(p[i], (new, ep + tiny + unit(p_type) * (new.abs() + ep + tiny)), f"p {n}")


def test_not_finite_gradients(gpu):
    """An element whose gradient is not finite becomes NaN; its block's others keep their codes."""
    import nnh
    p, g = tensors([128], 3, torch.float32, torch.float32)
    q, h = [p[0].clone()], [g[0].clone()]
    h[0][5], h[0][6] = math.inf, math.nan
    one, two = nnh.AdamW(p, g, bits=8, **HYPER), nnh.AdamW(q, h, bits=8, **HYPER)
    g[0][5] = g[0][6] = 0.0
    one.step()
    two.step()
    keep = torch.ones(128, dtype=torch.bool)
    keep[5:7] = False
    for a, b in ((one.m, two.m), (one.v, two.v)):
        assert torch.equal(a[0].cpu()[keep], b[0].cpu()[keep])
        assert bool(torch.isnan(b[0].cpu()[5:7].view(torch.float8_e4m3fn).float()).all())
    assert torch.equal(one.m_scale[0], two.m_scale[0]) and torch.equal(one.v_scale[0], two.v_scale[0])
    assert torch.equal(p[0].cpu()[keep], q[0].cpu()[keep]) and bool(torch.isnan(q[0].cpu()[5:7]).all())


def test_device_options_and_capture(gpu):
    """lr, the step's number and the gradients' factor from device memory; the step captured once and replayed with
    eager work between equals eager steps."""
    import nnh
    for bits in (32, 8):
        p, g = tensors([100, 5000], 4, torch.float32, torch.float32)
        q, h = [x.clone() for x in p], [x.clone() for x in g]
        one, two = nnh.AdamW(p, g, bits=bits, **HYPER), nnh.AdamW(q, h, bits=bits, **HYPER)
        lr, count, scale = torch.zeros(1, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), torch.ones(1, device="cuda")
        stream = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            two.step(grad_scale=scale, lr_device=lr, step_device=count)
        for step in range(1, 5):
            one.lr = float(torch.tensor(1e-3 * step))
            lr.fill_(1e-3 * step)
            count.fill_(step)
            scale.fill_(0.5 + 0.1 * step)
            for x, y in zip(g, h):
                x.mul_(-0.9)
                y.copy_(x)
            one.step(grad_scale=scale)
            graph.replay()
            torch.cuda.synchronize()
            for x, y in zip(one.m + one.v, two.m + two.v):
                assert torch.equal(x, y), (bits, step)
            for x, y in zip(p, q):  # the bias corrections' powers are computed on the device there
                torch.testing.assert_close(x, y, rtol=4 * U32, atol=1e-3 * step * 8 * U32)


def test_large_tensor(gpu):
    """More than 2^32 bytes in one tensor: the last elements."""
    import nnh
    n = (1 << 30) + 1000
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g[-5:] = torch.tensor([1.0, -2.0, 3.0, 0.5, 4.0], device="cuda").bfloat16()
    opt = nnh.AdamW([p], [g], bits=8, **HYPER)
    opt.step()
    want = -HYPER["lr"] * torch.sign(g[-5:].float())  # the first step's size, m / sqrt(v) = 1
    torch.testing.assert_close(p[-5:], want, rtol=1e-6, atol=0)
    assert int((p != 0).sum()) == 5 and int((opt.m[0] != 0).sum()) == 5
