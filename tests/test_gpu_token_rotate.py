"""GPU: per-head RMS norm with position rotation (csrc/qk_rotate.hip, opencood_iface/token_attention.py) against 64-bit formulas.

Tolerance of the fp32 arithmetic, relative to the size of the rotated pair: mean of squares and rsqrt <= 8 x 2^-24, gamma and the turn's products
4 x 2^-24, the angle's fp32 rest 2 pi 2^-26, cos / sin 2 ulp = 2^-23: together < 1.1e-6; 1.5e-6 is used.  A 16-bit result adds half its step.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TOL = 1.5e-6
EPS = 1e-6


def half(dt):
    return torch.finfo(dt).eps / 2


def ref(x, gamma, pos, freqs, inter, axes):
    """64-bit forward, written with complex numbers."""
    x, gamma = x.double(), gamma.double()
    d = x.shape[-1]
    u = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * gamma
    i = torch.arange(d // 2)
    ang = 2 * math.pi * torch.remainder(pos.double()[:, i // (d // 2 // axes)] * freqs, 1.0)
    z = torch.view_as_complex(u.unflatten(-1, (d // 2, 2)).contiguous()) if inter else torch.complex(u[..., :d // 2].contiguous(), u[..., d // 2:].contiguous())
    z = z * torch.polar(torch.ones_like(ang), ang)[:, None]
    return torch.view_as_real(z).flatten(-2) if inter else torch.cat([z.real, z.imag], -1)


def close(got, want, dt, what, scale=None, extra=1.0):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape, what
    scale = want.abs().amax(-1, keepdim=True) if scale is None else scale
    tol = half(dt) * (1 if dt != torch.float32 else 0) * want.abs() + TOL * extra * scale
    bad = (got - want).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {float(((got - want).abs() / tol.clamp_min(1e-300)).max()):.2f} x the tolerance"


def case(seed, rows, h, kv, d, dt, axes, far=0):
    from airv2x_perception_amd.opencood_iface import token_attention as A
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, h + 2 * kv, d, generator=g) * torch.randn(rows, 1, 1, generator=g).exp()).to(dt)
    gq, gk = 1 + 0.2 * torch.randn(d, generator=g), 1 + 0.2 * torch.randn(d, generator=g)
    pos = (torch.randint(0, 400, (rows, axes), generator=g) + far).int()
    return x, gq, gk, pos, A.rotation_freqs(d, axes)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,h,kv,d,axes,inter,far", [(1, 8, 8, 32, 2, False, 0), (77, 4, 1, 64, 1, True, 10 ** 6), (513, 16, 16, 16, 2, False, -500),
                                                          (65, 3, 3, 128, 2, True, 0), (9, 12, 4, 32, 2, False, 2 ** 31 - 500), (2, 1, 1, 128, 1, False, 7)])
def test_forward_and_gradients(dt, rows, h, kv, d, axes, inter, far):
    from airv2x_perception_amd.opencood_iface import token_attention as A
    x, gq, gk, pos, freqs = case(rows + d, rows, h, kv, d, dt, axes, far)
    g = torch.Generator().manual_seed(1)
    doq, dok, dov = (torch.randn(rows, n, d, generator=g).to(dt) for n in (h, kv, kv))
    xr, gqr, gkr = x.double().requires_grad_(), gq.double().requires_grad_(), gk.double().requires_grad_()
    rq, rk = ref(xr[:, :h], gqr, pos, freqs, inter, axes), ref(xr[:, h:h + kv], gkr, pos, freqs, inter, axes)
    want = torch.autograd.grad([rq, rk, xr[:, h + kv:]], [xr, gqr, gkr], [doq.double(), dok.double(), dov.double()])
    xd, gqd, gkd = x.cuda().requires_grad_(), gq.cuda().requires_grad_(), gk.cuda().requires_grad_()
    q, k, v = A.qkv_norm_rotate(xd, h, kv, gqd, gkd, pos.cuda(), freqs.cuda(), EPS, inter)
    close(q, rq, dt, "q")
    close(k, rk, dt, "k")
    assert torch.equal(v, xd[:, h + kv:])
    got = torch.autograd.grad([q, k, v], [xd, gqd, gkd], [doq.cuda(), dok.cuda(), dov.cuda()])
    # dx = (g - n mean(g n)) r: three terms of the size of r |g|, each with the forward's relative error, a cancellation of at most r (|g| + |n| |g|)
    r = 1 / (xr.detach().square().mean(-1, keepdim=True) + EPS).sqrt()
    gn = torch.cat([doq.double().norm(dim=-1, keepdim=True), dok.double().norm(dim=-1, keepdim=True), torch.zeros(rows, kv, 1, dtype=torch.double)], 1)
    close(got[0], want[0], dt, "dx", scale=r * gn * 2, extra=2.0)
    for a, b, n, do in ((got[1], want[1], h, doq), (got[2], want[2], kv, dok)):
        # sums over rows x heads: every term off by TOL of |du n|, the sum's own roundings by (rows / 2048 + 16) steps of sum |terms|
        terms = do.double().abs().sum((0, 1)).max() * 2.0
        assert float((a.cpu().double() - b).abs().max()) <= float(terms) * (TOL + 20 * 2 ** -24)
    # the two-tensor form from views of the same buffer: the same bits
    q2, k2 = A.qk_norm_rotate(xd.detach()[:, :h], xd.detach()[:, h:h + kv], gqd.detach(), gkd.detach(), pos.cuda(), freqs.cuda(), EPS, inter)
    assert torch.equal(q2, q) and torch.equal(k2, k)
    qs, ks = xd.detach()[:, :h].contiguous().requires_grad_(), xd.detach()[:, h:h + kv].contiguous().requires_grad_()
    q3, k3 = A.qk_norm_rotate(qs, ks, gqd, gkd, pos.cuda(), freqs.cuda(), EPS, inter)
    d3 = torch.autograd.grad([q3, k3], [qs, ks, gqd, gkd], [doq.cuda(), dok.cuda()])
    assert torch.equal(d3[0], got[0][:, :h]) and torch.equal(d3[1], got[0][:, h:h + kv]) and torch.equal(got[0][:, h + kv:].cpu(), dov)
    assert torch.equal(d3[2], got[1]) and torch.equal(d3[3], got[2])


def test_gradient_against_differences():
    from airv2x_perception_amd.opencood_iface import token_attention as A
    x, gq, gk, pos, freqs = case(5, 6, 2, 1, 16, torch.float32, 2)
    x, gq, gk, pos, freqs = x.cuda(), gq.cuda(), gk.cuda(), pos.cuda(), freqs.cuda()
    w = torch.randn(6, 2, 16, generator=torch.Generator().manual_seed(2)).cuda()
    f = lambda q: (A.qk_norm_rotate(q, None, gq, None, pos, freqs)[0].double() * w).sum()
    q = x[:, :2].clone().requires_grad_()
    f(q).backward()
    step = torch.randn(6, 2, 16, generator=torch.Generator().manual_seed(3)).cuda() * q.detach().abs().mean((1, 2), keepdim=True)
    e = 1e-3
    diff = float(f(q.detach() + e * step) - f(q.detach() - e * step)) / (2 * e)
    ana = float((q.grad * step).sum())
    # third derivative e^2 ~ 1e-6 of the size of the sum, fp32 values 6e-8 / e
    size = float((q.grad.abs() * step.abs()).sum())
    assert abs(diff - ana) <= size * 2e-4


def test_empty_inputs_batched_shapes_and_odd_strides():
    from airv2x_perception_amd.opencood_iface import token_attention as A
    x, gq, gk, pos, freqs = case(3, 12, 4, 2, 32, torch.bfloat16, 2)
    dev = [t.cuda() for t in (gq, gk, pos, freqs)]
    e = torch.zeros(0, 8, 32, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    gqd = gq.cuda().requires_grad_()
    q, k, v = A.qkv_norm_rotate(e, 4, 2, gqd, dev[1], pos.cuda()[:0], dev[3])
    assert q.shape == (0, 4, 32) and k.shape == (0, 2, 32) and v.shape == (0, 2, 32)
    d, dg = torch.autograd.grad(q.sum(), [e, gqd])
    assert d.shape == e.shape and not dg.any()
    xd = x.cuda()
    q0, k0 = A.qk_norm_rotate(xd[:, :4], xd[:, 4:6], dev[0], dev[1], dev[2], dev[3])
    # (B, T, H, D) with the batch in front
    q1, k1 = A.qk_norm_rotate(xd.view(3, 4, 8, 32)[:, :, :4], xd.view(3, 4, 8, 32)[:, :, 4:6], dev[0], dev[1], dev[2].view(3, 4, 2), dev[3])
    assert torch.equal(q1.flatten(0, 1), q0) and torch.equal(k1.flatten(0, 1), k0)
    # a last axis that is not contiguous, a head stride that is odd, an address between two groups of four
    wide = torch.zeros(12, 8, 64, device="cuda", dtype=torch.bfloat16)
    wide[:, :, ::2] = xd
    odd = torch.zeros(12, 8, 33, device="cuda", dtype=torch.bfloat16)
    odd[:, :, :32] = xd
    off = torch.zeros(12 * 8 * 32 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(12, 8, 32)
    off.copy_(xd)
    for y in (wide[:, :, ::2], odd[:, :, :32], off):
        q1, k1 = A.qk_norm_rotate(y[:, :4], y[:, 4:6], *dev)
        assert torch.equal(q1, q0) and torch.equal(k1, k0)
    # zeros stay zeros, an infinity or a NaN stays in its own head vector
    y = xd.clone()
    y[2, 1], y[3, 2, 5], y[4, 3, 6] = 0, float("nan"), float("inf")
    q1, _ = A.qk_norm_rotate(y[:, :4], y[:, 4:6], *dev)
    assert not q1[2, 1].any() and q1[3, 2].isnan().all() and q1[4, 3].isnan().any()
    same = torch.ones(12, 4, dtype=torch.bool)
    same[2, 1] = same[3, 2] = same[4, 3] = False
    assert torch.equal(q1.cpu()[same], q0.cpu()[same])


def test_graph_replay():
    from airv2x_perception_amd.opencood_iface import token_attention as A
    x, gq, gk, pos, freqs = [t.cuda() for t in case(8, 300, 8, 8, 32, torch.bfloat16, 2)]
    buf = torch.zeros_like(x).requires_grad_()
    do = torch.randn(300, 8, 32, device="cuda").bfloat16()

    def step():
        q, k, v = A.qkv_norm_rotate(buf, 8, 8, gq, gk, pos, freqs)
        return torch.autograd.grad([q, k], [buf], [do, do])[0], q.detach()

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        with torch.no_grad():
            buf.copy_(x * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        a, b = got[0].clone(), got[1].clone()
        want = step()
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])
