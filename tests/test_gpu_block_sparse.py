"""GPU: bounds, selection and attention over selected blocks (csrc/block_sparse.hip, opencood_iface/token_attention.py) against 64-bit formulas.

Bounds and selections are exact (whole numbers).  Attention: a score is off by at most e = D 2^-24 sum |q k| scale (products added in fp32), a probability by
2 e + 2^-21 of itself (numerator, denominator, exp2; 16-bit types hold it in two terms: 2^-16), a sum over keys by 40 x 2^-24 of the sum of sizes.  A 16-bit
result adds half its step, and without gradients the parts it is joined from (one a block, a convex combination: at most sum of p |v|) half a step each.  fp32 runs on two fp16 terms of values relative to the largest of a row or block: 2^-22 of those.  fp16 has no steps below 2^-24: a result is off by 2^-25 there, and a
probability or dS, held relative to the largest of its tile (at most a factor of 2 above it), by 2^-24 of that largest one.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF, HF = torch.float32, torch.bfloat16, torch.float16


def make(seed, b, t, n, h, kv, d, dt, masked=None):
    g = torch.Generator().manual_seed(seed)
    nb = (n + 63) // 64
    mid = torch.randn(b, nb, kv, d, generator=g)
    q = torch.randn(b, t, h, d, generator=g).to(dt)
    k = (0.8 * mid[:, torch.arange(n) // 64] + 0.6 * torch.randn(b, n, kv, d, generator=g)).to(dt)
    v = torch.randn(b, n, kv, d, generator=g).to(dt)
    do = torch.randn(b, t, h, d, generator=g).to(dt)
    mask = None
    if masked:
        mask = torch.rand(b, n, generator=g) < 0.8
        mask[:, 64:128] = False                       # a block that nobody sees
        if masked == "empty":
            mask[-1] = False                          # a sample without keys
    return q, k, v, do, mask


def bounds_of(k, mask):
    b, n, kv, d = k.shape
    nb = (n + 63) // 64
    ints, scale = torch.zeros(b, kv, nb, 2, d), torch.full((b, kv, nb), -1.0)
    for i in range(b):
        for j in range(nb):
            rows = torch.arange(j * 64, min(n, j * 64 + 64))
            if mask is not None:
                rows = rows[mask[i, rows]]
            if len(rows):
                x = k[i, rows].float()
                hi, lo = x.amax(0), x.amin(0)
                big = torch.maximum(hi.abs(), lo.abs()).amax(-1)
                m = torch.full_like(big, 127.0)
                r = (m / big.clamp_min(1e-30))[:, None]
                ints[i, :, j, 0], ints[i, :, j, 1] = (hi * r).round().clamp(-127, 127), (lo * r).round().clamp(-127, 127)
                scale[i, :, j] = big / m
    return ints.half(), scale


def chosen_of(q, ints, scale, n):
    b, t, h, d = q.shape
    kv = scale.shape[1]
    x = q.float().view(b, t, kv, h // kv, d)
    big = x.abs().amax((-1, -2), keepdim=True)
    x = (x * (torch.full_like(big, 127.0) / big.clamp_min(1e-30))).round().clamp(-127, 127).long()
    u, l = ints[:, :, :, 0].long(), ints[:, :, :, 1].long()
    out = torch.full((b, t, kv, n), -1, dtype=torch.int32)
    for i in range(b):
        for c in range(kv):
            s = torch.einsum("tgd,jd->tj", x[i, :, c].clamp_min(0), u[i, c]) + torch.einsum("tgd,jd->tj", x[i, :, c].clamp_max(0), l[i, c])
            assert int(s.abs().max() if s.numel() else 0) < 1 << 24
            f = s.float() * scale[i, c]
            for r in range(t):
                order = sorted((j for j in range(len(scale[i, c])) if scale[i, c, j] >= 0), key=lambda j: (-float(f[r, j]), j))[:n]
                out[i, r, c, :len(order)] = torch.tensor(sorted(order), dtype=torch.int32)
    return out


def dense(q, k, v, blocks, mask, scale):
    """How often every key counts for a (query, head), and 64-bit attention with it."""
    b, t, h, d = q.shape
    n, kv = k.shape[1:3]
    nb = (n + 63) // 64
    cnt = torch.zeros(b, t, kv, nb + 1, dtype=torch.double)
    idx = torch.where((blocks >= 0) & (blocks < nb), blocks, torch.full_like(blocks, nb)).long()
    cnt.scatter_add_(3, idx, torch.ones(idx.shape, dtype=torch.double))
    cnt = cnt[..., :nb].repeat_interleave(64, 3)[..., :n]
    if mask is not None:
        cnt = cnt * mask[:, None, None].double()
    cnt = cnt.repeat_interleave(h // kv, 2)                                                  # (B, T, H, N)
    kk, vv = k.repeat_interleave(h // kv, 2), v.repeat_interleave(h // kv, 2)
    s = torch.einsum("bthd,bnhd->bthn", q, kk) * scale
    top = s.masked_fill(cnt == 0, -math.inf).amax(-1, keepdim=True).clamp_min(-1e300)
    e = cnt * torch.exp((s - top).masked_fill(cnt == 0, 0.0))
    p = e / e.sum(-1, keepdim=True).clamp_min(1e-300)
    return p, torch.einsum("bthn,bnhd->bthd", p, vv), kk, vv


def check(q, k, v, do, blocks, mask, dt, scale=None, grads=True):
    from airv2x_perception_amd.opencood_iface import token_attention as A
    b, t, h, d = q.shape
    n, kv = k.shape[1:3]
    sc = 1 / math.sqrt(d) if scale is None else scale
    half = torch.finfo(dt).eps / 2 if dt != F32 else 0.0
    least, flat = (2.0 ** -25, 2.0 ** -24) if dt == HF else (1e-30, 0.0)
    Q, K, V = (x.double().requires_grad_(grads) for x in (q, k, v))
    p, o, kk, vv = dense(Q, K, V, blocks, mask, sc)
    dev = [x.cuda().requires_grad_(grads) for x in (q, k, v)]
    got = A.block_sparse_attention(*dev, blocks.cuda(), None if mask is None else mask.cuda(), scale)
    with torch.no_grad():
        es = d * U * torch.einsum("bthd,bnhd->bthn", Q.abs(), kk.abs()) * abs(sc)
        es = es.masked_fill(p == 0, 0.0).amax(-1, keepdim=True) * 2
        ep = es + 2.0 ** -21 + (2.0 ** -16 if dt != F32 else 0.0)
        po = torch.einsum("bthn,bnhd->bthd", p, vv.abs())
        exact = po * (ep * 2 + 40 * U)                # before any rounding to 16 bits
        ob = exact + (0 if grads else half) * po + half * o.abs() + least + flat * p.amax(-1, keepdim=True) * (p > 0).double().matmul(torch.ones(n, d, dtype=torch.double)) * vv.abs().max()
    far = ((got.detach().double().cpu() - o.detach()).abs() / ob).max()
    assert float(far) <= 1, f"out: {float(far):.2f} x the bound"
    if not grads:
        return got
    dO = do.double()
    want = torch.autograd.grad(o, [Q, K, V], dO)
    grad = torch.autograd.grad(got, dev, do.cuda())
    with torch.no_grad():
        g = h // kv
        dp = torch.einsum("bthd,bnhd->bthn", dO, vv)
        dpb = torch.einsum("bthd,bnhd->bthn", dO.abs(), vv.abs())
        delta = (dO * o).sum(-1, keepdim=True)
        # the output with its rounding error beside it: half a step of half a step is left
        deltab = (dO.abs() * (exact + least + half * half * o.abs())).sum(-1, keepdim=True) + (dO.abs() * o.abs()).sum(-1, keepdim=True) * 8 * U
        ds = p * (dp - delta) * abs(sc)
        dsb = ds.abs() * 2 * ep + p * (dpb * d * U * 2 + deltab + (dp.abs() + delta.abs()) * 2 * U) * abs(sc) + ds.abs() * (2.0 ** -16 if dt != F32 else 0) + flat * ds.abs().max() * (p > 0)
        fold = lambda x: x.view(b, n, kv, g, d).sum(3)
        size = lambda e, x: torch.einsum("bthn,bthd->bnhd", e, x)
        bq = torch.einsum("bthn,bnhd->bthd", dsb + 40 * U * ds.abs(), kk.abs())
        bk = fold(size(dsb + 40 * U * ds.abs(), Q.abs()))
        bv = fold(size(p * (2 * ep + 40 * U) + flat * (p > 0), dO.abs()))
    for name, a, w, bound in zip(("dq", "dk", "dv"), grad, want, (bq, bk, bv)):
        far = ((a.double().cpu() - w).abs() / (bound + half * w.abs() + least)).max()
        assert float(far) <= 1, f"{name}: {float(far):.2f} x the bound"
    again = torch.autograd.grad(A.block_sparse_attention(*dev, blocks.cuda(), None if mask is None else mask.cuda(), scale), dev, do.cuda())
    assert all(torch.equal(x, y) for x, y in zip(grad, again))
    return got


@pytest.mark.parametrize("dt", [F32, BF, HF])
@pytest.mark.parametrize("n,kv,d,masked", [(1, 1, 16, None), (64, 2, 32, None), (700, 3, 64, "some"), (333, 2, 128, "empty"), (1030, 8, 32, "some")])
def test_bounds(dt, n, kv, d, masked):
    from airv2x_perception_amd.opencood_iface import token_attention as A
    _, k, _, _, mask = make(n, 2, 1, n, kv, kv, d, dt, masked)
    ints, scale = bounds_of(k, mask)
    dead = k.clone()
    if mask is not None:
        dead[~mask] = float("nan")                     # masked places are not read
    got = A.block_bounds(dead.cuda(), None if mask is None else mask.cuda())
    assert torch.equal(got.scale.cpu(), scale) and torch.equal(got.ints.cpu(), ints)
    # a cache that changes: only the touched blocks are redone
    k2 = k.clone()
    lo, hi = n // 3, max(n // 3 + 1, n // 2)
    k2[:, lo:hi] *= -3
    A.update_block_bounds(got, k2.cuda(), lo, hi, None if mask is None else mask.cuda())
    ints, scale = bounds_of(k2, mask)
    assert torch.equal(got.scale.cpu(), scale) and torch.equal(got.ints.cpu(), ints)


@pytest.mark.parametrize("dt,t,n,h,kv,d,blocks,masked", [(F32, 1, 1, 1, 1, 16, 1, None), (BF, 17, 700, 8, 8, 32, 4, "some"), (HF, 33, 2500, 8, 2, 64, 64, "empty"),
                                                        (F32, 5, 35000, 2, 1, 16, 9, None), (HF, 70, 35000, 2, 2, 32, 16, None), (BF, 33, 900, 4, 2, 128, 12, "empty"), (BF, 16, 130, 4, 4, 128, 3, "some"), (F32, 3, 4000, 16, 1, 64, 63, "some")])
def test_selection(dt, t, n, h, kv, d, blocks, masked):
    from airv2x_perception_amd.opencood_iface import token_attention as A
    q, k, _, _, mask = make(t + n, 2, t, n, h, kv, d, dt, masked)
    q[0, 0] = 0                                        # every score is zero: the lowest blocks
    bounds = A.block_bounds(k.cuda(), None if mask is None else mask.cuda())
    got = A.select_blocks(q.cuda(), bounds, blocks).cpu()
    assert torch.equal(got, chosen_of(q, bounds.ints.cpu(), bounds.scale.cpu(), blocks))
    wide = torch.zeros(2, t, h, d + 1, dtype=dt, device="cuda")      # odd strides
    wide[..., :d] = q.cuda()
    assert torch.equal(A.select_blocks(wide[..., :d], bounds, blocks).cpu(), got)


def test_selection_of_equal_scores_and_of_odd_values():
    from airv2x_perception_amd.opencood_iface import token_attention as A
    k = torch.ones(1, 64 * 1300, 1, 16)                # 1300 equal blocks: three chunks of scores
    bounds = A.block_bounds(k.cuda())
    q = torch.randn(1, 20, 1, 16)
    got = A.select_blocks(q.cuda(), bounds, 7).cpu()
    assert torch.equal(got, torch.arange(7, dtype=torch.int32).expand(1, 20, 1, 7))
    k[0, 64 * 600:64 * 601] = 2                         # and one that beats them for positive sums
    bounds = A.block_bounds(k.cuda())
    got = A.select_blocks(q.abs().cuda(), bounds, 3).cpu()
    assert torch.equal(got, torch.tensor([0, 1, 600], dtype=torch.int32).expand(1, 20, 1, 3))
    # NaN and infinities: some choice, in range and ascending
    q[0, 1], q[0, 2, 0, 3], q[0, 3] = float("nan"), float("inf"), 1e-40
    k[0, 5], k[0, 64 * 9 + 1] = float("nan"), float("inf")
    got = A.select_blocks(q.cuda(), A.block_bounds(k.cuda()), 5).cpu()
    assert ((got >= 0) & (got < 1300)).all() and (got.diff(dim=-1) > 0).all()


@pytest.mark.parametrize("blocks", [1, 5, 16, 17])
def test_selection_where_every_block_beats_the_ones_before(blocks):
    """Scores that rise with the block for half of the queries and fall for the others, over three chunks and in ranges: every score is a newcomer."""
    from airv2x_perception_amd.opencood_iface import token_attention as A
    nb = 1300
    k = (1 + torch.arange(nb).repeat_interleave(64) / nb)[None, :, None, None] * torch.ones(1, 1, 1, 16)
    for t in (40, 5000):                               # ranges joined; one workgroup for all blocks
        q = torch.rand(1, t, 1, 16, generator=torch.Generator().manual_seed(t)) + 0.1
        q[:, 1::2] *= -1
        got = A.select_blocks(q.cuda(), A.block_bounds(k.cuda()), blocks).cpu()[0, :, 0]
        low = torch.arange(blocks, dtype=torch.int32)
        assert torch.equal(got[::2], (low + nb - blocks).expand(t // 2, blocks)) and torch.equal(got[1::2], low.expand(t // 2, blocks))


@pytest.mark.parametrize("dt", [F32, BF, HF])
@pytest.mark.parametrize("b,t,n,h,kv,d,blocks,masked", [(1, 1, 1, 1, 1, 16, 1, None), (2, 1, 700, 8, 8, 32, 4, "some"), (2, 37, 333, 4, 2, 64, 3, "empty"), (1, 5, 130, 16, 1, 64, 8, None),
                                                       (1, 130, 200, 3, 3, 16, 5, "some"), (1, 9, 257, 2, 2, 128, 2, None)])
def test_attention_few_queries(dt, b, t, n, h, kv, d, blocks, masked):
    from airv2x_perception_amd.opencood_iface import token_attention as A
    q, k, v, do, mask = make(t + n, b, t, n, h, kv, d, dt, masked)
    chosen = A.select_blocks(q.cuda(), A.block_bounds(k.cuda(), None if mask is None else mask.cuda()), blocks).cpu()
    assert b * t * kv * blocks <= A.FEW_MENTIONS
    check(q, k, v, do, chosen, mask, dt)
    check(q, k, v, do, chosen, mask, dt, grads=False)


@pytest.mark.parametrize("dt", [F32, BF, HF])
@pytest.mark.parametrize("b,t,n,h,kv,d,blocks,masked", [(1, 600, 700, 4, 4, 32, 4, None), (2, 300, 333, 4, 2, 64, 3, "empty"), (1, 257, 130, 8, 1, 16, 3, "some"), (1, 150, 200, 2, 2, 128, 4, "some"),
                                                       (1, 700, 64, 3, 3, 16, 2, None)])
def test_attention_many_queries(monkeypatch, dt, b, t, n, h, kv, d, blocks, masked):
    from airv2x_perception_amd.opencood_iface import token_attention as A
    monkeypatch.setattr(A, "FEW_MENTIONS", 0)
    q, k, v, do, mask = make(t + n, b, t, n, h, kv, d, dt, masked)
    chosen = A.select_blocks(q.cuda(), A.block_bounds(k.cuda(), None if mask is None else mask.cuda()), blocks).cpu()
    check(q, k, v, do, chosen, mask, dt)
    check(q, k, v, do, chosen, mask, dt, grads=False)


@pytest.mark.parametrize("few", [0, 1 << 30])
@pytest.mark.parametrize("dt", [F32, BF])
def test_any_choice_of_blocks(monkeypatch, few, dt):
    """Indices out of range, unordered, twice, none at all; what masked and unnamed places hold is never read; another scale."""
    from airv2x_perception_amd.opencood_iface import token_attention as A
    monkeypatch.setattr(A, "FEW_MENTIONS", few)
    q, k, v, do, mask = make(11, 2, 40, 400, 4, 2, 32, dt, "some")
    g = torch.Generator().manual_seed(2)
    blocks = torch.randint(-3, 9, (2, 40, 2, 6), generator=g).int()         # 7 blocks: -3 .. -1, 7, 8 are none
    blocks[0, 3] = -1
    blocks[0, 4] = 2 ** 31 - 1
    blocks[0, 5] = -2 ** 31
    blocks[0, 6] = 1                                                          # an invisible block, six times
    blocks[1, 7] = 4                                                          # one block, six times
    named = torch.zeros(2, 7, dtype=torch.bool)
    for i in range(2):
        for j in blocks[i].unique():
            if 0 <= j < 7:
                named[i, j] = True
    check(q, k, v, do, blocks, mask, dt, scale=-0.3, grads=False)
    out = check(q, k, v, do, blocks, mask, dt, scale=-0.3)
    assert not out[0, 3:7].any()
    kk, vv = k.clone(), v.clone()
    kk[~mask], vv[~mask] = float("nan"), float("inf")
    dev = [x.cuda().requires_grad_() for x in (q, kk, vv)]
    again = A.block_sparse_attention(*dev, blocks.cuda(), mask.cuda(), -0.3)
    assert torch.equal(again, out)
    for x in torch.autograd.grad(again, dev, do.cuda()):
        assert x.isfinite().all()
    assert not torch.autograd.grad(A.block_sparse_attention(*dev, blocks.cuda(), mask.cuda(), -0.3), dev, do.cuda())[1].cpu()[~mask].any()


@pytest.mark.parametrize("few", [0, 1 << 30])
def test_strides_and_empty_inputs(monkeypatch, few):
    from airv2x_perception_amd.opencood_iface import token_attention as A
    monkeypatch.setattr(A, "FEW_MENTIONS", few)
    q, k, v, do, _ = make(5, 1, 50, 300, 4, 4, 32, BF)
    blocks = A.select_blocks(q.cuda(), A.block_bounds(k.cuda()), 3)
    want = A.block_sparse_attention(q.cuda(), k.cuda(), v.cuda(), blocks)
    buf = torch.zeros(1, 300, 12, 32, dtype=BF, device="cuda")                # a fused projection
    buf[:, :50, :4], buf[:, :, 4:8], buf[:, :, 8:] = q.cuda(), k.cuda(), v.cuda()
    assert torch.equal(A.block_sparse_attention(buf[:, :50, :4], buf[:, :, 4:8], buf[:, :, 8:], blocks), want)
    bt = k.cuda().permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)          # channels apart
    hd = v.cuda().transpose(1, 2).contiguous().transpose(1, 2)                  # heads outside tokens
    assert torch.equal(A.block_sparse_attention(q.cuda(), bt, hd, blocks), want)
    off = torch.zeros(q.numel() + 3, dtype=BF, device="cuda")[3:].view(q.shape)
    off.copy_(q)
    assert torch.equal(A.block_sparse_attention(off, k.cuda(), v.cuda(), blocks), want)
    one = q.cuda()[:, :, :1].expand(1, 50, 4, 32)                               # one query for all heads
    assert torch.equal(A.block_sparse_attention(one, k.cuda(), v.cuda(), blocks), A.block_sparse_attention(one.contiguous(), k.cuda(), v.cuda(), blocks))
    # no queries, no keys
    e = A.block_sparse_attention(q.cuda()[:, :0], k.cuda(), v.cuda(), blocks[:, :0])
    assert e.shape == (1, 0, 4, 32)
    qr = q.cuda().requires_grad_()
    none = A.block_bounds(k.cuda()[:, :0])
    bl = A.select_blocks(qr, none, 2)
    assert (bl == -1).all()
    z = A.block_sparse_attention(qr, k.cuda()[:, :0], v.cuda()[:, :0], bl)
    assert z.shape == q.shape and not z.any() and not torch.autograd.grad(z.sum(), qr)[0].any()
    # a NaN of one query stays there
    bad = q.cuda().clone()
    bad[0, 7, 2, 3] = float("nan")
    out = A.block_sparse_attention(bad, k.cuda(), v.cuda(), blocks)
    same = torch.ones(50, 4, dtype=torch.bool)
    same[7, 2] = False
    assert out[0, 7, 2].isnan().all() and torch.equal(out.cpu()[0][same], want.cpu()[0][same])


def test_frozen_keys_and_values():
    from airv2x_perception_amd.opencood_iface import token_attention as A
    q, k, v, do, _ = [x.cuda() if x is not None else None for x in make(15, 1, 50, 300, 4, 2, 32, F32)]
    blocks = A.select_blocks(q, A.block_bounds(k), 3)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    full = torch.autograd.grad(A.block_sparse_attention(*leaves, blocks), leaves, do)
    for i in range(3):
        one = [x.clone().requires_grad_(j == i) for j, x in enumerate((q, k, v))]
        assert torch.equal(torch.autograd.grad(A.block_sparse_attention(*one, blocks), one[i], do)[0], full[i])


def test_gradients_against_differences():
    from airv2x_perception_amd.opencood_iface import token_attention as A
    q, k, v, do, mask = make(25, 1, 30, 300, 4, 2, 16, F32, "some")
    q, k, v, do, mask = [x.cuda() for x in (q, k, v, do, mask)]
    blocks = A.select_blocks(q, A.block_bounds(k, mask), 2)
    f = lambda *x: (A.block_sparse_attention(*x, blocks, mask).double() * do).sum()
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(f(*leaves), leaves)
    g = torch.Generator().manual_seed(3)
    e = 2.0 ** -8
    for i in range(3):
        step = torch.randn(leaves[i].shape, generator=g).cuda()
        up, dn = [q, k, v], [q, k, v]
        up[i], dn[i] = up[i] + e * step, dn[i] - e * step
        diff, ana = float(f(*up) - f(*dn)) / (2 * e), float((grads[i].double() * step).sum())
        size = float((grads[i].double().abs() * step.abs()).sum())
        assert abs(diff - ana) <= size * 2e-4           # e^2 / 6 times third derivatives of order ten; fp32 noise 1e-7 / e


def test_crowded_block_and_64_blocks(monkeypatch):
    """Every query names block 2 (its list is cut into work items), and 64 blocks a query."""
    from airv2x_perception_amd.opencood_iface import token_attention as A
    monkeypatch.setattr(A, "FEW_MENTIONS", 0)
    q, k, v, do, _ = make(35, 1, 1500, 64 * 70 - 5, 2, 2, 16, F32)
    blocks = torch.full((1, 1500, 2, 2), 2, dtype=torch.int32)
    blocks[..., 1] = torch.randint(3, 70, (1, 1500, 2), generator=torch.Generator().manual_seed(1)).int()
    check(q[:, :1500], k, v, do, blocks, None, F32)
    chosen = A.select_blocks(q.cuda()[:, :20], A.block_bounds(k.cuda()), 64)
    check(q[:, :20], k, v, do[:, :20], chosen.cpu(), None, F32)


def test_both_forms_on_another_stream_and_in_two_graphs(monkeypatch):
    from airv2x_perception_amd.opencood_iface import token_attention as A
    q, k, v, do, mask = [x.cuda() for x in make(45, 2, 200, 900, 8, 4, 32, BF, "some")]
    buf = [x.clone().requires_grad_() for x in (q, k, v)]

    def step():
        blocks = A.select_blocks(buf[0], A.block_bounds(buf[1], mask), 4)
        out = A.block_sparse_attention(*buf, blocks, mask)
        return [out.detach(), blocks] + list(torch.autograd.grad(out, buf, do))

    for few in (0, 1 << 30):
        monkeypatch.setattr(A, "FEW_MENTIONS", few)
        want = step()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            other = step()
        torch.cuda.current_stream().wait_stream(s)
        assert all(torch.equal(a, b) for a, b in zip(want, other))
        graphs = []
        for _ in range(2):                              # two graphs, each with workspaces of its own
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                got = step()
            graphs.append((graph, got))
        for i in range(3):
            with torch.no_grad():
                buf[0].copy_(q * (1 + i))
                buf[2].copy_(v.roll(i, 1))
            for graph, _ in graphs:
                graph.replay()
            torch.cuda.synchronize()
            kept = [[t.clone() for t in got] for _, got in graphs]
            want = step()
            assert all(torch.equal(a, b) for got in kept for a, b in zip(got, want))


@pytest.mark.parametrize("few", [0, 1 << 30])
def test_the_most_keys(monkeypatch, few):
    """32768 blocks: the choice is the formula's, and attention over them is bit for bit that over the chosen ones alone."""
    from airv2x_perception_amd.opencood_iface import token_attention as A
    monkeypatch.setattr(A, "FEW_MENTIONS", few)
    n = 64 * 32768
    q, k, v, do, _ = make(55, 1, 5, 64 * 50, 2, 1, 16, BF)
    g = torch.Generator().manual_seed(5)
    at = torch.randperm(32768, generator=g)[:50].sort()[0]
    big_k, big_v = (torch.full((1, 32768, 64, 1, 16), 0.01, dtype=BF) for _ in range(2))
    big_k[0, at], big_v[0, at] = k.view(50, 64, 1, 16), v.view(50, 64, 1, 16)
    big_k, big_v = big_k.view(1, n, 1, 16).cuda(), big_v.view(1, n, 1, 16).cuda()
    bounds = A.block_bounds(big_k)
    for m in (6, 20):
        blocks = A.select_blocks(q.cuda(), bounds, m)
        assert torch.equal(blocks.cpu(), chosen_of(q, bounds.ints.cpu(), bounds.scale.cpu(), m))
    blocks = at[torch.randint(0, 50, (1, 5, 1, 9), generator=g)].int()
    blocks[0, 0, 0, 0] = 32768                             # one behind the last
    back = torch.full((32769,), -1, dtype=torch.int32)
    back[at] = torch.arange(50, dtype=torch.int32)
    res = []
    for kk, vv, bl in ((big_k, big_v, blocks), (k.cuda(), v.cuda(), back[blocks.long()])):
        leaves = [x.detach().clone().requires_grad_() for x in (q.cuda(), kk, vv)]
        out = A.block_sparse_attention(*leaves, bl.cuda())
        res.append([out.detach()] + list(torch.autograd.grad(out, leaves, do.cuda())))
    assert torch.equal(res[0][0], res[1][0]) and torch.equal(res[0][1], res[1][1])
    for x, y in zip(res[0][2:], res[1][2:]):
        x = x.view(32768, 64, 1, 16)
        assert torch.equal(x[at.cuda()].view_as(y), y)
        x[at.cuda()] = 0
        assert not x.any()
    one_more = big_k.new_zeros(1, n + 1, 1, 16)
    with pytest.raises(ValueError, match="at most"):
        A.block_sparse_attention(q.cuda(), one_more, one_more, blocks.cuda())


@pytest.mark.parametrize("few", [0, 1 << 30])
def test_offsets_beyond_32_bits(monkeypatch, few):
    """Tokens 2^20 + 64 elements apart: the last ones lie 2^31 elements (2^32 bytes) behind the first."""
    from airv2x_perception_amd.opencood_iface import token_attention as A
    monkeypatch.setattr(A, "FEW_MENTIONS", few)
    t, step = 2060, (1 << 20) + 64
    q, k, v, do, mask = [x.cuda() for x in make(65, 1, t, t, 1, 1, 16, BF, "some")]
    buf = torch.empty((t - 1) * step + 64, dtype=BF, device="cuda")
    far = [buf.as_strided((1, t, 1, 16), (0, step, 16, 1), 16 * i) for i in range(3)]
    with torch.no_grad():
        for x, y in zip(far, (q, k, v)):
            x.copy_(y)
    assert far[1][0, -1].data_ptr() - far[1].data_ptr() > 1 << 32
    res = []
    for x in (far, (q, k, v)):
        leaves = [y.detach().requires_grad_() for y in x]
        bounds = A.block_bounds(leaves[1], mask)
        blocks = A.select_blocks(leaves[0], bounds, 3)
        out = A.block_sparse_attention(*leaves, blocks, mask)
        res.append([bounds.ints, bounds.scale, blocks, out.detach()] + list(torch.autograd.grad(out, leaves, do)))
    assert all(torch.equal(x, y) for x, y in zip(*res))


@pytest.mark.parametrize("few", [0, 1 << 30])
def test_tiny_and_huge_sizes_in_fp32(monkeypatch, few):
    """Powers of two on q, k, v and dO (taken out again through the scale) leave the results the same up to powers of two: nothing leaves fp32's range on the way."""
    from airv2x_perception_amd.opencood_iface import token_attention as A
    monkeypatch.setattr(A, "FEW_MENTIONS", few)
    q, k, v, do, _ = [x.cuda() if x is not None else None for x in make(75, 1, 40, 300, 2, 1, 32, F32)]
    blocks = A.select_blocks(q, A.block_bounds(k), 3)

    def run(eq, ek, ev, eo):
        leaves = [(x * 2.0 ** e).requires_grad_() for x, e in ((q, eq), (k, ek), (v, ev))]
        out = A.block_sparse_attention(*leaves, blocks, None, 0.25 * 2.0 ** -(eq + ek))
        g = torch.autograd.grad(out, leaves, do * 2.0 ** eo)
        return [x.double() * 2.0 ** -e for x, e in zip((out.detach(), *g), (ev, ev + eo - eq, ev + eo - ek, eo))]

    want = run(0, 0, 0, 0)
    for e in ((-50, -45, 0, 0), (40, -60, 0, 0), (0, 0, -20, -50), (0, 0, 50, -80), (30, 40, 0, -60)):
        assert all(torch.equal(x, y) for x, y in zip(run(*e), want)), e


def test_selection_with_infinite_and_huge_keys():
    """A key or query beyond 1e32, an infinity too, counts as 1e32: both selection kernels make the choice of that formula."""
    from airv2x_perception_amd.opencood_iface import token_attention as A
    q, k, _, _, _ = make(85, 1, 40, 64 * 40, 1, 1, 16, F32)
    k[0, 64 * 3 + 1, 0, 2], k[0, 64 * 7, 0, 5], k[0, 64 * 9, 0, 1] = math.inf, -math.inf, 3e38
    q[0, 4, 0, 3], q[0, 5, 0, 3] = math.inf, -2e35
    bounds = A.block_bounds(k.cuda())
    ints, scale = bounds_of(k.clamp(-1e32, 1e32), None)
    assert torch.equal(bounds.ints.cpu(), ints) and torch.equal(bounds.scale.cpu(), scale)
    for n in (5, 17):
        assert torch.equal(A.select_blocks(q.cuda(), bounds, n).cpu(), chosen_of(q.clamp(-1e32, 1e32), ints, scale, n))
