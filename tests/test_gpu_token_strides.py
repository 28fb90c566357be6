"""GPU: single tokens, heads and samples cut out of buffers of any pitch: an axis of one element may have any stride."""
import pytest
import torch

from tests.test_gpu_block_sparse import BF, F32, make

pytestmark = pytest.mark.gpu


def cut(x, pitch):
    """x (dense) as a view whose axes of one element step by ``pitch`` elements."""
    y = x.as_strided(x.shape, [pitch if n == 1 else s for n, s in zip(x.shape, x.stride())])
    assert torch.equal(y, x) and any(s == pitch for s in y.stride())
    return y


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("inter", [False, True])
def test_rotation_of_one_token_and_one_head(dt, inter):
    from airv2x_perception_amd.opencood_iface import token_attention as A
    g = torch.Generator().manual_seed(1)
    gq, gk = torch.randn(32, generator=g).cuda(), torch.randn(32, generator=g).cuda()
    fr = A.rotation_freqs(32, 1).cuda()
    for t, h, kv in ((1, 1, 1), (5, 1, 1), (1, 4, 1)):
        q, k = torch.randn(t, h, 32, generator=g).to(dt).cuda(), torch.randn(t, kv, 32, generator=g).to(dt).cuda()
        pos = torch.arange(t, dtype=torch.int32, device="cuda")[:, None] + 9
        wide = torch.zeros(t, 33, dtype=dt, device="cuda")          # a buffer with rows of 33
        res = []
        for f in (lambda x: x, lambda x: cut(x, 33)):
            leaves = [x.requires_grad_() for x in (q.clone(), k.clone())]
            out = A.qk_norm_rotate(f(leaves[0]), f(leaves[1]) if 1 in k.shape else leaves[1], gq, gk, pos, fr, interleaved=inter)
            res.append([x.detach() for x in out] + list(torch.autograd.grad(out, leaves, [torch.ones_like(x).cumsum(-1) for x in out])))
        if h == 1:
            wide[:, :32] = q[:, 0]
            out = A.qk_norm_rotate(wide[:, :32].unsqueeze(1), None, gq, None, pos, fr, interleaved=inter)
            assert torch.equal(out[0], res[0][0])
        assert all(torch.equal(a, b) for a, b in zip(*res))
    x = torch.randn(1, 3, 32, generator=g).to(dt).cuda()
    pos = torch.full((1, 1), 7, dtype=torch.int32, device="cuda")
    for a, b in zip(A.qkv_norm_rotate(cut(x, 101), 1, 1, gq, gk, pos, fr, interleaved=inter), A.qkv_norm_rotate(x, 1, 1, gq, gk, pos, fr, interleaved=inter)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("few", [0, 1 << 30])
@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("t,n,h,kv", [(1, 1, 1, 1), (1, 200, 4, 2), (20, 200, 1, 1)])
def test_attention_of_one_token_one_head_and_one_sample(monkeypatch, few, dt, t, n, h, kv):
    from airv2x_perception_amd.opencood_iface import token_attention as A
    monkeypatch.setattr(A, "FEW_MENTIONS", few)
    q, k, v, do, _ = [x.cuda() if x is not None else None for x in make(3, 1, t, n, h, kv, 32, dt)]
    res = []
    for f in (lambda x: x, lambda x: cut(x, 33)):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        views = [f(x) for x in leaves]
        bounds = A.block_bounds(views[1])
        blocks = A.select_blocks(views[0], bounds, 2)
        out = A.block_sparse_attention(*views, blocks)
        A.update_block_bounds(bounds, views[1], 0, 1)
        res.append([bounds.ints, bounds.scale, blocks, out.detach()] + list(torch.autograd.grad(out, leaves, do)))
    assert all(torch.equal(a, b) for a, b in zip(*res))
