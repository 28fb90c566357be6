"""GPU: what the attention over selected blocks (csrc/block_sparse.hip) keeps of its inputs' precision, against the 64-bit formulas and the bounds of
test_gpu_block_sparse.

A 16-bit output is rounded once, from sums and block results in fp32: the bound of a call with gradients (half a step of the output and fp32 arithmetic, nothing for
the parts it is joined from) holds for every call.
"""
import pytest
import torch

from tests.test_gpu_block_sparse import BF, F32, HF, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("few", [0, 1 << 30])
@pytest.mark.parametrize("dt", [F32, BF, HF])
@pytest.mark.parametrize("b,t,n,h,kv,d,blocks,masked", [(1, 1, 700, 8, 8, 32, 6, None), (2, 75, 900, 8, 2, 64, 5, "empty"), (1, 130, 400, 3, 3, 16, 4, "some"), (1, 40, 300, 2, 2, 128, 3, None)])
def test_outputs_do_not_depend_on_gradients(monkeypatch, few, dt, b, t, n, h, kv, d, blocks, masked):
    from airv2x_perception_amd.opencood_iface import token_attention as A
    monkeypatch.setattr(A, "FEW_MENTIONS", few)
    q, k, v, do, mask = make(t + n + d, b, t, n, h, kv, d, dt, masked)
    seen = None if mask is None else mask.cuda()
    chosen = A.select_blocks(q.cuda(), A.block_bounds(k.cuda(), seen), blocks)
    out = check(q, k, v, do, chosen.cpu(), mask, dt)              # the bound without any part's rounding
    assert torch.equal(A.block_sparse_attention(q.cuda(), k.cuda(), v.cuda(), chosen, seen), out)


@pytest.mark.parametrize("few", [0, 1 << 30])
@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("what", ["value", "key"])
def test_a_huge_key_or_value_takes_nothing_from_its_block(monkeypatch, few, d, what):
    """One key of every block that no query gives weight to (score -40 sqrt(d) to -60, or far below) has a value of 1e10, or is itself 1e9 long: the others count in full precision.
    The bounds are relative to sum p |v| and to the scores that have weight, whatever else the block holds."""
    from airv2x_perception_amd.opencood_iface import token_attention as A
    monkeypatch.setattr(A, "FEW_MENTIONS", few)
    q, k, v, do, _ = make(91 + d, 1, 60, 300, 4, 2, d, F32)
    q[..., 0] = 8.0
    k[..., 0] = 0.0
    k[:, 5::64] = 0.0
    k[:, 5::64, :, 0] = -1e9 if what == "key" else -8.0 * d ** 0.5
    if what == "value":
        v[:, 5::64] *= 1e10
    blocks = A.select_blocks(q.cuda(), A.block_bounds(k.cuda()), 3)
    check(q, k, v, do, blocks.cpu(), None, F32)


@pytest.mark.parametrize("few", [0, 1 << 30])
def test_infinities_in_fp32(monkeypatch, few):
    """As the formula has them: a key of -inf in a channel where the query is positive has no weight; a value of inf with weight gives inf, in its channel alone."""
    from airv2x_perception_amd.opencood_iface import token_attention as A
    monkeypatch.setattr(A, "FEW_MENTIONS", few)
    q, k, v, _, _ = [x.cuda() if x is not None else None for x in make(97, 1, 50, 300, 4, 2, 32, F32)]
    q[..., 0] = q[..., 0].abs() + 0.1
    blocks = A.select_blocks(q, A.block_bounds(k), 3)
    seen = torch.ones(1, 300, dtype=torch.bool, device="cuda")
    seen[:, 7::64] = False
    want = A.block_sparse_attention(q, k, v, blocks, seen)
    k2 = k.clone()
    k2[:, 7::64, :, 0] = -float("inf")
    assert torch.equal(A.block_sparse_attention(q, k2, v, blocks), want)
    v2 = v.clone()
    v2[:, 9::64, :, 3] = float("inf")
    out, plain = A.block_sparse_attention(q, k, v2, blocks), A.block_sparse_attention(q, k, v, blocks)
    rest = torch.arange(32) != 3
    assert (out[..., 3] == float("inf")).all() and torch.equal(out[..., rest], plain[..., rest])


@pytest.mark.parametrize("few", [0, 1 << 30])
@pytest.mark.parametrize("dt", [BF, HF])
def test_infinities_in_16_bits(monkeypatch, few, dt):
    """Not finite where the formula is not, and only there; masked ones count for nothing."""
    from airv2x_perception_amd.opencood_iface import token_attention as A
    monkeypatch.setattr(A, "FEW_MENTIONS", few)
    q, k, v, _, _ = [x.cuda() if x is not None else None for x in make(99, 1, 50, 300, 4, 2, 32, dt)]
    blocks = A.select_blocks(q, A.block_bounds(k), 3)
    plain = A.block_sparse_attention(q, k, v, blocks)
    v2 = v.clone()
    v2[:, 9::64, :, 3] = float("inf")
    out = A.block_sparse_attention(q, k, v2, blocks)
    rest = torch.arange(32) != 3
    assert not out[..., 3].isfinite().any() and torch.equal(out[..., rest], plain[..., rest])
    seen = torch.ones(1, 300, dtype=torch.bool, device="cuda")
    seen[:, 9::64] = False
    assert torch.equal(A.block_sparse_attention(q, k, v2, blocks, seen), A.block_sparse_attention(q, k, v, blocks, seen))


@pytest.mark.parametrize("dim,heads,kv,dh", [(32, 1, 1, 32), (64, 4, 2, 16), (1024, 8, 8, 64)])
def test_layer_widths_in_8_bits(dim, heads, kv, dh):
    """Every width that the layer's documentation names for 8-bit activations (2 % in the gradients, as test_gpu_token_layer derives)."""
    from tests.test_gpu_token_layer import choice, layer, reference, rel
    m = layer(21, dim, heads, kv, dh, 2)
    m.act8 = True
    g = torch.Generator().manual_seed(21)
    x, dy = torch.randn(1, 150, dim, generator=g).cuda().requires_grad_(), torch.randn(1, 150, dim, generator=g).cuda()
    pos = torch.stack([torch.arange(150) // 13, torch.arange(150) % 13], 1).int().cuda()
    y = m(x, pos)
    names = [n for n, _ in m.named_parameters()]
    grads = torch.autograd.grad(y, [x] + list(m.parameters()), dy)
    want, xr, P = reference(m, x, pos, None, choice(m, x.detach(), pos, None))
    assert rel(y, want) <= 2e-5
    for n, a, r in zip(["x"] + names, grads, torch.autograd.grad(want, [xr] + [P[n] for n in names], dy.double().cpu())):
        assert rel(a, r) <= 0.02, (n, rel(a, r))
    if dim not in (256, 512):
        m.act8 = False
        with pytest.raises(RuntimeError, match="256/512"):
            m(x, pos)
