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
