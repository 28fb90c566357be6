"""Global attention over long token maps: norm and rotation of queries and keys, selection of key blocks, attention over them
(csrc/qk_rotate.hip, csrc/block_sparse.hip).

The fusions' window and grid attentions (train_fusion_ops, swap_fusion_modules.py:78-127, mswin.py:52-96) see 4 x 4 tokens of every agent at
once; a 100 x 352 map of four agents has 140 800.  Here every query attends to the blocks of 64 keys that matter to it, and positions enter as a
rotation instead of a table tied to a window:

    q, k, v = qkv_norm_rotate(qkv, heads, kv_heads, gamma_q, gamma_k, positions, freqs)
    bounds = block_bounds(k, mask)                  # of a cache that grows: update_block_bounds
    blocks = select_blocks(q, bounds, n)            # (B, T, KV, n), exact: integer scores
    out = block_sparse_attention(q, k, v, blocks, mask)

Tensors are fp32, bf16 or fp16 on the current HIP device; sums, softmax statistics and gradients of gammas are fp32.  There is no CPU path.
Everything runs on the current stream and allocates through torch: a step can be captured into a HIP graph.  (A backward pass only while no eager graph of the same
leaves is alive: torch's engine waits for the stream of a leaf's old node, which ends the capture and the process.)
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .. import _lib
from . import act8_ops as A8
from . import train_fusion_ops as F
from . import train_ops as T
from .autograd import _P, _runner

BLOCK = 64                      # keys of one block
DIMS = (16, 32, 64, 128)        # channels of a head
MAX_BLOCKS = 64                 # blocks of one query
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
# Few queries: one wave takes each (query, head group, block) mention and reads its block directly.  Many: the mentions are sorted by block and a block is read once
# for all its queries, which costs four launches and more work items the more blocks there are.  The waves' time goes with heads x channels, so up to this many
# mentions x heads of a group x max(D, 64) / 64, more by one part in 1536 for every block, the waves are taken.  Measured (us, waves / sorted):
#   8 heads of 32, bf16          8800 keys: 8192 mentions 19 / 24, 16384: 28 / 25     140800 keys: 16384: 38 / 48, 32768: 65 / 53
#   8 heads of 32, fp32          8800 keys: 8192 mentions 24 / 30, 16384: 35 / 33     140800 keys: 16384: 40 / 67, 32768: 68 / 79
#   8 heads of 64 over 2, bf16   8800 keys: 1024 mentions 23 / 26, 4096: 36 / 34      140800 keys: 4096: 39 / 42, 8192: 64 / 47
#   4 heads of 128, fp32         8800 keys: 4096 mentions 43 / 47, 8192: 67 / 58      140800 keys: 8192: 76 / 161, 32768: 272 / 257
FEW_MENTIONS = 12288


class BlockBounds(NamedTuple):
    """What the score of a block needs: ints (B, KV, NB, 2, D) fp16 -- upper and lower bound of every channel over the block's visible keys as
    whole numbers up to 127 -- and scale (B, KV, NB) fp32 (-1: no key of the block is visible)."""
    ints: torch.Tensor
    scale: torch.Tensor


def _check_token(what, x, dim_axes, name):
    if x.device.type != "cuda" or x.dtype not in _DTYPES:
        raise RuntimeError(f"{what}: {name} must be an fp32, bf16 or fp16 HIP tensor (no CPU path exists)")
    if x.device.index is not None and x.device.index != torch.cuda.current_device():
        raise RuntimeError(f"{what}: {name} lives on {x.device}, the current HIP device is cuda:{torch.cuda.current_device()}")
    if x.dim() != dim_axes:
        raise ValueError(f"{what}: {name} has shape {tuple(x.shape)}, {dim_axes} axes are needed")
    if x.shape[-1] not in DIMS:
        raise ValueError(f"{what}: heads of {x.shape[-1]} channels ({', '.join(map(str, DIMS))} are supported)")


def _steps(x):
    """Strides of the axes before the channels; an axis of one element takes no steps, whatever its stride says."""
    steps, shape = x.stride()[:-1], x.shape
    return steps if 1 not in shape else [s if n > 1 else 0 for s, n in zip(steps, shape)]


def _strided(x, elems):
    """x itself where the kernels can read it in pieces of ``elems`` elements, else a contiguous copy."""
    if x.stride(-1) == 1 and x.data_ptr() % (elems * x.element_size()) == 0 and all(s % elems == 0 for s in _steps(x)):
        return x
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _host64(*v):
    return (ctypes.c_int64 * len(v))(*v)


# ------------------------------------------------------------------------------------------------ norm + rotation
def rotation_freqs(dim_head, axes=2, base=10000.0, device=None):
    """Turns per unit of position of the dim_head / 2 rotated pairs, (dim_head / 2,) fp64: the pairs are shared out evenly over the axes (row and column
    of a BEV map), pair i of an axis turns by base ** (-i / pairs of the axis) radians per step."""
    if dim_head not in DIMS or axes < 1 or (dim_head // 2) % axes:
        raise ValueError(f"rotation_freqs: {axes} axes for heads of {dim_head} channels")
    per = dim_head // 2 // axes
    f = (float(base) ** (-torch.arange(per, dtype=torch.float64) / per)) / (2 * math.pi)
    return f.repeat(axes).to(device)


def _check_rotation(what, dim, rows, gammas, positions, freqs, device):
    for g in gammas:
        if g is not None:
            T._check_dev(g)
            if tuple(g.shape) != (dim,):
                raise ValueError(f"{what}: gamma of shape {tuple(g.shape)} for heads of {dim} channels")
    if positions.device != device or positions.dtype != torch.int32 or positions.dim() < 2 or positions.numel() != rows * positions.shape[-1]:
        raise ValueError(f"{what}: positions must be int32 (tokens, axes) on the tensors' device, got {positions.dtype} {tuple(positions.shape)} for {rows} tokens")
    axes = positions.shape[-1]
    if axes < 1 or (dim // 2) % axes:
        raise ValueError(f"{what}: {axes} axes do not divide {dim // 2} pairs")
    if freqs.device != device or freqs.dtype != torch.float64 or tuple(freqs.shape) != (dim // 2,):
        raise ValueError(f"{what}: freqs must be fp64 ({dim // 2},) on the tensors' device (rotation_freqs)")
    return axes


def _rows(x):
    """(..., T, H, D) as (rows, H, D) without a copy where the strides allow it."""
    return x if x.dim() == 3 else x.flatten(0, -3)


def _rotate_forward(q, k, gq, gk, pos, freqs, eps, inter):
    r = _runner(q.device)
    rows, h, d = q.shape
    kv = k.shape[1] if k is not None else 0
    oq = torch.empty((rows, h, d), dtype=q.dtype, device=q.device)
    ok = torch.empty((rows, kv, d), dtype=q.dtype, device=q.device) if k is not None else None
    st = _host64(*_steps(q), *(_steps(k) if kv else (0, 0)))
    _lib.check(r.lib.av2x_qk_norm_rotate(_P(q), _P(k), st, _P(gq), _P(gk), _P(pos), _P(freqs), _P(oq), _P(ok), rows, h, kv, d, pos.shape[-1], 1 if inter else 0,
                                         _DTYPES[q.dtype], eps, r.stream()), "av2x_qk_norm_rotate")
    return oq, ok


def _rotate_backward(q, k, gq, gk, pos, freqs, eps, inter, doq, dok, dov, dq, dk, dv, want):
    r = _runner(q.device)
    rows, h, d = q.shape
    kv = k.shape[1] if k is not None else 0
    dgq = torch.empty_like(gq) if want[0] else None
    dgk = torch.empty_like(gk) if kv and want[1] else None
    ws = torch.empty(int(r.lib.av2x_qk_norm_rotate_backward_workspace_bytes(d)), dtype=torch.uint8, device=q.device)
    st = _host64(*_steps(q), *(_steps(k) if kv else (0, 0)))
    dst = _host64(*_steps(dq), *(_steps(dk) if kv else (0, 0)), *(_steps(dv) if dv is not None else (0, 0)))
    fit = lambda t: A8._aligned(t) if t is not None else None
    doq, dok, dov = fit(doq), fit(dok), fit(dov)
    _lib.check(r.lib.av2x_qk_norm_rotate_backward(_P(q), _P(k), st, _P(gq), _P(gk), _P(pos), _P(freqs), _P(doq), _P(dok), _P(dov), _P(dq), _P(dk), _P(dv), dst,
                                                  _P(dgq), _P(dgk), rows, h, kv, d, pos.shape[-1], 1 if inter else 0, _DTYPES[q.dtype], eps, _P(ws), r.stream()),
               "av2x_qk_norm_rotate_backward")
    return dgq, dgk


class _QkNormRotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, gq, gk, pos, freqs, eps, inter):
        ctx.set_materialize_grads(False)
        oq, ok = _rotate_forward(q, k, gq, gk, pos, freqs, eps, inter)
        ctx.save_for_backward(q, k, gq, gk, pos, freqs)
        ctx.cfg = (eps, inter)
        return oq, ok

    @staticmethod
    @once_differentiable
    def backward(ctx, doq, dok):
        q, k, gq, gk, pos, freqs = ctx.saved_tensors
        dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        dk = torch.empty(k.shape, dtype=k.dtype, device=k.device) if k is not None else None
        need = ctx.needs_input_grad
        dgq, dgk = _rotate_backward(q, k, gq, gk, pos, freqs, *ctx.cfg, doq, dok, None, dq, dk, None, (need[2], need[3]))
        return dq, dk, dgq, dgk, None, None, None, None


class _QkvNormRotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, h, kv, gq, gk, pos, freqs, eps, inter):
        ctx.set_materialize_grads(False)
        oq, ok = _rotate_forward(qkv[:, :h], qkv[:, h:h + kv], gq, gk, pos, freqs, eps, inter)
        ctx.save_for_backward(qkv, gq, gk, pos, freqs)
        ctx.cfg = (h, kv, eps, inter)
        return oq, ok, qkv[:, h + kv:]

    @staticmethod
    @once_differentiable
    def backward(ctx, doq, dok, dov):
        qkv, gq, gk, pos, freqs = ctx.saved_tensors
        h, kv, eps, inter = ctx.cfg
        d = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)      # the whole buffer's gradient in one pass
        need = ctx.needs_input_grad
        dgq, dgk = _rotate_backward(qkv[:, :h], qkv[:, h:h + kv], gq, gk, pos, freqs, eps, inter, doq, dok, dov, d[:, :h], d[:, h:h + kv], d[:, h + kv:],
                                    (need[3], need[4]))
        return d, None, None, dgq, dgk, None, None, None, None


def qk_norm_rotate(q, k, gamma_q, gamma_k, positions, freqs, eps=1e-6, interleaved=False):
    """RMS norm of every head vector, times gamma, then the rotation by the token's position; q (..., T, H, D), k (..., T, KV, D) or None -> the same shapes,
    contiguous.  ``positions`` int32 (..., T, axes), ``freqs`` of rotation_freqs; ``interleaved``: pairs of neighbouring channels instead of (i, i + D / 2)."""
    what = "qk_norm_rotate"
    if q.dim() < 3:
        raise ValueError(f"{what}: q has shape {tuple(q.shape)}, (..., tokens, heads, channels) is needed")
    shape = q.shape
    q3 = _rows(q)
    _check_token(what, q3, 3, "q")
    k3 = kshape = None
    if k is not None:
        kshape = k.shape
        if k.dim() != q.dim() or k.shape[:-2] != shape[:-2] or k.shape[-1] != shape[-1] or k.dtype != q.dtype or k.device != q.device:
            raise ValueError(f"{what}: k {tuple(k.shape)} {k.dtype} does not fit q {tuple(shape)} {q.dtype}")
        if gamma_k is None:
            raise ValueError(f"{what}: k needs its gamma")
        k3 = _rows(k)
    _check_rotation(what, shape[-1], q3.shape[0], (gamma_q, gamma_k if k is not None else None), positions, freqs, q.device)
    q3 = _strided(q3, 4)
    k3 = _strided(k3, 4) if k3 is not None else None
    pos, freqs = positions.reshape(-1, positions.shape[-1]).contiguous(), freqs.contiguous()
    gq, gk = A8._aligned(gamma_q), A8._aligned(gamma_k) if k is not None else None
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q3, k3, gq, gk)):
        oq, ok = _QkNormRotate.apply(q3, k3, gq, gk, pos, freqs, float(eps), bool(interleaved))
    else:
        oq, ok = _rotate_forward(q3, k3, gq, gk, pos, freqs, float(eps), bool(interleaved))
    if q.dim() == 3:
        return oq, ok
    return oq.view(shape), ok.view(kshape) if ok is not None else None


def qkv_norm_rotate(qkv, heads, kv_heads, gamma_q, gamma_k, positions, freqs, eps=1e-6, interleaved=False):
    """The same on a fused projection: qkv (..., T, heads + 2 kv_heads, D) = [q | k | v] -> q, k (contiguous), v (a view of qkv).  Its backward writes the
    gradient of the whole buffer in one pass, the values' part included."""
    what = "qkv_norm_rotate"
    if qkv.dim() < 3 or heads < 1 or kv_heads < 1 or qkv.shape[-2] != heads + 2 * kv_heads:
        raise ValueError(f"{what}: qkv has shape {tuple(qkv.shape)}, (..., tokens, {heads} + 2 x {kv_heads}, channels) is needed")
    lead = tuple(qkv.shape[:-2])
    x = _rows(qkv)
    _check_token(what, x, 3, "qkv")
    _check_rotation(what, x.shape[-1], x.shape[0], (gamma_q, gamma_k), positions, freqs, x.device)
    x = _strided(x, 4)
    pos, freqs = positions.reshape(-1, positions.shape[-1]).contiguous(), freqs.contiguous()
    gq, gk = A8._aligned(gamma_q), A8._aligned(gamma_k)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, gq, gk)):
        q, k, v = _QkvNormRotate.apply(x, heads, kv_heads, gq, gk, pos, freqs, float(eps), bool(interleaved))
    else:
        q, k = _rotate_forward(x[:, :heads], x[:, heads:heads + kv_heads], gq, gk, pos, freqs, float(eps), bool(interleaved))
        v = x[:, heads + kv_heads:]
    if len(lead) == 1:
        return q, k, v
    d = x.shape[-1]
    return q.view(lead + (heads, d)), k.view(lead + (kv_heads, d)), v.unflatten(0, lead)


# ------------------------------------------------------------------------------------------------ blocks
def _check_mask(what, mask, batch, keys, device):
    if mask is None:
        return None
    if mask.device != device or mask.dtype not in (torch.bool, torch.uint8) or tuple(mask.shape) != (batch, keys):
        raise ValueError(f"{what}: mask must be bool ({batch}, {keys}) on the tensors' device, got {mask.dtype} {tuple(mask.shape)} on {mask.device}")
    return mask.contiguous()


def _check_bounds(what, bounds, batch, kv, dim, device):
    ints, scale = bounds
    if ints.device != device or ints.dtype != torch.float16 or scale.device != device or scale.dtype != torch.float32:
        raise ValueError(f"{what}: bounds must be fp16 and fp32 on the tensors' device")
    nb = scale.shape[-1]
    if tuple(scale.shape) != (batch, kv, nb) or ints.numel() != scale.numel() * 2 * dim or ints.shape[:3] != scale.shape:
        raise ValueError(f"{what}: bounds {tuple(ints.shape)}, {tuple(scale.shape)} for batch {batch}, {kv} kv heads of {dim} channels")
    if not ints.is_contiguous() or not scale.is_contiguous() or ints.data_ptr() % 16:
        raise ValueError(f"{what}: bounds must be contiguous")
    return nb


def _launch_bounds(k, mask, ints, scale, first, count):
    r = _runner(k.device)
    b, n, kv, d = k.shape
    k = _strided(k, 4)
    _lib.check(r.lib.av2x_block_bounds(_P(k), _P(mask), _host64(*_steps(k)), b, n, kv, d, _DTYPES[k.dtype], first, count, _P(ints), _P(scale), r.stream()),
               "av2x_block_bounds")


def block_bounds(k, mask=None):
    """k (B, N, KV, D), mask (B, N) bool of visible keys -> BlockBounds of its ceil(N / 64) blocks.  Not differentiable (selection is a choice)."""
    _check_token("block_bounds", k, 4, "k")
    k = k.detach()
    b, n, kv, d = k.shape
    mask = _check_mask("block_bounds", mask, b, n, k.device)
    nb = (n + BLOCK - 1) // BLOCK
    ints = torch.empty((b, kv, nb, 2, d), dtype=torch.float16, device=k.device)
    scale = torch.empty((b, kv, nb), dtype=torch.float32, device=k.device)
    if nb and b:
        _launch_bounds(k, mask, ints, scale, 0, nb)
    return BlockBounds(ints, scale)


def update_block_bounds(bounds, k, first, last, mask=None):
    """Recomputes, in place, the bounds of the blocks that hold the tokens first .. last - 1 of the cache k (B, N, KV, D) -- what appending or replacing tokens
    costs: one block per sample and head instead of the whole cache."""
    what = "update_block_bounds"
    _check_token(what, k, 4, "k")
    k = k.detach()
    b, n, kv, d = k.shape
    nb = _check_bounds(what, bounds, b, kv, d, k.device)
    mask = _check_mask(what, mask, b, n, k.device)
    if nb != (n + BLOCK - 1) // BLOCK:
        raise ValueError(f"{what}: bounds of {nb} blocks for {n} keys")
    if not 0 <= first <= last <= n:
        raise ValueError(f"{what}: tokens {first} .. {last} of {n}")
    if first < last and b:
        lo, hi = first // BLOCK, (last - 1) // BLOCK + 1
        _launch_bounds(k, mask, bounds.ints, bounds.scale, lo, hi - lo)
    return bounds


def select_blocks(q, bounds, blocks):
    """q (B, T, H, D), BlockBounds -> int32 (B, T, KV, blocks): for every query and kv head the blocks whose bound on q . k is largest (summed over the head
    group, q as whole numbers), ties to the lowest, ascending, -1 behind the last.  The score is an integer times the block's scale: exact."""
    what = "select_blocks"
    _check_token(what, q, 4, "q")
    q = q.detach()
    b, t, h, d = q.shape
    kv = bounds.scale.shape[1] if bounds.scale.dim() == 3 else 0
    if kv < 1 or h % kv:
        raise ValueError(f"{what}: {h} query heads over {kv} kv heads")
    nb = _check_bounds(what, bounds, b, kv, d, q.device)
    _check_sizes(what, b, t, nb * BLOCK, h, kv, d, blocks)
    out = torch.empty((b, t, kv, blocks), dtype=torch.int32, device=q.device)
    if b and t:
        r = _runner(q.device)
        if q.stride(-1) != 1:
            q = q.contiguous()
        size = int(r.lib.av2x_select_blocks_workspace_bytes(b, t, nb * BLOCK, kv, blocks))
        ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
        _lib.check(r.lib.av2x_select_blocks(_P(q), _host64(*_steps(q)), _P(bounds.ints), _P(bounds.scale), b, t, nb * BLOCK, h, kv, d, blocks, _DTYPES[q.dtype],
                                            _P(out), _P(ws), r.stream()), "av2x_select_blocks")
    return out


def _check_sizes(what, b, t, n, h, kv, d, blocks):
    if not 1 <= blocks <= MAX_BLOCKS:
        raise ValueError(f"{what}: {blocks} blocks a query (1 .. {MAX_BLOCKS})")
    if h // kv > 16 or h // kv * d > 1024:
        raise ValueError(f"{what}: {h // kv} heads of {d} channels share their keys (at most 16 heads and 1024 channels)")
    if (n + BLOCK - 1) // BLOCK > 32768:
        raise ValueError(f"{what}: {n} keys (at most {32768 * BLOCK})")
    if t > 1 << 25 or t * blocks * (h // kv) > (1 << 31) - 1 - 4096 or b * kv > 65535:
        raise ValueError(f"{what}: too many queries ({b} x {t})")


def _launch_lists(r, blocks, n, h):
    b, t, kv, s = blocks.shape
    lists = torch.empty(int(r.lib.av2x_block_lists_bytes(b, t, n, h, kv, s)), dtype=torch.uint8, device=blocks.device)
    _lib.check(r.lib.av2x_block_lists(_P(blocks), b, t, n, h, kv, s, _P(lists), r.stream()), "av2x_block_lists")
    return lists


def _strides9(q, k, v):
    return _host64(*_steps(q), *_steps(k), *_steps(v))


def _attend(q, k, v, blocks, mask, scale, grads):
    r = _runner(q.device)
    b, t, h, d = q.shape
    n, kv, s = k.shape[1], k.shape[2], blocks.shape[3]
    out = torch.empty((b, t, h, d), dtype=q.dtype, device=q.device)
    lse = torch.empty((b, t, h), dtype=torch.float32, device=q.device) if grads else None
    rest = torch.empty_like(out) if grads and q.dtype != torch.float32 else None
    few = b * t * h * s * max(d, 64) <= 64 * FEW_MENTIONS * (1 + (n + BLOCK - 1) // BLOCK / 1536)
    lists = None if few else _launch_lists(r, blocks, n, h)
    ws = torch.empty(int(r.lib.av2x_block_sparse_workspace_bytes(b, t, n, h, kv, d, s, 0)), dtype=torch.uint8, device=q.device)
    _lib.check(r.lib.av2x_block_sparse_attention(_P(q), _P(k), _P(v), _strides9(q, k, v), _P(mask), _P(blocks), _P(lists), b, t, n, h, kv, d, s, _DTYPES[q.dtype],
                                                 scale, _P(out), _P(lse), _P(rest), _P(ws), r.stream()), "av2x_block_sparse_attention")
    return out, lse, rest, lists


class _BlockSparseAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, blocks, mask, scale):
        out, lse, rest, lists = _attend(q, k, v, blocks, mask, scale, True)
        ctx.save_for_backward(q, k, v, blocks, mask, out, rest, lse, lists)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, blocks, mask, out, rest, lse, lists = ctx.saved_tensors
        r = _runner(q.device)
        b, t, h, d = q.shape
        n, kv, s = k.shape[1], k.shape[2], blocks.shape[3]
        need = ctx.needs_input_grad
        if lists is None:
            lists = _launch_lists(r, blocks, n, h)
        new = lambda x: torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dq, dk, dv = new(q), new(k) if need[1] else None, new(v) if need[2] else None
        ws = torch.empty(int(r.lib.av2x_block_sparse_workspace_bytes(b, t, n, h, kv, d, s, 1)), dtype=torch.uint8, device=q.device)
        _lib.check(r.lib.av2x_block_sparse_attention_backward(_P(q), _P(k), _P(v), _strides9(q, k, v), _P(mask), _P(blocks), _P(lists), _P(out), _P(rest), _P(lse),
                                                              _P(A8._aligned(dout)), b, t, n, h, kv, d, s, _DTYPES[q.dtype], ctx.scale, _P(dq), _P(dk), _P(dv), _P(ws),
                                                              r.stream()), "av2x_block_sparse_attention_backward")
        return dq, dk, dv, None, None, None


def block_sparse_attention(q, k, v, blocks, mask=None, scale=None):
    """softmax(scale q k^T) v of every query over the visible keys of its blocks: q (B, T, H, D), k, v (B, N, KV, D), blocks int32 (B, T, KV, n) (select_blocks, or any
    choice: indices outside 0 .. ceil(N / 64) - 1 are none, a block named twice counts twice), mask (B, N) bool of visible keys.  A query without a
    visible key gets zeros, and what stands in masked places is never read.  scale: 1 / sqrt(D).  Differentiable in q, k, v, bit for bit the same every time, with and
    without gradients.  A visible infinity or NaN gives outputs that are not finite (fp32: those of the formula; 16 bits: NaN, where the formula may have an infinity)."""
    what = "block_sparse_attention"
    for x, name in ((q, "q"), (k, "k"), (v, "v")):
        _check_token(what, x, 4, name)
    b, t, h, d = q.shape
    n, kv = k.shape[1:3]
    if k.shape != v.shape or k.shape[0] != b or k.shape[3] != d or kv < 1 or h % kv or not (q.dtype == k.dtype == v.dtype) or not (q.device == k.device == v.device):
        raise ValueError(f"{what}: q {tuple(q.shape)} {q.dtype}, k {tuple(k.shape)} {k.dtype}, v {tuple(v.shape)} {v.dtype} do not fit")
    if blocks.dtype != torch.int32 or blocks.device != q.device or blocks.dim() != 4 or tuple(blocks.shape[:3]) != (b, t, kv):
        raise ValueError(f"{what}: blocks must be int32 ({b}, {t}, {kv}, n) on the tensors' device, got {blocks.dtype} {tuple(blocks.shape)}")
    _check_sizes(what, b, t, n, h, kv, d, blocks.shape[3])
    mask = _check_mask(what, mask, b, n, q.device)
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if b == 0 or t == 0 or n == 0:
        # zeros that stay on the graph, whatever q holds
        return q.masked_fill(torch.ones_like(q, dtype=torch.bool), 0.0) + ((k.sum() + v.sum()) * 0.0).to(q.dtype)
    elems = 16 // q.element_size()
    q, k, v, blocks = _strided(q, elems), _strided(k, elems), _strided(v, elems), A8._aligned(blocks)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _BlockSparseAttention.apply(q, k, v, blocks, mask, scale)
    return _attend(q, k, v, blocks, mask, scale, False)[0]


# ------------------------------------------------------------------------------------------------ the layer
class BlockSparseAttention(nn.Module):
    """x + to_out(attention(LayerNorm(x))) over all tokens of a sample: x (B, T, dim) fp32, positions int32 (T, axes) or (B, T, axes), mask (B, T) bool of
    visible tokens -> (B, T, dim); dim 256 or 512 (act8: any multiple of 32 up to 1024), parameters fp32.  A global counterpart of the fusions' PreNorm windowed
    attentions.  Under ``torch.autocast`` (or ``amp = True``) the attention runs in bf16; ``act8 = True`` keeps the Linears' inputs in 8 bits for the backward."""

    def __init__(self, dim, heads=8, dim_head=32, blocks=8, kv_heads=None, axes=2, base=10000.0, eps=1e-6):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if heads % kv_heads:
            raise ValueError(f"BlockSparseAttention: {heads} heads over {kv_heads} kv heads")
        self.heads, self.kv_heads, self.dim_head, self.blocks, self.eps = heads, kv_heads, dim_head, blocks, eps
        self.act8, self.amp = False, None
        self.norm = nn.LayerNorm(dim)
        self.to_qkv = nn.Linear(dim, (heads + 2 * kv_heads) * dim_head, bias=False)
        self.q_gamma, self.k_gamma = nn.Parameter(torch.ones(dim_head)), nn.Parameter(torch.ones(dim_head))
        self.to_out = nn.Linear(heads * dim_head, dim)
        self.rotation = (dim_head, axes, base)
        self.register_buffer("freqs", rotation_freqs(*self.rotation), persistent=False)

    def _apply(self, fn, recurse=True):
        """Moves and casts (.to, .float, .half, ..): the frequencies move along and stay fp64."""
        freqs = self.freqs
        super()._apply(fn, recurse)
        device = self.freqs.device
        self.freqs = freqs.to(device) if not freqs.is_meta else rotation_freqs(*self.rotation, device=device)
        return self

    def forward(self, x, positions, mask=None):
        from .airv2x_where2com import _amp_requested
        if x.device.type != "cuda":
            raise RuntimeError("BlockSparseAttention (MI355X build) has no CPU path: move the module to the GPU")
        b, t, c = x.shape
        amp = _amp_requested(self)
        x = x.contiguous()
        with T.amp_scope(amp):
            w = self.to_qkv.weight
            if self.act8:
                qkv = A8.norm_linear(x, self.norm.weight, self.norm.bias, w)
            else:
                qkv = F.linear(F.layer_norm(x.view(b, 1, t, c), self.norm.weight, self.norm.bias), w)
            qkv = qkv.view(b, t, self.heads + 2 * self.kv_heads, self.dim_head)
            if amp:
                qkv = qkv.to(torch.bfloat16)
            pos = positions if positions.dim() == 3 else positions.expand(b, *positions.shape)
            q, k, v = qkv_norm_rotate(qkv, self.heads, self.kv_heads, self.q_gamma, self.k_gamma, pos, self.freqs, self.eps)
            chosen = select_blocks(q, block_bounds(k, mask), self.blocks)
            o = block_sparse_attention(q, k, v, chosen, mask).float().view(b, 1, t, self.heads * self.dim_head)
            lin = A8.linear if self.act8 else F.linear
            return lin(o, self.to_out.weight, self.to_out.bias, x.view(b, 1, t, c)).view(b, t, c)
