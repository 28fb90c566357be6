"""Token layers whose saved activation is held in 8 bits: Linear, LayerNorm -> Linear, GELU and GELU -> Linear as autograd nodes
(csrc/act8.hip; the products of the forward and the data gradient are the framework's GEMM, as in train_fusion_ops.LinearFn).

A Linear keeps its input for the weight gradient, a LayerNorm for its own backward, a GELU its argument: in fp32 a FeedForward block holds
x, LN(x), z and gelu(z), 16 bytes per token and channel of the hidden width.  Here a node keeps

    x8 = q scale,   scale = max|x| / 127 over 128 channels of a row,   q = clamp(rint(x (127 / max(max|x|, 1e-30))), -127, 127)

one byte and 1/32, and LayerNorm -> Linear or GELU -> Linear share ONE such copy.  The forward is unchanged; the backward is the exact
derivative taken at x8 instead of x:

    linear        dW = dY^T x8                           dx = dY W
    norm_linear   u = (x8 - mean) rstd (the forward's statistics)   dW = dY^T (u gamma + beta)   a = (dY W) gamma
                  dx = rstd (a - mean(a) - u mean(a u))  dgamma = sum (dY W) u = sum_o W (dY^T u)    dbeta = sum dY W = sum_o W db
    gelu(_linear) dW = dY^T gelu(z8)                     dz = (dY W) gelu'(z8)

The stored values are off by at most scale / 2, 1/254 of the group's largest |x|; LayerNorm's backward sees that error times rstd, so a row whose mean is large beside its
spread (|mean| = 10 standard deviations: 4 % of one in u) has noisier gradients than the residual stream's centred rows.

A group with an infinity or a NaN has a NaN scale: the gradients show it, as they would without the 8 bits (GradScaler's check works).  In the products an infinity, split
into three terms, gives NaN.
A step can be captured into a HIP graph, while no eager graph of the same leaves is alive (torch's engine would wait for the stream of a leaf's old node); its weights are
packed on every replay, and in every later eager call (train_ops.forget_packings: for weights that a replay changes without running their layers).
``model.act8 = True`` trains Airv2xCoBEVT / Airv2xV2XVit's fusion with these nodes (train_ops.act8_scope).
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from . import train_ops as T
from .autograd import _P, _runner

GROUP = 128           # channels of one scale
LN_EPS = 1e-5
# Up to this many multiply-adds the products run on av2x_act8_gemm, which reads the weight as it lies; from there on on the framework's GEMM, whose weights are
# packed and split into terms first, once for every new value of a weight.  Measured (us, forward + data gradient, packing included, small / large):
#   256 -> 256    4400 rows: 27 / 40,  16384: 51 / 53,   32768: 98 / 71
#   256 -> 768    2200 rows: 40 / 60,  4400: 58 / 65,    8192: 69 / 74,   16384: 129 / 97
#   512 -> 512    2200 rows: 43 / 65,  4400: 73 / 69,    8192: 85 / 78,   16384: 162 / 111
SMALL_PRODUCT = 1 << 30


class Packed8(NamedTuple):
    """q (..., C) int8 and scale (rows, ceil(C / 128)) fp32."""
    q: torch.Tensor
    scale: torch.Tensor


def _check(what, x, weight=None, bias=None, residual=None, vectors=(), most=1 << 20):
    T._check_dev(x)
    if x.dim() < 1:
        raise ValueError(f"{what}: a tensor with a channel axis is needed")
    c = x.shape[-1]
    if c < 4 or c % 4 or c > most:
        raise ValueError(f"{what}: {c} channels (a multiple of 4, at most {most})")
    for v in vectors:
        T._check_dev(v)
        if tuple(v.shape) != (c,):
            raise ValueError(f"{what}: a parameter of shape {tuple(v.shape)} for {c} channels")
    if weight is not None:
        T._check_dev(weight)
        if weight.dim() != 2 or weight.shape[1] != c or c % 32 or weight.shape[0] < 32 or weight.shape[0] % 32:
            raise ValueError(f"{what}: a weight of shape {tuple(weight.shape)} for {c} channels (the GEMM takes multiples of 32)")
        cout = weight.shape[0]
        if (x.numel() // c) * max(c, cout) >= 1 << 31:
            raise ValueError(f"{what}: {x.numel() // c} rows of {max(c, cout)} channels: the GEMM addresses 2^31 elements, split the rows")
        if bias is not None:
            T._check_dev(bias)
            if tuple(bias.shape) != (cout,):
                raise ValueError(f"{what}: a bias of shape {tuple(bias.shape)} for {cout} outputs")
        if residual is not None:
            T._check_dev(residual)
            if tuple(residual.shape) != tuple(x.shape[:-1]) + (cout,):
                raise ValueError(f"{what}: a residual of shape {tuple(residual.shape)}")


def _aligned(x):
    """Contiguous, on a 16-byte address (a view into the middle of a buffer may not be)."""
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _maybe(x):
    return _aligned(x) if x is not None else None


def _empty_pack(x):
    c = x.shape[-1]
    rows = x.numel() // c
    return rows, c, torch.empty(x.shape, dtype=torch.int8, device=x.device), torch.empty((rows, (c + GROUP - 1) // GROUP), dtype=torch.float32, device=x.device)


def pack(x):
    """(..., C) fp32 -> Packed8."""
    _check("pack", x)
    r = _runner(x.device)
    x = _aligned(x.detach())
    rows, c, q, s = _empty_pack(x)
    _lib.check(r.lib.av2x_act8_pack(_P(x), _P(q), _P(s), rows, c, r.stream()), "av2x_act8_pack")
    return Packed8(q, s)


def unpack(p):
    """Packed8 -> the fp32 values it stands for."""
    q, s = p
    if q.device.type != "cuda" or q.dtype != torch.int8 or s.dtype != torch.float32 or s.device != q.device or q.dim() < 1:
        raise RuntimeError("unpack: an int8 and an fp32 HIP tensor")
    T._check_dev(s)
    c = q.shape[-1]
    if c < 4 or c % 4 or tuple(s.shape) != (q.numel() // c, (c + GROUP - 1) // GROUP):
        raise ValueError(f"unpack: scale of shape {tuple(s.shape)} for {tuple(q.shape)}")
    r = _runner(q.device)
    q, s = _aligned(q), _aligned(s)
    out = torch.empty(q.shape, dtype=torch.float32, device=q.device)
    _lib.check(r.lib.av2x_act8_unpack(_P(q), _P(s), _P(out), q.numel() // c, c, r.stream()), "av2x_act8_unpack")
    return out


# ------------------------------------------------------------------------------------------------ raw launches
def _gemm(r, x, weight, bias, residual):
    """x W^T (+ b) (+ residual): the engine's launcher with the rows as one image line, or for few rows a GEMM on the parameter as it lies."""
    from .engine import ConvLayer
    cout, cin = weight.shape
    rows = x.numel() // cin
    y = torch.empty(tuple(x.shape[:-1]) + (cout,), dtype=torch.float32, device=x.device)
    if rows == 0:
        return y
    if rows * cin * cout <= SMALL_PRODUCT and not T.AMP_STEP[0]:
        T._may_keep(weight)                               # (a recorded step uses it, though it packs nothing)
        _lib.check(r.lib.av2x_act8_gemm(_P(x), _P(_aligned(weight)), _P(bias), _P(residual), _P(y), rows, cout, cin, 0, r.stream()), "av2x_act8_gemm")
        return y
    wp, coutp, _, ent = T._packed(r, weight.detach().view(cout, cin, 1, 1), owner=weight)
    L = ConvLayer(wp, None, bias.detach() if bias is not None else T._zeros(cout, x.device), cin, cout, coutp, 1, 1, 0, 0)
    T.seed_x3p(r, L, ent)
    r.amp = T.AMP_STEP[0] and cin % 8 == 0
    try:
        r.conv(L, x, 1, 1, rows, y, residual=residual)
    finally:
        r.amp = False
    return y


def _dgrad(dy, weight, amp):
    """dY W in the forward's precision."""
    if amp != T.AMP_STEP[0]:
        with T.amp_scope(amp):
            return _dgrad(dy, weight, amp)
    cout, cin = weight.shape
    rows = dy.numel() // cout
    if rows == 0:
        return torch.empty(tuple(dy.shape[:-1]) + (cin,), dtype=torch.float32, device=dy.device)
    if rows * cin * cout <= SMALL_PRODUCT and not T.AMP_STEP[0]:
        r = _runner(dy.device)
        T._may_keep(weight)
        dx = torch.empty(tuple(dy.shape[:-1]) + (cin,), dtype=torch.float32, device=dy.device)
        _lib.check(r.lib.av2x_act8_gemm(_P(dy), _P(_aligned(weight)), None, None, _P(dx), rows, cin, cout, 1, r.stream()), "av2x_act8_gemm")
        return dx
    w4 = weight.detach().view(cout, cin, 1, 1)
    return T.conv_dgrad(dy.view(1, 1, rows, cout), w4, 1, 0, (1, rows), owner=weight).view(tuple(dy.shape[:-1]) + (cin,))


def _wgrad(r, kind, dy, q, s, cin, stats=None, gamma=None, beta=None, want_w=True, want_b=True, weight=None, dgamma=None, dbeta=None):
    """(dW, db) and, for LayerNorm -> Linear, its affine's gradients into dgamma, dbeta."""
    cout = dy.shape[-1]
    rows = dy.numel() // cout
    dw = torch.empty((cout, cin), dtype=torch.float32, device=dy.device) if want_w else None
    db = torch.empty(cout, dtype=torch.float32, device=dy.device) if want_b else None
    ws = torch.empty(int(r.lib.av2x_act8_wgrad_workspace_bytes(rows, cout, cin)), dtype=torch.uint8, device=dy.device)
    _lib.check(r.lib.av2x_act8_wgrad(_P(dy), _P(q), _P(s), _P(stats), _P(gamma), _P(beta), _P(weight), kind, rows, cout, cin, _P(dw), _P(db), _P(dgamma), _P(dbeta), _P(ws),
                                     r.stream()),
               "av2x_act8_wgrad")
    return dw, db


def _bias_grad(r, dy):
    """Column sums alone (a frozen weight)."""
    from .train_fusion_ops import _chan_sum
    cout = dy.shape[-1]
    rows = dy.numel() // cout
    return _chan_sum(r, dy, rows, cout) if rows else torch.zeros(cout, device=dy.device)


def _gelu_forward(r, z, want_pack=True):
    rows, c, q, s = _empty_pack(z)
    h = torch.empty_like(z)
    _lib.check(r.lib.av2x_act8_gelu(_P(z), _P(h), _P(q), _P(s), rows, c, r.stream()), "av2x_act8_gelu")
    return h, q, s


# ------------------------------------------------------------------------------------------------ nodes
class _Linear8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, keep):
        r = _runner(x.device)
        x, weight = _aligned(x), weight.contiguous()
        y = _gemm(r, x, weight, _maybe(bias), _maybe(residual))
        q = s = None
        if keep:                                          # only the weight gradient reads the input
            q, s = pack(x)
        ctx.save_for_backward(weight, q, s)
        ctx.amp = T.AMP_STEP[0]
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        weight, q, s = ctx.saved_tensors
        dy = _aligned(dy)
        r = _runner(dy.device)
        need = ctx.needs_input_grad
        dx = _dgrad(dy, weight, ctx.amp) if need[0] else None
        dw = db = None
        if need[1]:
            dw, db = _wgrad(r, 0, dy, q, s, weight.shape[1], want_b=need[2])
        elif need[2]:
            db = _bias_grad(r, dy)
        return dx, dw, db, dy if need[3] else None, None


class _NormLinear8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, weight, bias):
        r = _runner(x.device)
        x, weight, gamma, beta = _aligned(x), weight.contiguous(), _aligned(gamma), _aligned(beta)
        rows, c, q, s = _empty_pack(x)
        xn, stats = torch.empty_like(x), torch.empty((rows, 2), dtype=torch.float32, device=x.device)
        _lib.check(r.lib.av2x_act8_layernorm(_P(x), _P(gamma), _P(beta), _P(xn), _P(q), _P(s), _P(stats), rows, c, LN_EPS, r.stream()), "av2x_act8_layernorm")
        y = _gemm(r, xn, weight, _maybe(bias), None)
        ctx.save_for_backward(weight, gamma, beta, q, s, stats)
        ctx.amp = T.AMP_STEP[0]
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        weight, gamma, beta, q, s, stats = ctx.saved_tensors
        dy = _aligned(dy)
        r = _runner(dy.device)
        need = ctx.needs_input_grad
        rows, c = stats.shape[0], weight.shape[1]
        dx = dgamma = dbeta = dw = db = None
        if need[1] or need[2] or need[3]:
            # dgamma, dbeta need no pass over the rows: they are sums over the weight gradient's sum dY^T u and over db
            dgamma = torch.empty_like(gamma) if need[1] else None
            dbeta = torch.empty_like(beta) if need[2] else None
            dw, db = _wgrad(r, 1, dy, q, s, c, stats, gamma, beta, need[3], need[4], weight, dgamma, dbeta)
        elif need[4]:
            db = _bias_grad(r, dy)
        if need[0]:
            dx = _dgrad(dy, weight, ctx.amp)
            # in place: a wave has read its row before it writes it
            _lib.check(r.lib.av2x_act8_layernorm_backward(_P(q), _P(s), _P(stats), _P(gamma), _P(dx), _P(dx), rows, c, r.stream()), "av2x_act8_layernorm_backward")
        return dx, dgamma, dbeta, dw, db


class _Gelu8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z):
        h, q, s = _gelu_forward(_runner(z.device), _aligned(z))
        ctx.save_for_backward(q, s)
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        q, s = ctx.saved_tensors
        dh = _aligned(dh)
        return _gelu_backward(_runner(dh.device), q, s, dh)


def _gelu_backward(r, q, s, dh, out=None):
    dz = torch.empty_like(dh) if out is None else out
    c = dh.shape[-1]
    _lib.check(r.lib.av2x_act8_gelu_backward(_P(q), _P(s), _P(dh), _P(dz), dh.numel() // c, c, r.stream()), "av2x_act8_gelu_backward")
    return dz


class _GeluLinear8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, weight, bias, residual):
        r = _runner(z.device)
        z, weight = _aligned(z), weight.contiguous()
        h, q, s = _gelu_forward(r, z)
        y = _gemm(r, h, weight, _maybe(bias), _maybe(residual))
        ctx.save_for_backward(weight, q, s)
        ctx.amp = T.AMP_STEP[0]
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        weight, q, s = ctx.saved_tensors
        dy = _aligned(dy)
        r = _runner(dy.device)
        need = ctx.needs_input_grad
        dz = dw = db = None
        if need[0]:
            dh = _dgrad(dy, weight, ctx.amp)
            dz = _gelu_backward(r, q, s, dh, dh)          # element by element, in place
        if need[1]:
            dw, db = _wgrad(r, 2, dy, q, s, weight.shape[1], want_b=need[2])
        elif need[2]:
            db = _bias_grad(r, dy)
        return dz, dw, db, dy if need[3] else None


def linear(x, weight, bias=None, residual=None):
    """x W^T (+ b) (+ residual) over the last axis; W is nn.Linear's (cout, cin).  Keeps x in 8 bits for dW."""
    _check("linear", x, weight, bias, residual)
    return _Linear8.apply(x, weight, bias, residual, torch.is_grad_enabled() and weight.requires_grad)


def norm_linear(x, gamma, beta, weight, bias=None):
    """LayerNorm(x) W^T (+ b), eps 1e-5; at most 1024 channels.  Keeps x in 8 bits and two statistics a row for both backward passes."""
    _check("norm_linear", x, weight, bias, None, (gamma, beta), 1024)
    return _NormLinear8.apply(x, gamma, beta, weight, bias)


def gelu(z):
    """Exact GELU; keeps z in 8 bits."""
    _check("gelu", z)
    return _Gelu8.apply(z)


def gelu_linear(z, weight, bias=None, residual=None):
    """gelu(z) W^T (+ b) (+ residual).  Keeps z in 8 bits; the weight gradient evaluates gelu(z8) while it reads."""
    _check("gelu_linear", z, weight, bias, residual)
    return _GeluLinear8.apply(z, weight, bias, residual)
