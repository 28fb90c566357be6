"""CPU: refusals of the token operators -- in Python before anything is launched, in the C-ABI before any HIP call -- and their sizes."""
import ctypes

import pytest
import torch

from airv2x_perception_amd import _lib
from airv2x_perception_amd.opencood_iface import act8_ops, token_attention as A


def test_there_is_no_cpu_path():
    x = torch.randn(4, 64)
    for f in (lambda: act8_ops.pack(x), lambda: act8_ops.linear(x, torch.randn(32, 64)), lambda: act8_ops.gelu(x), lambda: act8_ops.gelu_linear(x, torch.randn(32, 64)),
              lambda: act8_ops.norm_linear(x, x[0], x[0], torch.randn(32, 64)), lambda: act8_ops.unpack(act8_ops.Packed8(torch.zeros(4, 64, dtype=torch.int8), torch.ones(4, 1))),
              lambda: A.qk_norm_rotate(torch.randn(4, 2, 32), None, torch.ones(32), None, torch.zeros(4, 2, dtype=torch.int32), A.rotation_freqs(32)),
              lambda: A.block_bounds(torch.randn(1, 4, 2, 32)), lambda: A.BlockSparseAttention(64, 2, 32)(torch.randn(1, 4, 64), torch.zeros(4, 2, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="HIP|GPU"):
            f()


def test_rotation_freqs():
    f = A.rotation_freqs(32, 2, 100.0)
    assert f.dtype == torch.float64 and f.shape == (16,) and torch.equal(f[:8], f[8:])
    assert abs(float(f[0]) * 6.283185307179586 - 1) < 1e-15 and abs(float(f[4]) * 6.283185307179586 - 0.1) < 1e-15
    for bad in ((24, 2), (32, 3), (32, 0)):
        with pytest.raises(ValueError):
            A.rotation_freqs(*bad)


def _err():
    return _lib.load().av2x_last_error().decode()


def test_c_abi_refusals_of_the_rotation():
    lib = _lib.load()
    st = (ctypes.c_int64 * 4)(64, 32, 64, 32)
    ok = dict(q=64, k=64, st=st, gq=64, gk=64, pos=64, fr=64, oq=64, ok=64, rows=4, h=2, kv=2, d=32, axes=2, inter=0, dt=0, eps=1e-6)

    def call(**kw):
        a = {**ok, **kw}
        return lib.av2x_qk_norm_rotate(a["q"], a["k"], a["st"], a["gq"], a["gk"], a["pos"], a["fr"], a["oq"], a["ok"], a["rows"], a["h"], a["kv"], a["d"], a["axes"],
                                       a["inter"], a["dt"], a["eps"], None)

    for kw, word in ((dict(d=24), "dim"), (dict(dt=3), "dtype"), (dict(h=0), "heads"), (dict(axes=3), "axes"), (dict(rows=-1), "rows"), (dict(pos=None), "positions"),
                     (dict(q=None), "null"), (dict(k=None), "null"), (dict(q=68), "aligned"), (dict(st=(ctypes.c_int64 * 4)(64, 33, 64, 32)), "strides"), (dict(gq=72), "gamma")):
        assert call(**kw) != 0 and word in _err(), (kw, _err())
    assert call(rows=0) == 0
    assert lib.av2x_qk_norm_rotate_backward_workspace_bytes(32) > 0


def test_c_abi_refusals_of_the_8_bit_layers():
    lib = _lib.load()
    for c, word in ((6, "channels"), (0, "channels"), (-4, "channels")):
        assert lib.av2x_act8_pack(64, 64, 64, 4, c, None) != 0 and word in _err()
    assert lib.av2x_act8_pack(None, 64, 64, 4, 64, None) != 0 and "null" in _err()
    assert lib.av2x_act8_pack(68, 64, 64, 4, 64, None) != 0 and "aligned" in _err()
    assert lib.av2x_act8_pack(64, 64, 64, -1, 64, None) != 0 and "rows" in _err()
    assert lib.av2x_act8_pack(None, None, None, 0, 64, None) == 0
    assert lib.av2x_act8_layernorm(64, 64, 64, 64, 64, 64, 64, 4, 1028, 1e-5, None) != 0 and "1024" in _err()
    wg = lambda kind=0, rows=4, co=8, ci=64, stats=64, gamma=64, dw=64, dg=None, w=None: lib.av2x_act8_wgrad(64, 64, 64, stats, gamma, 64, w, kind, rows, co, ci, dw, 64, dg, None, 64, None)
    for kw, word in ((dict(kind=3), "kind"), (dict(co=6), "outputs"), (dict(ci=2), "channels"), (dict(kind=1, stats=None), "statistics"), (dict(kind=1, gamma=None), "statistics"),
                     (dict(dw=8), "aligned"), (dict(dg=64, w=64), "LayerNorm"), (dict(kind=1, dg=64), "weight")):
        assert wg(**kw) != 0 and word in _err(), (kw, _err())
    # slabs for every split of the rows, and two sums an output
    assert lib.av2x_act8_wgrad_workspace_bytes(1, 8, 64) == (2 * 8 * 64 + 3 * 8) * 4
    assert lib.av2x_act8_wgrad_workspace_bytes(10 ** 6, 256, 256) <= 513 * (256 * 256 + 512) * 4
    gemm = lambda a=64, rows=4, n=64, k=64: lib.av2x_act8_gemm(a, 64, None, None, 64, rows, n, k, 0, None)
    for kw, word in ((dict(a=None), "null"), (dict(a=72), "aligned"), (dict(k=48), "multiple of 32"), (dict(n=6), "of 4"), (dict(rows=-1), "rows")):
        assert gemm(**kw) != 0 and word in _err(), (kw, _err())
    assert gemm(rows=0, a=None) == 0


def test_c_abi_refusals_of_the_blocks():
    lib = _lib.load()
    s3, s9 = (ctypes.c_int64 * 3)(1024, 64, 32), (ctypes.c_int64 * 9)(*[1024, 64, 32] * 3)
    bounds = lambda k=64, b=1, n=100, kv=2, d=32, dt=0, first=0, count=2, st=s3: lib.av2x_block_bounds(k, None, st, b, n, kv, d, dt, first, count, 64, 64, None)
    for kw, word in ((dict(d=48), "dim"), (dict(dt=5), "dtype"), (dict(first=1), "blocks 1 .. 3 of 2"), (dict(first=-1), "blocks"), (dict(count=-1), "blocks"), (dict(k=None), "null"),
                     (dict(k=72), "aligned"), (dict(st=(ctypes.c_int64 * 3)(1024, 66, 32)), "aligned"), (dict(n=2 ** 21 + 1), "keys"), (dict(b=0), "batch")):
        assert bounds(**kw) != 0 and word in _err(), (kw, _err())
    assert bounds(count=0, k=None) == 0
    sel = lambda q=64, t=4, h=2, kv=2, d=32, n=2, ints=64: lib.av2x_select_blocks(q, s3, ints, 64, 1, t, 100, h, kv, d, n, 0, 64, None, None)
    for kw, word in ((dict(n=0), "blocks"), (dict(n=65), "blocks"), (dict(h=3), "heads"), (dict(h=34, kv=1), "share"), (dict(h=16, kv=1, d=128), "share"), (dict(q=None), "null"),
                     (dict(ints=72), "16 bytes"), (dict(t=2 ** 26), "queries")):
        assert sel(**kw) != 0 and word in _err(), (kw, _err())
    att = lambda q=64, k=64, t=4, blocks=64, lists=None, out=64, st=s9, ws=64: lib.av2x_block_sparse_attention(q, k, 64, st, None, blocks, lists, 1, t, 100, 2, 2, 32, 2, 0, 1.0, out, None, None, ws, None)
    for kw, word in ((dict(q=None), "null"), (dict(k=72), "aligned"), (dict(blocks=None), "null"), (dict(out=72), "unaligned"), (dict(ws=None), "null"), (dict(lists=72), "unaligned"),
                     (dict(st=(ctypes.c_int64 * 9)(*[1024, 66, 32] * 3)), "aligned")):
        assert att(**kw) != 0 and word in _err(), (kw, _err())
    assert att(t=0, q=None) == 0
    back = lambda lists=64, t=4, n=100, dk=64: lib.av2x_block_sparse_attention_backward(64, 64, 64, s9, None, 64, lists, 64, None, 64, 64, 1, t, n, 2, 2, 32, 2, 0, 1.0, 64, dk, 64, 64, None)
    for kw, word in ((dict(lists=None), "null"), (dict(t=0), "no queries"), (dict(n=0), "no keys"), (dict(dk=72), "unaligned")):
        assert back(**kw) != 0 and word in _err(), (kw, _err())
    assert lib.av2x_block_lists(64, 1, 4, 100, 2, 2, 2, None, None) != 0 and "null" in _err()
    # the mentions, the starts, the items (one per 512 rows and block) fit
    assert lib.av2x_block_lists_bytes(1, 1000, 640, 4, 2, 3) >= 4 * (2 * 3000 + 2 * 11 + 2 * 2 * (6000 // 512 + 10))
    assert lib.av2x_block_sparse_workspace_bytes(1, 100, 640, 4, 2, 32, 3, 0) >= 4 * (100 * 4 * 3 * (32 + 2))


def test_module_declares_its_parameters():
    m = A.BlockSparseAttention(256, 8, 32, blocks=8, kv_heads=2)
    assert {k: tuple(v.shape) for k, v in m.state_dict().items()} == {
        "q_gamma": (32,), "k_gamma": (32,), "norm.weight": (256,), "norm.bias": (256,), "to_qkv.weight": (384, 256), "to_out.weight": (256, 256), "to_out.bias": (256,)}
    with pytest.raises(ValueError):
        A.BlockSparseAttention(256, 8, 32, kv_heads=3)


def test_the_bindings_have_the_headers_types():
    import os
    import re
    txt = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "airv2x_hip.h")).read()
    txt = re.sub(r"/\*.*?\*/", "", txt, flags=re.S)
    types = {"int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "uint64_t": ctypes.c_uint64, "float": ctypes.c_float, "int": ctypes.c_int32, "av2x_stream_t": ctypes.c_void_p}
    seen = 0
    for res, name, args in re.findall(r"(\w+)\s+(av2x_(?:qk_|act8_|block_|select_)\w+)\s*\((.*?)\);", txt, re.S):
        want = [ctypes.c_void_p if "*" in a else types[a.split()[0]] for a in args.split(",")]
        assert _lib.SIGNATURES[name] == (types[res], want), name
        seen += 1
    assert seen >= 18
