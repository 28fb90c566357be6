"""CPU: the global attention layer as a module -- moves and casts."""
import pytest
import torch

from airv2x_perception_amd.opencood_iface import token_attention as A


@pytest.mark.parametrize("cast", [lambda m: m.float(), lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.double(), lambda m: m.to(torch.float32), lambda m: m.half().float(),
                                  lambda m: m.to("meta").to_empty(device="cpu"), lambda m: m.to("cpu"), lambda m: m.share_memory(), lambda m: __import__("copy").deepcopy(m).float()])
def test_a_cast_leaves_the_frequencies(cast):
    m = A.BlockSparseAttention(64, 2, 32, axes=1, base=500.0)
    own = torch.rand(16, dtype=torch.float64)
    want = A.rotation_freqs(32, 1, 500.0)
    assert torch.equal(m.freqs, want)
    got = cast(m)
    assert got.freqs.dtype == torch.float64 and torch.equal(got.freqs, want)
    assert "freqs" not in got.state_dict() and dict(got.named_buffers())["freqs"] is got.freqs
    got.freqs = own                                              # somebody's own frequencies are kept too
    assert torch.equal(got.float().freqs, own)


def test_a_layer_built_without_storage():
    with torch.device("meta"):
        m = A.BlockSparseAttention(64, 2, 32)
    assert m.freqs.is_meta
    m = m.to_empty(device="cpu")
    assert torch.equal(m.freqs, A.rotation_freqs(32, 2))


@pytest.mark.parametrize("scope,flag", [("act8_scope", "ACT8_STEP"), ("amp_scope", "AMP_STEP")])
def test_a_steps_flags_are_its_threads(scope, flag):
    """Two models in forward on two threads: neither sees the other's setting, in either order of entering and leaving."""
    import threading
    from airv2x_perception_amd.opencood_iface import train_ops as T
    scope, flag = getattr(T, scope), getattr(T, flag)
    inside, leave, seen = threading.Event(), threading.Event(), []

    def other():
        with scope(True):
            inside.set()
            leave.wait(20)
            seen.append(flag[0])
        seen.append(flag[0])

    t = threading.Thread(target=other)
    t.start()
    assert inside.wait(20)
    assert flag == [False] and not flag[0]
    with scope(True):
        with scope(False):
            leave.set()
            t.join(20)
            assert not flag[0]
        assert flag[0]
    assert not flag[0] and seen == [True, False]
