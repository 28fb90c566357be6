"""GPU: recorded steps of the token operators and of the layer made of them, replayed with weights that changed since the recording, against eager steps.

A backward pass is recorded only while no eager graph of the same leaves is alive, so a step keeps none.
"""
import copy

import pytest
import torch

from tests.test_gpu_token_layer import layer

pytestmark = pytest.mark.gpu


def on_a_side_stream(f):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        f()
    torch.cuda.current_stream().wait_stream(s)


def make_step(m, t=260):
    g = torch.Generator().manual_seed(t)
    x = torch.randn(1, t, 256, generator=g).cuda().requires_grad_()
    dy = torch.randn(1, t, 256, generator=g).cuda()
    pos = torch.stack([torch.arange(t) // 20, torch.arange(t) % 20], 1).int().cuda()

    def step(m=m):
        y = m(x, pos)
        return [y.detach()] + list(torch.autograd.grad(y, [x] + list(m.parameters()), dy))
    return step


@pytest.mark.parametrize("act8", [False, True])
@pytest.mark.parametrize("warm", [False, True])
def test_a_recorded_layer_follows_its_weights(monkeypatch, warm, act8):
    """With packings of the weights left by an eager step before the recording, and with none; eager calls before the first replay and between replays."""
    from airv2x_perception_amd.opencood_iface import act8_ops as A8, train_ops as T
    monkeypatch.setattr(A8, "SMALL_PRODUCT", 0)                 # every Linear on the GEMM that packs its weights
    m = layer(7, 256, 8, 2, 32, 3)
    m.act8 = act8
    step = make_step(m)
    on_a_side_stream(step if warm else lambda: step(copy.deepcopy(m)))
    if not warm:
        monkeypatch.setattr(T, "_PACKED", {})
        monkeypatch.setattr(T, "_ZEROS", {})
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    want = step(copy.deepcopy(m))
    assert all(torch.equal(a, b) for a, b in zip(step(), want))  # before any replay
    for i in range(3):
        with torch.no_grad():
            for p in m.parameters():
                p.mul_(1 + 0.25 * (i + 1)).add_(0.01)
        graph.replay()
        torch.cuda.synchronize()
        have = [t.clone() for t in got]
        want = step(copy.deepcopy(m))                           # parameters that no cache knows
        assert all(torch.equal(a, b) for a, b in zip(have, want))
        assert all(torch.equal(a, b) for a, b in zip(step(), want))


@pytest.mark.parametrize("recorded,eager", [(0, 0), (1 << 62, 0), (0, 1 << 62)])
@pytest.mark.parametrize("act8", [False, True])
def test_eager_calls_follow_weights_that_replays_change(monkeypatch, act8, recorded, eager):
    """A recorded step of gradient descent changes the weights without moving their version counters: eager calls between its replays use them as they are.
    ``recorded``, ``eager``: which of the 8-bit layers' products the recording and the eager calls run."""
    from airv2x_perception_amd.opencood_iface import act8_ops as A8
    m = layer(9, 256, 8, 2, 32, 3)
    m.act8 = act8
    step = make_step(m)

    def descend():
        for p, g in zip(m.parameters(), step()[2:]):
            with torch.no_grad():
                p.sub_(g, alpha=1e-3)

    monkeypatch.setattr(A8, "SMALL_PRODUCT", recorded)
    on_a_side_stream(descend)
    monkeypatch.setattr(A8, "SMALL_PRODUCT", eager)
    on_a_side_stream(step)                                      # packings of the last eager version
    monkeypatch.setattr(A8, "SMALL_PRODUCT", recorded)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        descend()
    monkeypatch.setattr(A8, "SMALL_PRODUCT", eager)
    before = None
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        got, want = step(), step(copy.deepcopy(m))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert before is None or not torch.equal(before, got[0])
        before = got[0]


def test_packings_are_forgotten_on_demand():
    """A graph that updates weights without running their layers."""
    from airv2x_perception_amd.opencood_iface import train_ops as T
    m = layer(10, 256, 8, 2, 32, 3)
    step = make_step(m)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with torch.no_grad():
            for p in m.parameters():
                p.mul_(1.5)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        T.forget_packings()
        assert all(torch.equal(a, b) for a, b in zip(step(), step(copy.deepcopy(m))))


@pytest.mark.parametrize("act8", [False, True])
def test_a_weight_packed_on_a_busy_stream(monkeypatch, act8):
    """A layer called on two streams at once: the second call does not take a packing (or zeros) that the first stream has yet to write."""
    from airv2x_perception_amd.opencood_iface import act8_ops as A8, train_fusion_ops as F, train_ops as T
    monkeypatch.setattr(A8, "SMALL_PRODUCT", 0)
    g = torch.Generator().manual_seed(17)
    x = torch.randn(1, 10, 20, 256, generator=g).cuda()
    w = torch.nn.Parameter(torch.randn(256, 256, generator=g).cuda())
    f = (lambda w: A8.linear(x, w)) if act8 else (lambda w: F.linear(x, w))
    want = f(copy.deepcopy(w)).detach()
    big = torch.randn(4096, 4096, device="cuda")
    monkeypatch.setattr(T, "_PACKED", {})
    monkeypatch.setattr(T, "_ZEROS", {})
    torch.empty(1 << 22, device="cuda").fill_(float("nan"))          # what freshly taken memory holds
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(one):
        for _ in range(40):                                          # some 40 ms of work
            big = (big @ big).clamp_(-1, 1)
        a = f(w).detach()
    with torch.cuda.stream(two):
        b = f(w).detach()
    two.synchronize()
    got = b.cpu()
    torch.cuda.synchronize()
    assert torch.equal(got, want.cpu()) and torch.equal(a, want)
