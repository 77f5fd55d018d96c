"""expert_gated_rows where its schedule and its offsets have room to go wrong: many experts with few rows
beside a few with many, and tensors of more than 2^31 elements."""
import pytest
import torch

from block_ref import gated64, within
from forge import engine

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _check(rows, offs, wg, wu, dh):
    leaves = [t.clone().requires_grad_(True) for t in (rows, wg, wu)]
    h = engine.expert_gated_rows(leaves[0], offs, leaves[1], leaves[2])
    grads = torch.autograd.grad(h, leaves, dh)
    (want, bound), wants = gated64(rows, offs, wg, wu, "silu", dh)
    within(h.detach(), want, bound)
    for got, (w, b) in zip(grads, wants):
        within(got, w, b)


@pytest.mark.parametrize("big", [(), (700, 300), (5000,)], ids=["small", "two-big", "one-big"])
@pytest.mark.parametrize("H,I", [(1288, 648), (264, 128)])
def test_experts_with_few_rows_between_the_others(hip, big, H, I):
    g = torch.Generator(device=DEV).manual_seed(H + len(big))
    counts = [1 + (37 * e) % 130 for e in range(70)]
    for i, n in enumerate(big):
        counts[20 + 15 * i] = n
    counts[3] = counts[69] = 0
    offs = [0] + torch.tensor(counts).cumsum(0).tolist()
    mk = lambda s, *sh: (s * torch.randn(*sh, generator=g, device=DEV)).bfloat16()   # noqa: E731
    N, E = offs[-1], len(counts)
    _check(mk(1.0, N, H), offs, mk(H ** -0.5, E, I, H), mk(H ** -0.5, E, I, H), mk(1.0, N, I))


def test_rows_behind_two_to_the_31st_element(hip):
    N, H, I, k = 300_100, 7168, 24, 70
    g = torch.Generator(device=DEV).manual_seed(1)
    mk = lambda s, *sh: (s * torch.randn(*sh, generator=g, device=DEV)).bfloat16()   # noqa: E731
    rows = torch.zeros(N, H, dtype=torch.bfloat16, device=DEV)
    rows[-k:] = mk(1.0, k, H)
    wg, wu, dh = mk(H ** -0.5, 1, I, H), mk(H ** -0.5, 1, I, H), torch.zeros(N, I, device=DEV).bfloat16()
    dh[-k:] = mk(1.0, k, I)
    offs = torch.tensor([N - k, N], dtype=torch.int32, device=DEV)
    h, gate, up = hip.gated_rows(rows, offs, wg, wu, "silu", keep=True)
    dx, dwg, dwu = hip.gated_rows_backward(dh, gate, up, rows, offs, wg, wu)
    (want, bound), wants = gated64(rows[-k:], [0, k], wg, wu, "silu", dh[-k:])
    within(h[-k:], want, bound)
    for got, (w, b) in zip((dx[-k:], dwg, dwu), wants):
        within(got, w, b)
    assert not h[:-k].any() and not dx[:-k].any()


def test_weights_behind_two_to_the_31st_element(hip):
    E, H, I, k = 150, 7168, 2048, 300
    g = torch.Generator(device=DEV).manual_seed(2)
    mk = lambda s, *sh: (s * torch.randn(*sh, generator=g, device=DEV)).bfloat16()   # noqa: E731
    wg, wu = (torch.zeros(E, I, H, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    wg[-1], wu[-1] = mk(H ** -0.5, I, H), mk(H ** -0.5, I, H)
    rows, dh = mk(1.0, k, H), mk(1.0, k, I)
    offs = torch.tensor([0] * E + [k], dtype=torch.int32, device=DEV)
    h, gate, up = hip.gated_rows(rows, offs, wg, wu, "silu", keep=True)
    dx, dwg, dwu = hip.gated_rows_backward(dh, gate, up, rows, offs, wg, wu)
    (want, bound), wants = gated64(rows, [0, k], wg[-1:], wu[-1:], "silu", dh)
    within(h, want, bound)
    for got, (w, b) in zip((dx, dwg[-1:], dwu[-1:]), wants):
        within(got, w, b)
    assert not dwg[:-1].any() and not dwu[:-1].any()


@pytest.mark.parametrize("I", [40, 41])
def test_gradients_of_gradients_are_refused(hip, I):
    g = torch.Generator(device=DEV).manual_seed(I)
    mk = lambda *sh: (0.3 * torch.randn(*sh, generator=g, device=DEV)).bfloat16()   # noqa: E731
    x, wg, wu = (t.requires_grad_(True) for t in (mk(10, 24), mk(2, I, 24), mk(2, I, 24)))
    h = engine.expert_gated_rows(x, [0, 4, 10], wg, wu)
    for leaf in (x, wg, wu):                          # also where the incoming gradient asks for none
        with pytest.raises(RuntimeError, match="gradients of its gradients"):
            torch.autograd.grad(h.sum(), leaf, create_graph=True)
    torch.autograd.grad(h.sum(), (x, wg, wu))


def test_tensors_on_different_devices_are_refused_in_training(hip):
    x = torch.randn(4, 16, device=DEV).bfloat16().requires_grad_(True)
    w = torch.randn(1, 8, 16).bfloat16()
    with pytest.raises(RuntimeError):
        engine.expert_gated_rows(x, [0, 4], w, w)


def test_training_is_not_captured_through_autograd(hip):
    """refused, with the leaves' eager graph alive; without gradients the same call is captured"""
    g = torch.Generator(device=DEV).manual_seed(9)
    mk = lambda *sh: (0.3 * torch.randn(*sh, generator=g, device=DEV)).bfloat16()   # noqa: E731
    x, wg, wu = (t.requires_grad_(True) for t in (mk(10, 24), mk(2, 40, 24), mk(2, 40, 24)))
    offs = torch.tensor([0, 4, 10], dtype=torch.int32, device=DEV)
    alive = engine.expert_gated_rows(x, offs, wg, wu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            engine.expert_gated_rows(x, offs, wg, wu)
        with torch.no_grad():
            h = engine.expert_gated_rows(x, offs, wg, wu)
    for _ in range(3):
        h.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(h, alive)
    alive.sum().backward()
    assert x.grad is not None and wg.grad is not None
