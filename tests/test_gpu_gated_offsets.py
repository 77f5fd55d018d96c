"""expert_gated_rows and offsets that are not what routed_rows returns."""
import pytest
import torch

from block_ref import gated64, within
from forge import engine

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _inputs(N, E, H, I, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    mk = lambda s, *sh: (s * torch.randn(*sh, generator=g, device=DEV)).bfloat16()   # noqa: E731
    return mk(1.0, N, H), mk(H ** -0.5, E, I, H), mk(H ** -0.5, E, I, H), mk(1.0, N, I)


@pytest.mark.parametrize("N", [70, 600])
def test_wide_offsets_outside_the_rows_are_clamped(hip, N):
    rows, wg, wu, dh = _inputs(N, 3, 64, 48)
    for offs, same in (([0, 2 ** 32 + 3, 2 ** 33, 2 ** 40], [0, N, N, N]), ([0, 20, 2 ** 31 + 5, 2 ** 32], [0, 20, N, N]),
                       ([-2 ** 32 + 7, -2 ** 31 - 1, 9, N + 1], [0, 0, 9, N]), ([2 ** 32] * 4, [N] * 4)):
        want, bound = gated64(rows, same, wg, wu, "silu")
        leaf = rows.clone().requires_grad_(True)
        h = engine.expert_gated_rows(leaf, torch.tensor(offs, device=DEV), wg, wu)
        within(h.detach(), want, bound)
        plain = rows.clone().requires_grad_(True)
        h2 = engine.expert_gated_rows(plain, torch.tensor(same, device=DEV), wg, wu)
        assert torch.equal(h, h2)
        assert torch.equal(torch.autograd.grad(h, leaf, dh)[0], torch.autograd.grad(h2, plain, dh)[0])


@pytest.mark.parametrize("N", [0, 1, 33, 700])
def test_dense_rows_need_nothing_of_the_host(hip, N):
    """offsets None: the same as [0, N], eager, in training and captured"""
    rows, wg, wu, dh = _inputs(N, 1, 72, 40, seed=N)
    want, bound = gated64(rows, [0, N], wg, wu, "silu")
    leaves = [t.clone().requires_grad_(True) for t in (rows, wg[0], wu[0])]
    h = engine.expert_gated_rows(leaves[0], None, leaves[1], leaves[2])
    within(h.detach(), want, bound)
    same = [t.clone().requires_grad_(True) for t in (rows, wg[0], wu[0])]
    h2 = engine.expert_gated_rows(same[0], [0, N], same[1], same[2])
    assert torch.equal(h, h2)
    for a, b in zip(torch.autograd.grad(h, leaves, dh), torch.autograd.grad(h2, same, dh)):
        assert torch.equal(a, b)
    if N == 0:
        return
    with torch.no_grad():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = engine.expert_gated_rows(rows, None, wg[0], wu[0])
        for k in range(3):
            rows.mul_(1 + k)
            out.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, engine.expert_gated_rows(rows, None, wg[0], wu[0]))
            torch.randn(500, 500, device=DEV).sum().item()


def test_offsets_on_the_host_are_not_captured(hip):
    rows, wg, wu, _ = _inputs(50, 2, 64, 48)
    o = torch.tensor([0, 20, 50], dtype=torch.int32, device=DEV)
    want = engine.expert_gated_rows(rows, o, wg, wu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for host in ([0, 20, 50], o.new_tensor([0, 20, 50], device="cpu")):
            with pytest.raises(RuntimeError, match="cannot be captured"):
                engine.expert_gated_rows(rows, host, wg, wu)
        out = engine.expert_gated_rows(rows, o, wg, wu)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
