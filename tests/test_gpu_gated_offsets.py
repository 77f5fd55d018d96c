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
