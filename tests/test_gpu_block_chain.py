"""The operators as they are used together: norm with the residual -> router -> rows by expert ->
gated rows -> the down projections' Hessians, solve and packing -> product with the packed weights."""
import pytest
import torch

from block_ref import NORM_F32, gated64, half_step, int4_64, norm64, within
from forge import engine, export
from forge.moe import ExpertGroupGPTQ

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_calibrate_solve_and_run_a_block(hip):
    g = torch.Generator(device=DEV).manual_seed(0)
    mk = lambda s, *sh: (s * torch.randn(*sh, generator=g, device=DEV)).bfloat16()   # noqa: E731
    T, H, I, E, K = 220, 256, 128, 6, 2
    hidden, attn, w = mk(1.0, T, H), mk(0.5, T, H), mk(1.0, H)
    router = mk(0.1, E, H)
    wg, wu, wd = mk(0.06, E, I, H), mk(0.06, E, I, H), mk(0.06, E, H, I)

    normed, stream = engine.rms_norm(attn, w, residual=hidden)
    y64, s64 = norm64(attn, w, 1e-6, hidden)
    hs = half_step(torch.bfloat16)
    within(normed, y64, (hs + NORM_F32) * y64.abs())
    within(stream, s64, (hs + 2 ** -23) * s64.abs())

    logits = normed.float() @ router.float().T
    logits[:, 4] = -1e9                                            # an expert without rows
    rw, ri = torch.softmax(logits, -1).topk(K, dim=-1)
    rows, offs = engine.routed_rows(normed, ri, None, E)
    h = engine.expert_gated_rows(rows, offs, wg, wu)
    want, bound = gated64(rows, offs, wg, wu, "silu")
    within(h, want, bound)

    group = ExpertGroupGPTQ([wd], bits=4, group_size=128, symmetric=True, device=DEV)
    group.update(h, offs)
    (codes, scales, zeros), = group.quantize()
    out = torch.zeros(T, H, dtype=torch.float64, device=DEV)
    for e in range(E):
        rec = export.pack_weight(export.layer_record(codes[e], scales[e], zeros[e], 128, 4, (H, I)), 4, True, 128)
        he = h[offs[e]:offs[e + 1]]
        ye = engine.linear_int4(he, rec, group_size=128)
        want, bound = int4_64(he, rec["weight_packed"], rec["weight_scale"], 128, None, None, None)
        within(ye, want, bound)
        if he.shape[0]:
            # the solved weights do the original weights' work: 4 bits of random weights leave about
            # 1/sqrt(12) of a step of max|w|/7 ~ 0.4 sigma, i.e. 0.12 of the output, never half of it
            ref = he.double() @ wd[e].double().T
            assert (ye.double() - ref).norm() < 0.5 * ref.norm()
    assert out.shape == (T, H)


def test_on_another_device_than_the_current_one_is_the_tensors_own(hip):
    """every operator works on its tensors' device; tensors of two devices are refused"""
    x = torch.randn(4, 64, device="cuda:0").bfloat16()
    with pytest.raises(RuntimeError):
        engine.rms_norm(x, torch.ones(64).bfloat16())
    with pytest.raises(RuntimeError):
        engine.expert_gated_rows(x, [0, 4], torch.zeros(1, 8, 64).bfloat16(), torch.zeros(1, 8, 64).bfloat16())
    with pytest.raises(RuntimeError):
        engine.linear_int4(x.cpu(), dict(weight_packed=torch.zeros(8, 8, dtype=torch.int32),
                                         weight_scale=torch.ones(8, 1), weight_shape=torch.tensor([8, 64])))
