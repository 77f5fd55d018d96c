"""The 8-bit norm's codes are the nearest to y / scale_inv, y being what rms_norm gives for the same rows in f32
(the two share their arithmetic): every code bit for bit, values between two codes among them."""
import pytest
import torch

from forge import engine

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("T,C", [(4099, 2048), (1, 7168), (3, 8), (5, 129), (64, 4096), (33, 2047), (9, 8200), (2, 20001),
                                 (200, 136)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("residual", [False, True], ids=["plain", "residual"])
def test_codes_are_the_nearest(hip, T, C, dtype, residual):
    g = torch.Generator(device=DEV).manual_seed(T + C)
    mk = lambda s: (s * torch.randn(T, C, generator=g, device=DEV)).to(dtype)   # noqa: E731
    x, r, w = mk(1.0), mk(3.0) if residual else None, (1 + 0.1 * torch.randn(C, generator=g, device=DEV)).to(dtype)
    if not residual:                       # rows of few values: quotients of small whole numbers, many of them ties
        x[::2] = x[::2].sign() * torch.randint(0, 29, x[::2].shape, generator=g, device=DEV).to(dtype)
        w = torch.ones_like(w)
    out = engine.rms_norm_fp8(x, w, residual=r)
    codes, scale = out[0], out[1]
    y = engine.rms_norm(x.float(), w, residual=None if r is None else r.float())
    y = y if r is None else y[0]
    per = scale.repeat_interleave(128, 1)[:, :C]
    G = scale.shape[1]
    top = torch.nn.functional.pad(y.abs(), (0, G * 128 - C)).view(T, G, 128).amax(-1).clamp_min(1e-12)
    # (a tensor as the divisor: torch divides a GPU tensor by a number as a product with its reciprocal)
    assert torch.equal(scale, top / torch.full_like(top, 448.0))
    want = (y / per).cpu().to(torch.float8_e4m3fn)
    assert torch.equal(codes.cpu().view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("C", [256, 257])
def test_codes_of_extreme_rows(hip, C):
    """the same where a run's largest value is tiny, huge or infinite"""
    g = torch.Generator(device=DEV).manual_seed(C)
    x = torch.randn(6, C, generator=g, device=DEV)
    w = torch.ones(6, C, device=DEV)
    w[0], w[1], w[2], w[3] = 1e-20, 1e30, 1e37, 1e-11
    for k in range(6):
        x[5, 3] = float("inf") if k == 5 else 1.0
        codes, scale = engine.rms_norm_fp8(x[k:k + 1], w[k], 1e-6)
        y = engine.rms_norm(x[k:k + 1], w[k], 1e-6)
        want = (y / scale.repeat_interleave(128, 1)[:, :C]).cpu().to(torch.float8_e4m3fn).float()
        got = codes.cpu().float()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(), want.nan_to_num())
    assert torch.isnan(got).any() and (got == 0).any()
