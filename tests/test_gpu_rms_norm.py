"""rms_norm and rms_norm_fp8 against their float64 forms (tests/block_ref.py)."""
import pytest
import torch

from block_ref import NORM_F32, half_step, norm64, within
from forge import engine

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _inputs(T, C, dtype, seed, residual=True, pitch=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    mk = lambda s: (s * torch.randn(T, C + pitch, generator=g, device=DEV)).to(dtype)[:, :C]   # noqa: E731
    return mk(1.0), (1 + 0.1 * torch.randn(C, generator=g, device=DEV)).to(dtype), mk(3.0) if residual else None


def _check(out, x, w, r, eps=1e-6):
    y, s = norm64(x, w, eps, r)
    hs = half_step(x.dtype)
    if r is None:
        within(out, y, (hs + NORM_F32) * y.abs())
    else:
        within(out[0], y, (hs + NORM_F32) * y.abs())
        within(out[1], s, (hs + 2 ** -23) * s.abs())


SHAPES = [(1, 1), (1, 7168), (3, 8), (5, 129), (7, 2047), (33, 2048), (130, 2056), (4, 8192), (3, 8200),
          (2, 16384), (2, 16392), (2, 20001), (1025, 768)]


@pytest.mark.parametrize("T,C", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("residual", [False, True], ids=["plain", "residual"])
def test_norm(hip, T, C, dtype, residual):
    x, w, r = _inputs(T, C, dtype, T * C, residual)
    _check(engine.rms_norm(x, w, residual=r), x, w, r)


def _check_fp8(codes, scale, x, w, r, eps=1e-6):
    T, C = x.shape
    y, _ = norm64(x, w, eps, r)
    G = (C + 127) // 128
    assert codes.dtype == torch.float8_e4m3fn and tuple(scale.shape) == (T, G) and scale.dtype == torch.float32
    m = torch.stack([y[:, g * 128:(g + 1) * 128].abs().amax(-1) for g in range(G)], 1).clamp_min(1e-12) / 448
    within(scale, m, (NORM_F32 + 2 ** -23) * m)
    v = y / m.repeat_interleave(128, 1)[:, :C]
    # half a step of e4m3: 2^-4 of the value, 2^-10 where the exponent has run out
    got = codes.float().double()
    over = (got - v).abs() - (2 ** -4 * v.abs()).clamp_min(2 ** -10) - 4 * NORM_F32 * v.abs()
    assert (over <= 0).all(), over.max()
    # and nearest: the next code up or down is never nearer than rounding noise explains
    assert got.abs().max() <= 448


@pytest.mark.parametrize("T,C", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_norm_fp8(hip, T, C, dtype):
    for residual in (False, True):
        x, w, r = _inputs(T, C, dtype, T + C, residual)
        out = engine.rms_norm_fp8(x, w, residual=r)
        _check_fp8(out[0], out[1], x, w, r)
        if residual:
            s = norm64(x, w, 1e-6, r)[1]
            within(out[2], s, (half_step(dtype) + 2 ** -23) * s.abs())


def test_norm_fp8_reads_back_through_the_block_dequant(hip):
    x, w, r = _inputs(64, 1024, torch.bfloat16, 3)
    codes, scale, _ = engine.rms_norm_fp8(x, w, residual=r)
    y = hip.fp8_block_dequant(codes, scale, torch.float32)
    assert torch.equal(y, codes.float() * scale.repeat_interleave(128, 1))
    ref = norm64(x, w, 1e-6, r)[0]
    m = ref.view(64, 8, 128).abs().amax(-1, keepdim=True).expand(-1, -1, 128).reshape(64, 1024) / 448
    assert ((y.double() - ref).abs() <= (2 ** -4 * ref.abs()).clamp_min(2 ** -10 * m) * (1 + 1e-4)).all()


@pytest.mark.parametrize("pitch,shift", [(8, 0), (3, 0), (8, 1), (16, 8)])
def test_norm_pitch_and_alignment(hip, pitch, shift):
    """rows of a wider tensor, starting off the 16-byte grid, the residual with a pitch of its own"""
    T, C = 19, 512
    g = torch.Generator(device=DEV).manual_seed(pitch)
    big = torch.randn(T, C + pitch + shift, generator=g, device=DEV).bfloat16()
    x = big[:, shift:shift + C]
    r = torch.randn(T, 2 * C, generator=g, device=DEV).bfloat16()[:, C:]
    w = torch.randn(C, generator=g, device=DEV)                       # f32 weight over bf16 rows
    _check(engine.rms_norm(x, w, residual=r), x, w, r)
    out = engine.rms_norm_fp8(x, w, residual=r)
    _check_fp8(out[0], out[1], x, w, r)
    # transposed and expanded inputs
    xt = torch.randn(C, T, generator=g, device=DEV).bfloat16().t()
    _check(engine.rms_norm(xt, w, residual=r[:1].expand(T, C)), xt, w, r[:1].expand(T, C))


def test_norm_shapes_empty_and_leading_dimensions(hip):
    w = torch.ones(64, device=DEV).bfloat16()
    x = torch.randn(2, 3, 5, 64, device=DEV).bfloat16()
    y, s = engine.rms_norm(x, w, residual=x)
    assert y.shape == s.shape == x.shape and torch.equal(s, x + x)
    assert engine.rms_norm(x[0, 0, 0], w).shape == (64,)
    assert engine.rms_norm(x[:0], w).shape == (0, 3, 5, 64)
    c, sc = engine.rms_norm_fp8(x[:0], w)
    assert c.shape == (0, 3, 5, 64) and sc.shape == (0, 3, 5, 1)
    assert torch.equal(engine.rms_norm(x.view(-1, 64), w).view(x.shape), engine.rms_norm(x, w))


@pytest.mark.parametrize("C", [512, 513])
def test_norm_special_values(hip, C):
    """zero rows, infinities and NaN stay in their own row (and, in 8 bits, make their runs NaN)"""
    x = torch.randn(6, C, device=DEV).bfloat16()
    x[1] = 0
    x[2, 7] = float("nan")
    x[3, 300] = float("inf")
    x[4] = 1e-30
    w = torch.ones(C, device=DEV).bfloat16()
    y = engine.rms_norm(x, w)
    v = x.float()
    want = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-6)
    assert (y[1] == 0).all() and torch.isnan(y[2]).all()
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.isfinite(y[[0, 1, 4, 5]]).all()
    codes, scale = engine.rms_norm_fp8(x, w)
    assert (codes[1].float() == 0).all() and (scale[1] > 0).all()
    assert torch.isnan(scale[2]).all() and torch.isnan(codes[2].float()).all()
    assert torch.isnan(codes[3].float()[300]) and torch.isnan(scale[3, 2]) and scale[3, 0] > 0
    assert torch.isfinite(codes[[0, 1, 4, 5]].float()).all()


def test_norm_large_row_offset(hip):
    """row offsets past 2^31 elements (a strided view keeps the memory small)"""
    C, T = 64, 3
    pitch = (1 << 30) + 8
    buf = torch.empty((T - 1) * pitch + C, dtype=torch.bfloat16, device=DEV)
    x = buf.as_strided((T, C), (pitch, 1))
    g = torch.Generator(device=DEV).manual_seed(1)
    x.copy_(torch.randn(T, C, generator=g, device=DEV).bfloat16())
    w = torch.ones(C, device=DEV).bfloat16()
    _check(engine.rms_norm(x, w, residual=x), x, w, x)
