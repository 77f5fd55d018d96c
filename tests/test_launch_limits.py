"""Sizes at which one launch would have 2^32 threads or more: the norm takes them in several launches, what is not
taken is refused before a launch."""
import ctypes

import pytest
import torch

DEV = "cuda"


def test_refused_before_a_launch():
    from forge.backend.hip import load_library
    lib, P = load_library(), ctypes.c_void_p(4096)     # never dereferenced: every call is refused
    err = lib.forge_last_error
    assert lib.forge_pad_rows(P, 0, 128, P, 1, 1 << 29, 128, 1 << 29, 128, None, None) == 1 and b"too large" in err()
    E = 65535
    assert lib.forge_gated_rows(P, 8, P, P, P, 8, 8 * 16384, E, E, 8, 16384, 1, P, None, None, None) == 1
    assert b"workgroups" in err()
    assert lib.forge_gated_rows_backward(P, P, P, P, 16384, P, P, P, 16384, 16384 * 16, E, E, 16384 * 2, 8, 1, P, P, P, P,
                                         1 << 40, None) == 1 and b"row pitch" in err()
    H = 32768
    assert lib.forge_gated_rows_backward(P, P, P, P, H, P, P, P, H, H * 8, E, E, H, 8, 1, P, P, P, P, 1 << 40, None) == 1
    assert b"workgroups" in err()
    assert lib.forge_linear_int4(P, 32, P, P, 32, None, None, 0, 1 << 30, 32, 256, 0, P, None) == 1
    assert b"workgroups" in err()
    assert lib.forge_linear_int4(P, 7, P, P, 3, None, None, 0, 1 << 30, 7, 8, 0, P, None) == 1
    assert b"workgroups" in err()


@pytest.mark.gpu
@pytest.mark.parametrize("T,C,fp8", [((1 << 24) + 5, 3, False), ((1 << 24) + 5, 3, True), ((1 << 26) + 7, 8, False),
                                     ((1 << 26) + 7, 8, True)])
def test_norm_of_very_many_rows(hip, T, C, fp8):
    """the rows on either side of the border between two launches and the last ones, against the same rows alone"""
    from forge import engine
    g = torch.Generator(device=DEV).manual_seed(C)
    x = torch.randn(T, C, generator=g, device=DEV).bfloat16()
    r = torch.randn(T, C, generator=g, device=DEV).bfloat16()
    w = torch.randn(C, generator=g, device=DEV).bfloat16()
    f = engine.rms_norm_fp8 if fp8 else engine.rms_norm
    out = f(x, w, residual=r)
    border = (2 ** 32 - 1) // 256 * (1 if C % 8 else 4)
    assert border < T
    for a, b in ((0, 9), (border - 9, border + 5), (T - 9, T)):
        part = f(x[a:b].contiguous(), w, residual=r[a:b].contiguous())
        for got, want in zip(out, part):
            got = got[a:b]
            if fp8 and got.dtype == torch.float8_e4m3fn:
                got, want = got.view(torch.uint8), want.view(torch.uint8)
            assert torch.equal(got, want)
    # and no row in between was left out
    s = x.float().add_(r.float())
    assert torch.equal(out[-1], s.bfloat16())
    assert not torch.isnan(out[0].float()).any()
    y = out[0].float() if not fp8 else out[0].float() * out[1]
    assert int((y.abs().amax(1) > 0).sum()) >= T - 10
