"""What the operators around the solve refuse, before anything reaches a GPU: in Python (shapes,
types, missing gradients) and at the C entry points."""
import ctypes

import pytest
import torch

from forge import engine


def _bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("fn", [engine.rms_norm, engine.rms_norm_fp8])
def test_norm_refusals(fn):
    x, w = _bf(4, 16), _bf(16)
    with pytest.raises(ValueError, match="expected float32 or bfloat16"):
        fn(x.half(), w)
    with pytest.raises(ValueError, match="weight is"):
        fn(x, w.half())
    with pytest.raises(ValueError, match="does not fit"):
        fn(x, _bf(15))
    with pytest.raises(ValueError, match="does not fit"):
        fn(_bf(4, 0), _bf(0))
    with pytest.raises(ValueError, match="residual"):
        fn(x, w, residual=_bf(4, 15))
    with pytest.raises(ValueError, match="residual"):
        fn(x, w, residual=torch.zeros(4, 16))
    with pytest.raises(ValueError, match="eps"):
        fn(x, w, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        fn(x, w, eps=float("nan"))
    with pytest.raises(RuntimeError, match="no backward pass"):
        fn(x.requires_grad_(True), w)


def test_gated_refusals():
    rows, wg = _bf(6, 16), _bf(2, 8, 16)
    f = engine.expert_gated_rows
    with pytest.raises(ValueError, match="unknown activation"):
        f(rows, [0, 3, 6], wg, wg, activation="tanh")
    with pytest.raises(ValueError, match="rows is"):
        f(rows.float(), [0, 3, 6], wg, wg)
    with pytest.raises(ValueError, match="w_up is"):
        f(rows, [0, 3, 6], wg, wg.float())
    with pytest.raises(ValueError, match="w_gate"):
        f(rows, [0, 3, 6], wg, _bf(2, 9, 16))
    with pytest.raises(ValueError, match="do not fit"):
        f(_bf(6, 15), [0, 3, 6], wg, wg)
    with pytest.raises(ValueError, match="need offsets"):
        f(rows, None, wg, wg)
    with pytest.raises(ValueError, match="empty weights"):
        f(rows, [0], _bf(0, 8, 16), _bf(0, 8, 16))
    for bad in ([0, 3], [0, 3, 7], [0, 4, 3], [-1, 3, 6], torch.tensor([0, 3, 7])):
        with pytest.raises(ValueError, match="ascending"):
            f(rows, bad, wg, wg)


def test_int4_refusals():
    rec = dict(weight_packed=torch.zeros(5, 8, dtype=torch.int32), weight_scale=torch.ones(5, 2),
               weight_shape=torch.tensor([5, 64]))
    x = _bf(3, 64)
    f = engine.linear_int4
    with pytest.raises(ValueError, match="unknown activation"):
        f(x, rec, activation="tanh")
    with pytest.raises(ValueError, match="x is"):
        f(x.float(), rec)
    with pytest.raises(ValueError, match="does not fit"):
        f(_bf(3, 63), rec)
    with pytest.raises(ValueError, match="weight_packed"):
        f(x, dict(rec, weight_packed=torch.zeros(5, 7, dtype=torch.int32)))
    with pytest.raises(ValueError, match="weight_scale"):
        f(x, dict(rec, weight_scale=torch.ones(4, 2)))
    with pytest.raises(ValueError, match="pass group_size"):
        f(x, dict(rec, weight_scale=torch.ones(5, 3)))
    with pytest.raises(ValueError, match="does not give"):
        f(x, rec, group_size=64)
    with pytest.raises(ValueError, match="bias"):
        f(x, rec, bias=_bf(4))
    with pytest.raises(ValueError, match="residual"):
        f(x, rec, residual=_bf(3, 4))
    with pytest.raises(RuntimeError, match="no backward pass"):
        f(x.requires_grad_(True), rec)


def test_c_entry_points_reject_before_a_launch():
    from forge.backend.hip import load_library
    lib = load_library()
    err = lib.forge_last_error
    P = ctypes.c_void_p(4096)          # never dereferenced: every call below is refused or empty
    assert lib.forge_rms_norm(P, 7, 8, None, 0, P, 1, 4, 8, 1e-6, P, None, None) == 1 and b"dtype=7" in err()
    assert lib.forge_rms_norm(P, 1, 7, None, 0, P, 1, 4, 8, 1e-6, P, None, None) == 1 and b"row pitch" in err()
    assert lib.forge_rms_norm(P, 1, 8, P, 8, P, 1, 4, 8, 1e-6, P, None, None) == 1 and b"go together" in err()
    assert lib.forge_rms_norm(P, 1, 8, None, 0, P, 1, 4, 8, float("nan"), P, None, None) == 1 and b"eps" in err()
    assert lib.forge_rms_norm(None, 1, 8, None, 0, P, 1, 4, 8, 1e-6, P, None, None) == 1 and b"null" in err()
    assert lib.forge_rms_norm_fp8(P, 1, 8, None, 0, P, 1, 4, 8, 1e-6, P, None, None, None) == 1 and b"null" in err()
    assert lib.forge_rms_norm(None, 1, 8, None, 0, None, 1, 0, 8, 1e-6, None, None, None) == 0    # no rows
    big = 1 << 31
    assert lib.forge_rms_norm(P, 1, 8, None, 0, P, 1, big, 8, 1e-6, P, None, None) == 1 and b"2^31" in err()

    def gated(ldx=16, off=P, ldw=16, ws=128, N=6, E=2, H=16, I=8, act=1, h=P, g=None, u=None):
        return lib.forge_gated_rows(P, ldx, off, P, P, ldw, ws, N, E, H, I, act, h, g, u, None)

    assert gated(off=None) == 1 and b"null" in err()
    assert gated(h=None) == 1 and b"null" in err()
    assert gated(ldx=15) == 1 and b"row pitch" in err()
    assert gated(ws=127) == 1 and b"expert stride" in err()
    assert gated(act=4) == 1 and b"act=4" in err()
    assert gated(E=0) == 1 and gated(E=70000) == 1 and b"too large" in err()
    assert gated(N=big) == 1 and b"too large" in err()
    assert gated(g=P) == 1 and b"go together" in err()
    assert gated(N=0) == 0
    need = lib.forge_gated_rows_backward_workspace_bytes(6, 8)
    assert need >= 2 * 6 * 8 * 2 and lib.forge_gated_rows_backward_workspace_bytes(0, 8) == 0

    def backward(ws=P, nbytes=need, dh=P):
        return lib.forge_gated_rows_backward(dh, P, P, P, 16, P, P, P, 16, 128, 6, 2, 16, 8, 1, P, P, P, ws,
                                             nbytes, None)

    assert backward(dh=None) == 1 and b"null" in err()
    assert backward(ws=None) == 1 and b"null" in err()
    assert backward(nbytes=need - 1) == 1 and b"workspace" in err()
    assert backward(ws=ctypes.c_void_p(4104)) == 1 and b"aligned" in err()

    def int4(x=P, ldx=64, gs=32, res=None, ldr=0, M=3, C=64, R=5, act=0):
        return lib.forge_linear_int4(x, ldx, P, P, gs, None, res, ldr, M, C, R, act, P, None)

    assert int4(x=None) == 1 and b"null" in err()
    assert int4(ldx=63) == 1 and b"row pitch" in err()
    assert int4(res=P, ldr=4) == 1 and b"row pitch" in err()
    assert int4(gs=0) == 1 and int4(act=-1) == 1 and int4(R=0) == 1
    assert int4(C=1 << 25, ldx=1 << 25) == 1 and b"too large" in err()
    assert int4(M=0) == 0
