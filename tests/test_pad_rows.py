"""Padded copies of 16-bit matrices, and the shapes of the gated rows that need them."""
import ctypes

import pytest
import torch

from block_ref import gated64, within
from forge import engine

DEV = "cuda"


def test_refusals_at_the_c_entries():
    from forge.backend.hip import load_library
    lib, p = load_library(), ctypes.c_void_p(4096)
    pad = lambda src=p, ld=5, out=p, b=1, R=3, C=5, Rp=3, Cp=8: lib.forge_pad_rows(   # noqa: E731
        src, 0, ld, out, b, R, C, Rp, Cp, None, None)
    for bad, text in ((dict(Cp=7), "Cp=7"), (dict(Cp=0), "Cp=0"), (dict(Rp=2), "Rp=2"), (dict(R=-1), "R=-1"),
                      (dict(C=0), "C=0"), (dict(b=-1), "batch=-1"), (dict(b=65536), "too large"),
                      (dict(Rp=1 << 30), "too large"), (dict(ld=4), "pitch"), (dict(src=None), "null"),
                      (dict(out=None), "null"), (dict(out=ctypes.c_void_p(4104)), "aligned"),
                      (dict(src=ctypes.c_void_p(4097)), "aligned")):
        assert pad(**bad) != 0
        assert text in lib.forge_last_error().decode(), bad
    assert pad(b=0, src=None, out=None) == 0 and pad(R=0, Rp=0, src=None, out=None) == 0

    def gated(x=p, ldx=16, wg=p, ldw=16, ws=128, H=16, I=8):
        return lib.forge_gated_rows(x, ldx, p, wg, p, ldw, ws, 6, 2, H, I, 0, p, None, None, None)
    for bad in (dict(H=15), dict(I=7), dict(ldx=17), dict(ldw=20, ws=160), dict(ws=129), dict(x=ctypes.c_void_p(4098)),
                dict(wg=ctypes.c_void_p(4104))):
        assert gated(**bad) != 0
        assert "multiples of 8" in lib.forge_last_error().decode(), bad


@pytest.mark.gpu
@pytest.mark.parametrize("B,R,C,lead,pitch,Rp", [
    (1, 1, 1, 0, 1, 1), (1, 3, 5, 1, 7, 3), (2, 7, 8, 0, 8, 8), (3, 5, 9, 1, 9, 8), (2, 33, 513, 3, 517, 40),
    (1, 9, 64, 1, 67, 9), (1, 300, 1030, 2, 1031, 304), (4, 16, 24, 8, 48, 16), (1, 4, 16, 5, 17, 4)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_pad_rows(hip, B, R, C, lead, pitch, Rp, dtype):
    flat = torch.full((lead + B * R * pitch + 3,), float("nan"), dtype=dtype, device=DEV)
    t = flat[lead:lead + B * R * pitch].view(B, R, pitch)[:, :, :C]
    t.copy_(torch.randn(B, R, C, device=DEV))
    want = torch.zeros(B, Rp, -(-C // 8) * 8, dtype=dtype, device=DEV)
    want[:, :R, :C] = t
    assert torch.equal(hip.pad_rows(t, Rp), want)
    if Rp == R:
        assert torch.equal(hip.pad_rows(t[-1]), want[-1])


@pytest.mark.gpu
def test_matrices_without_rows_are_left(hip):
    t = torch.randn(4, 5, 9, device=DEV).bfloat16()
    offs = torch.tensor([0, 3, 3, 7, 7], dtype=torch.int32, device=DEV)
    out = torch.full((4, 8, 16), 7.0, device=DEV).bfloat16()
    rc = hip._lib.forge_pad_rows(t.data_ptr(), t.stride(0), t.stride(1), out.data_ptr(), 4, 5, 9, 8, 16,
                                 offs.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    for e in (0, 2):
        assert torch.equal(out[e, :5, :9], t[e]) and out[e, 5:].eq(0).all() and out[e, :, 9:].eq(0).all()
    assert out[1].eq(7).all() and out[3].eq(7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("H,I", [(33, 64), (64, 33), (33, 35)])
@pytest.mark.parametrize("counts", [(1, 0, 3), (300, 0, 41)])
def test_gated_rows_of_odd_sizes(hip, counts, H, I):
    """NaN in the weights of an expert without rows reaches nothing, and a captured call replays"""
    g = torch.Generator(device=DEV).manual_seed(H + I)
    mk = lambda s, *sh: (s * torch.randn(*sh, generator=g, device=DEV)).bfloat16()   # noqa: E731
    N, offs = sum(counts), [0, counts[0], counts[0], sum(counts)]
    rows, wg, wu, dh = mk(1.0, N, H), mk(H ** -0.5, 3, I, H), mk(H ** -0.5, 3, I, H), mk(1.0, N, I)
    wg[1], wu[1] = float("nan"), float("nan")
    leaves = [t.clone().requires_grad_(True) for t in (rows, wg, wu)]
    h = engine.expert_gated_rows(leaves[0], offs, leaves[1], leaves[2])
    grads = torch.autograd.grad(h, leaves, dh)
    z = [torch.nan_to_num(t) for t in (wg, wu)]
    (want, bound), wants = gated64(rows, offs, z[0], z[1], "silu", dh)
    within(h, want, bound)
    for got, like, (w, b) in zip(grads, leaves, wants):
        assert got.shape == like.shape
        within(got, w, b)
    o = torch.tensor(offs, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        hip.gated_rows(rows, o, wg, wu)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept, gate, up = hip.gated_rows(rows, o, wg, wu, "silu", keep=True)
        back = hip.gated_rows_backward(dh, gate, up, rows, o, wg, wu)
    for scale in (1.0, -0.5, 2.0):
        rows.copy_(leaves[0].detach() * scale)
        graph.replay()
        torch.cuda.synchronize()
        e, eg, eu = hip.gated_rows(rows, o, wg, wu, "silu", keep=True)
        assert torch.equal(kept, e)
        assert all(torch.equal(a, b) for a, b in zip(back, hip.gated_rows_backward(dh, eg, eu, rows, o, wg, wu)))


@pytest.mark.gpu
@pytest.mark.parametrize("counts,H,I", [([2100], 136, 72), ([4096, 0, 2300], 264, 40)])
def test_weight_gradients_of_experts_with_many_rows(hip, counts, H, I):
    g = torch.Generator(device=DEV).manual_seed(H)
    mk = lambda s, *sh: (s * torch.randn(*sh, generator=g, device=DEV)).bfloat16()   # noqa: E731
    offs = [0] + torch.tensor(counts).cumsum(0).tolist()
    N, E = offs[-1], len(counts)
    leaves = [t.requires_grad_(True) for t in (mk(1.0, N, H), mk(H ** -0.5, E, I, H), mk(H ** -0.5, E, I, H))]
    dh = mk(1.0, N, I)
    h = engine.expert_gated_rows(leaves[0], offs, leaves[1], leaves[2])
    grads = torch.autograd.grad(h, leaves, dh)
    (want, bound), wants = gated64(*[t.detach() for t in leaves[:1]], offs, *[t.detach() for t in leaves[1:]], "silu", dh)
    within(h.detach(), want, bound)
    for got, (w, b) in zip(grads, wants):
        within(got, w, b)


@pytest.mark.gpu
def test_weight_gradients_hand_their_tiles_out_once(hip):
    """more tiles than workgroups, experts of very different lengths: every tile is written, in every one of
    several passes and replays alike"""
    g = torch.Generator(device=DEV).manual_seed(5)
    counts = [900, 0, 3, 60, 0, 200, 1, 40] * 6
    offs = [0] + torch.tensor(counts).cumsum(0).tolist()
    N, E, H, I = offs[-1], len(counts), 520, 264
    mk = lambda s, *sh: (s * torch.randn(*sh, generator=g, device=DEV)).bfloat16()   # noqa: E731
    rows, wg, wu, dh = mk(1.0, N, H), mk(0.05, E, I, H), mk(0.05, E, I, H), mk(1.0, N, I)
    o = torch.tensor(offs, dtype=torch.int32, device=DEV)
    _, gate, up = hip.gated_rows(rows, o, wg, wu, "silu", keep=True)
    first = hip.gated_rows_backward(dh, gate, up, rows, o, wg, wu)
    _, wants = gated64(rows, offs, wg, wu, "silu", dh)
    for got, (w, b) in zip(first, wants):
        within(got, w, b)
    for need in ((False, True, False), (False, False, True)):
        part = hip.gated_rows_backward(dh, gate, up, rows, o, wg, wu, need=need)
        assert all(p is None or torch.equal(p, f) for p, f in zip(part, first))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = hip.gated_rows_backward(dh, gate, up, rows, o, wg, wu)
    for _ in range(3):
        for t in kept:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        again = hip.gated_rows_backward(dh, gate, up, rows, o, wg, wu)
        assert all(torch.equal(a, f) and torch.equal(b, f) for a, b, f in zip(kept, again, first))
    # no rows at all: nothing counts the tiles, all are zero
    zero = torch.zeros(E + 1, dtype=torch.int32, device=DEV)
    empty = hip.gated_rows_backward(dh[:0], gate[:0], up[:0], rows[:0], zero, wg, wu)
    assert all((t == 0).all() for t in empty[1:])


@pytest.mark.gpu
@pytest.mark.parametrize("per", [1, 9], ids=["few", "many"])
def test_more_experts_than_a_workgroup_has_threads(hip, per):
    """offsets of 1300 experts, most of them without rows"""
    g = torch.Generator(device=DEV).manual_seed(per)
    E, H, I = 1300, 48, 40
    counts = [0] * E
    for e in range(3, E, 13):
        counts[e] = per * (1 + e % 3)
    counts[700] = 130
    offs = [0] + torch.tensor(counts).cumsum(0).tolist()
    mk = lambda s, *sh: (s * torch.randn(*sh, generator=g, device=DEV)).bfloat16()   # noqa: E731
    rows, wg, wu, dh = mk(1.0, offs[-1] + 5, H), mk(0.15, E, I, H), mk(0.15, E, I, H), mk(1.0, offs[-1] + 5, I)
    leaves = [t.clone().requires_grad_(True) for t in (rows, wg, wu)]
    h = engine.expert_gated_rows(leaves[0], torch.tensor(offs, device=DEV), leaves[1], leaves[2])
    grads = torch.autograd.grad(h, leaves, dh)
    n = offs[-1]
    assert (h[n:] == 0).all() and (grads[0][n:] == 0).all()
    (want, bound), wants = gated64(rows[:n], offs, wg, wu, "silu", dh[:n])
    within(h[:n], want, bound)
    for got, (w, b) in zip((grads[0][:n], *grads[1:]), wants):
        within(got, w, b)


def test_pitch_of_rows():
    from forge.backend.hip import _pitch
    t = torch.zeros(4, 24)
    assert _pitch(t) == 24 and _pitch(t[:, 3:11]) == 24 and _pitch(t[::2]) == 48
    assert _pitch(t[:1].as_strided((1, 24), (3, 1))) == 24 and _pitch(t[:0]) == 24
    assert _pitch(torch.zeros(2, 4, 24)[:, :, :8]) == 24
    for bad in (t[:1].expand(4, 24), t.as_strided((4, 24), (23, 1)), torch.zeros(2, 1, 8).expand(2, 3, 8)):
        with pytest.raises(RuntimeError, match="overlap"):
            _pitch(bad)


def test_unit_rows():
    from forge.backend.hip import _pieces, _unit_rows
    t = torch.zeros(4, 24, dtype=torch.bfloat16)
    assert _unit_rows(t) is t and _unit_rows(t[:, 3:11]).data_ptr() == t[:, 3:11].data_ptr()
    for odd in (t.t(), t[:1].expand(4, 24), torch.zeros(1, 5).t(), torch.zeros(1, 5, 7).transpose(0, 2)[..., :1]):
        u = _unit_rows(odd)
        assert u.stride(-1) == 1 and u.is_contiguous() and torch.equal(u, odd)
    assert _pieces(t) and not _pieces(t[:, :23]) and not _pieces(t[:, 1:17]) and _pieces(t[:, 8:16])
    assert not _pieces(torch.zeros(4, 27, dtype=torch.bfloat16)[:, :8])


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 5])
def test_a_single_column_of_any_stride(hip, rows):
    mk = lambda *sh: torch.randn(*sh, device=DEV).bfloat16()   # noqa: E731
    x, w = mk(1, rows).t(), mk(3, 1, 1).transpose(1, 2)
    norm_w = mk(1)
    assert torch.equal(engine.rms_norm(x, norm_w), engine.rms_norm(x.clone(memory_format=torch.contiguous_format), norm_w))
    offs = [0, rows, rows, rows]
    assert torch.equal(engine.expert_gated_rows(x, offs, w, w),
                       engine.expert_gated_rows(x.clone(memory_format=torch.contiguous_format), offs, w, w))
    rec = dict(weight_packed=torch.full((8, 1), 0x7, dtype=torch.int32, device=DEV),
               weight_scale=torch.ones(8, 1, device=DEV), weight_shape=torch.tensor([8, 1]))
    assert torch.equal(engine.linear_int4(x, rec), (-x).expand(rows, 8))


@pytest.mark.gpu
def test_rows_over_each_other_are_refused_or_copied(hip):
    """the kernels' calls refuse them, the engine's copy them"""
    one = torch.randn(1, 64, device=DEV).bfloat16()
    rows, w = one.expand(9, 64), torch.randn(1, 40, 64, device=DEV).bfloat16()
    offs = torch.tensor([0, 9], dtype=torch.int32, device=DEV)
    norm_w = torch.ones(64, device=DEV).bfloat16()
    packed = torch.zeros(8, 8, dtype=torch.int32, device=DEV)
    scale = torch.ones(8, 1, device=DEV)
    dense = rows.contiguous()
    h, g, u = hip.gated_rows(dense, offs, w, w, "silu", keep=True)
    for call in (lambda: hip.rms_norm(rows, norm_w, 1e-6), lambda: hip.rms_norm(dense, norm_w, 1e-6, rows),
                 lambda: hip.rms_norm_fp8(rows, norm_w, 1e-6), lambda: hip.gated_rows(rows, offs, w, w),
                 lambda: hip.gated_rows_backward(h, g, u, rows, offs, w, w), lambda: hip.pad_rows(rows),
                 lambda: hip.gated_rows(dense, offs, *2 * (w[:, :1].expand(1, 40, 64),)),
                 lambda: hip.linear_int4(rows, packed, scale, 64),
                 lambda: hip.linear_int4(dense, packed, scale, 64, None, None, one[:, :8].expand(9, 8))):
        with pytest.raises(RuntimeError, match="overlap"):
            call()
    assert torch.equal(engine.expert_gated_rows(rows, [0, 9], w, w), h)
    assert torch.equal(engine.rms_norm(rows, norm_w), engine.rms_norm(dense, norm_w))


@pytest.mark.gpu
@pytest.mark.parametrize("I", [40, 41])
def test_the_result_is_a_tensor_of_its_own(hip, I):
    """dense and free to be changed in place, whatever its width"""
    g = torch.Generator(device=DEV).manual_seed(I)
    mk = lambda *sh: (0.3 * torch.randn(*sh, generator=g, device=DEV)).bfloat16()   # noqa: E731
    x, wg, wu = mk(10, 24), mk(2, I, 24), mk(2, I, 24)
    plain = engine.expert_gated_rows(x, [0, 4, 10], wg, wu)
    assert plain.is_contiguous() and plain.shape == (10, I)
    leaf = x.clone().requires_grad_(True)
    h = engine.expert_gated_rows(leaf, [0, 4, 10], wg, wu)
    assert h.is_contiguous() and torch.equal(h, plain)
    h.mul_(2)
    h.sum().backward()
    again = x.clone().requires_grad_(True)
    engine.expert_gated_rows(again, [0, 4, 10], wg, wu).backward(torch.full_like(plain, 2.0))
    assert torch.equal(leaf.grad, again.grad)
