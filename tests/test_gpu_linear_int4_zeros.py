"""linear_int4 on records with zero points (asymmetric grids), all rows against the layer's own weights
(code - zero) * scale in float64; and the many-row tiles on symmetric records."""
import pytest
import torch

from block_ref import ACT, L1, U, act64, half_step, int4_64, within
from forge import engine, export

DEV = "cuda"


def weights_64(x, codes, zero, scale, gs, bias=None, act=None, residual=None):
    """The product with (code - zero) * scale, and how far f32 sums rounded once may be from it (the error
    model of block_ref.py: C exact products, a group's sum times its scale, G groups, the epilogue)."""
    R, C = codes.shape
    col = torch.arange(C, device=x.device) // gs
    W = (codes.double() - zero.double()[:, col]) * scale.double()[:, col]
    xd = x.double()
    v = xd @ W.T
    e = (C + 2 * scale.shape[1] + 8) * U * (xd.abs() @ W.abs().T)
    if bias is not None:
        v = v + bias.double()
        e = e + U * v.abs()
    y = act64(act, v)
    e = L1[act] * e + (ACT if act else 0) * y.abs()
    if residual is not None:
        y = y + residual.double()
        e = e + U * y.abs()
    r = half_step(torch.bfloat16)
    return y, e * (1 + r) + r * y.abs()


def record(R, C, gs, zeros, seed, zero_dtype=torch.int32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    G = -(-C // gs)
    codes = torch.randint(0, 16, (R, C), generator=g, device=DEV, dtype=torch.uint8)
    scale = 0.01 * (0.1 + torch.rand(R, G, generator=g, device=DEV))
    if zeros == "each":
        zero = torch.randint(0, 16, (R, G), generator=g, device=DEV)
    else:
        zero = torch.full((R, G), zeros, device=DEV)
    zero = zero.to(zero_dtype)
    rec = export.pack_weight({"qweight": codes, "scale": scale, "zero": zero}, 4, False, gs)
    return codes, zero, scale, rec


def _mk(seed, *s):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*s, generator=g, device=DEV).bfloat16()


CASES = [
    # M, C, R, group: few rows of x
    (1, 2048, 1024, 128), (1, 320, 17, 64), (16, 7168, 512, 128), (5, 544, 33, 32), (3, 100, 16, 256), (16, 8, 1, 8),
    # 32 rows of x, 64 rows of x per workgroup
    (40, 2048, 768, 128), (33, 1504, 257, 32), (100, 264, 130, 64), (70, 90, 70, 128), (256, 1024, 513, 256),
    (300, 4096, 2048, 128), (290, 1216, 2048, 64), (513, 1504, 2057, 32), (300, 96, 2048, 96),
    # the many-row tiles
    (3201, 512, 1000, 128), (1700, 1472, 2048, 64), (1700, 1440, 2050, 32), (3201, 72, 1000, 128), (3300, 136, 1000, 8192),
    (3201, 672, 1000, 96), (1700, 128, 2048, 128),
    # groups that are not multiples of 32 columns
    (1, 100, 33, 40), (40, 1000, 70, 48), (300, 96, 70, 3), (9, 33, 20, 33),
]


@pytest.mark.gpu
@pytest.mark.parametrize("M,C,R,gs", CASES)
def test_all_rows_with_zero_points(hip, M, C, R, gs):
    codes, zero, scale, rec = record(R, C, gs, "each", M + C + R)
    x, bias, residual = _mk(1, M, C), _mk(2, R), _mk(3, M, R)
    y = engine.linear_int4(x, rec, group_size=gs)
    within(y, *weights_64(x, codes, zero, scale, gs))
    y = engine.linear_int4(x, rec, bias=bias, activation="silu", residual=residual, group_size=gs)
    within(y, *weights_64(x, codes, zero, scale, gs, bias, "silu", residual))


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", [0, 1, 5, 7, 8, 12, 15, -3, 20])
@pytest.mark.parametrize("M,R,gs", [(1, 100, 128), (40, 100, 64), (300, 2048, 32), (3201, 1000, 128), (20, 70, 24)])
def test_every_zero_point(hip, zeros, M, R, gs):
    C = 384
    codes, zero, scale, rec = record(R, C, gs, zeros, zeros + M + 9)
    x = _mk(4, M, C)
    y = engine.linear_int4(x, rec, group_size=gs)
    within(y, *weights_64(x, codes, zero, scale, gs))
    if zeros == 8:                                   # the symmetric record of the same codes
        plain = {k: v for k, v in rec.items() if k != "weight_zero_point"}
        assert torch.equal(y, engine.linear_int4(x, plain, group_size=gs))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.int8, torch.uint8, torch.int64])
def test_types_and_strides_of_the_zero_points(hip, dtype):
    codes, zero, scale, rec = record(48, 256, 64, "each", 3, dtype)
    x = _mk(5, 10, 256)
    want = engine.linear_int4(x, rec, group_size=64)
    within(want, *weights_64(x, codes, zero, scale, 64))
    wide = zero.repeat_interleave(2, 1)[:, ::2]
    assert not wide.is_contiguous()
    assert torch.equal(engine.linear_int4(x, dict(rec, weight_zero_point=wide), group_size=64), want)
    odd = torch.zeros(10, 259, device=DEV).bfloat16()
    odd[:, 1:257] = x                                # rows off the 16-byte grid
    assert torch.equal(engine.linear_int4(odd[:, 1:257], rec, group_size=64), want)


@pytest.mark.gpu
@pytest.mark.parametrize("sym", [True, False])
@pytest.mark.parametrize("gs", [128, 64, 32])
def test_the_product_is_the_solved_layers(hip, sym, gs):
    """quantise, pack and multiply: all rows against the weights that are written back into the layer"""
    from forge.gptq import GPTQ
    g = torch.Generator().manual_seed(7)
    R, C = 1000, 384
    layer = torch.nn.Linear(C, R, bias=False)
    layer.weight.data = 0.02 * torch.randn(R, C, generator=g) + (0 if sym else 0.01)
    q = GPTQ(layer.to(DEV), bits=4, group_size=gs, symmetric=sym, device=DEV)
    q.update(torch.randn(500, C, generator=g).to(DEV))
    codes, scales, zeros = q.quantize()
    rec = export.pack_weight(export.layer_record(codes, scales, zeros, gs, 4, (R, C)), 4, sym, gs)
    W = engine.dequantize_forge_full(torch.float32, codes, scales, zeros, gs, DEV).double()
    if not sym:
        assert zeros.unique().numel() > 1
    for M in (1, 40, 300, 3201):
        x = torch.randn(M, C, generator=g).bfloat16().to(DEV)
        want, bound = weights_64(x, codes, zeros.view(R, -1), scales.view(R, -1), gs)
        y = engine.linear_int4(x, rec, group_size=gs)
        within(y, want, bound)
        # the written-back weights are rounded to f32 once more
        within(y, x.double() @ W.T, bound + U * (x.double().abs() @ W.abs().T))


@pytest.mark.gpu
@pytest.mark.parametrize("M,C,R,gs", [(3201, 512, 1000, 128), (1700, 1472, 2048, 64), (1700, 1440, 2050, 32),
                                      (3201, 72, 1000, 128), (3300, 136, 1000, 8192), (3201, 672, 1000, 96),
                                      (1700, 128, 2048, 128), (3265, 2048, 1001, 128)])
def test_many_rows_of_x_without_zero_points(hip, M, C, R, gs):
    g = torch.Generator(device=DEV).manual_seed(M + C + R)
    words = torch.randint(-2 ** 31, 2 ** 31, (R, (C + 7) // 8), generator=g, device=DEV).to(torch.int32)
    scale = 0.01 * (0.1 + torch.rand(R, -(-C // gs), generator=g, device=DEV))
    rec = dict(weight_packed=words, weight_scale=scale, weight_shape=torch.tensor([R, C]))
    x, bias, residual = _mk(1, M, C), _mk(2, R), _mk(3, M, R)
    y = engine.linear_int4(x, rec, bias=bias, activation="gelu", residual=residual, group_size=gs)
    within(y, *int4_64(x, words, scale, gs, bias, "gelu", residual))


@pytest.mark.gpu
def test_zero_points_in_a_graph(hip):
    for M, R in ((1, 272), (40, 272), (300, 2048), (3201, 1000)):
        codes, zero, scale, rec = record(R, 512, 128, "each", M)
        x, bias, residual = _mk(1, M, 512), _mk(2, R), _mk(3, M, R)
        f = lambda: engine.linear_int4(x, rec, bias=bias, activation="relu", residual=residual)   # noqa: E731,B023
        want = f()
        assert torch.equal(want, f())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f()
        keep = x.clone()
        for k in range(3):
            x.copy_(keep * (k + 1))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, f())
            torch.randn(500, 500, device=DEV).sum().item()


def test_refusals():
    rec = dict(weight_packed=torch.zeros(5, 8, dtype=torch.int32), weight_scale=torch.ones(5, 2),
               weight_shape=torch.tensor([5, 64]), weight_zero_point=torch.zeros(5, 2, dtype=torch.int32))
    x = torch.zeros(3, 64, dtype=torch.bfloat16)
    for dt in (torch.float32, torch.bfloat16, torch.bool):
        with pytest.raises(ValueError, match="weight_zero_point is"):
            engine.linear_int4(x, dict(rec, weight_zero_point=torch.zeros(5, 2, dtype=dt)))
    for shape in ((5, 1), (10,), (4, 2)):
        with pytest.raises(ValueError, match="weight_zero_point"):
            engine.linear_int4(x, dict(rec, weight_zero_point=torch.zeros(*shape, dtype=torch.int32)))


def test_refusals_at_the_c_entry():
    import ctypes
    from forge.backend.hip import load_library
    lib, P = load_library(), ctypes.c_void_p(4096)     # never dereferenced

    def call(x=P, zero=P, ldx=64, gs=32, res=None, ldr=0, M=3, C=64, R=5, act=0):
        return lib.forge_linear_int4_zeros(x, ldx, P, P, zero, gs, None, res, ldr, M, C, R, act, P, None)

    err = lib.forge_last_error
    assert call(x=None) == 1 and b"null" in err()
    assert call(zero=None) == 1 and b"forge_linear_int4_zeros: null" in err()
    assert call(ldx=63) == 1 and b"row pitch" in err()
    assert call(res=P, ldr=4) == 1 and b"row pitch" in err()
    assert call(gs=0) == 1 and call(act=-1) == 1 and call(R=0) == 1
    assert call(C=1 << 25, ldx=1 << 25) == 1 and b"too large" in err()
    assert call(M=0, x=None, zero=None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M,C,R,gs", [(300_100, 7168, 24, 128), (300_100, 7168, 10, 56), (70_000, 64, 32_000, 32)])
def test_behind_two_to_the_31st_element(hip, M, C, R, gs, zeros):
    """of x, or of the residual and y: the last rows against the same rows alone in float64, the first ones too"""
    k = 70
    codes, zero, scale, rec = record(R, C, gs, "each" if zeros else 8, 5)
    if not zeros:
        del rec["weight_zero_point"]
    x = torch.zeros(M, C, dtype=torch.bfloat16, device=DEV)
    x[:k], x[-k:] = _mk(1, k, C), _mk(2, k, C)
    res = torch.zeros(M, R, dtype=torch.bfloat16, device=DEV)
    res[-k:] = _mk(3, k, R)
    y = engine.linear_int4(x, rec, residual=res, group_size=gs)
    within(y[:k], *weights_64(x[:k], codes, zero, scale, gs, residual=res[:k]))
    within(y[-k:], *weights_64(x[-k:], codes, zero, scale, gs, residual=res[-k:]))
    assert not y[k:-k].any()
