"""linear_int4 against its float64 form (tests/block_ref.py)."""
import pytest
import torch

from block_ref import int4_64, unpack_int4, within
from forge import engine, export

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _inputs(M, C, R, gs, bias=True, residual=True, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + M + C + R)
    words = torch.randint(-2 ** 31, 2 ** 31, (R, (C + 7) // 8), generator=g, device=DEV).to(torch.int32)
    scale = 0.01 * (0.1 + torch.rand(R, (C + gs - 1) // gs, generator=g, device=DEV))
    mk = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()   # noqa: E731
    rec = dict(weight_packed=words, weight_scale=scale, weight_shape=torch.tensor([R, C]))
    return mk(M, C), rec, mk(R) if bias else None, mk(M, R) if residual else None


def _check(x, rec, bias, act, residual, gs):
    y = engine.linear_int4(x, rec, bias=bias, activation=act, residual=residual, group_size=gs)
    want, bound = int4_64(x, rec["weight_packed"], rec["weight_scale"], gs, bias, act, residual)
    within(y, want, bound)
    return y


CASES = [
    # M, C, R, group
    (1, 1, 1, 1), (1, 8, 1, 8), (1, 128, 16, 128), (1, 2048, 7168, 128), (2, 7168, 256, 128), (3, 136, 40, 32),
    (16, 7168, 512, 128), (17, 2048, 1000, 64), (5, 100, 33, 128), (31, 1000, 70, 48), (32, 512, 100, 512),
    (33, 768, 2048, 32), (64, 1536, 96, 128), (65, 2048, 768, 128), (100, 264, 130, 128), (129, 4096, 300, 64),
    (256, 1024, 513, 256), (300, 2048, 768, 128), (513, 1504, 257, 32), (1000, 7168, 384, 128), (40, 7, 9, 128),
    (7, 320, 17, 64), (9, 8200, 24, 128), (260, 200, 131, 40), (1, 30000, 48, 128), (12, 640, 16, 96),
    (300, 1000, 70, 1000), (270, 672, 40, 96), (400, 104, 129, 32), (290, 72, 20, 128), (700, 2048, 130, 2048),
    (20, 1000, 70, 1000), (50, 72, 20, 128), (300, 320, 64, 64),
]


@pytest.mark.parametrize("M,C,R,gs", CASES)
def test_linear_int4(hip, M, C, R, gs):
    x, rec, bias, residual = _inputs(M, C, R, gs)
    _check(x, rec, None, None, None, gs)
    _check(x, rec, bias, "silu", residual, gs)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu", None])
@pytest.mark.parametrize("M", [1, 20, 300])
@pytest.mark.parametrize("bias,residual", [(True, False), (False, True)])
def test_epilogue(hip, act, M, bias, residual):
    x, rec, b, r = _inputs(M, 512, 144, 128, bias, residual)
    _check(x, rec, b, act, r, 128)


@pytest.mark.parametrize("M", [1, 16, 40, 300])
@pytest.mark.parametrize("C", [256, 1000])
def test_strides_and_alignment(hip, M, C):
    R = 72
    x, rec, bias, res = _inputs(M, C, R, 64 if C == 256 else 128)
    gs = 64 if C == 256 else 128
    want = _check(x, rec, bias, None, res, gs)
    for lead, pad in ((8, 8), (1, 2)):
        wide = torch.full((M, C + lead + pad), float("nan"), device=DEV).bfloat16()
        wide[:, lead:lead + C] = x
        wr = torch.full((M, R + lead + pad), float("nan"), device=DEV).bfloat16()
        wr[:, lead:lead + R] = res
        _check(wide[:, lead:lead + C], rec, bias, None, wr[:, lead:lead + R], gs)
    y = engine.linear_int4(x.t().contiguous().t(), rec, bias=bias, residual=res, group_size=gs)
    assert torch.equal(y, want)
    # packed words that start off the 16-byte grid
    buf = torch.zeros(R * rec["weight_packed"].shape[1] + 1, dtype=torch.int32, device=DEV)
    off = buf[1:].view(R, -1)
    off.copy_(rec["weight_packed"])
    _check(x, dict(rec, weight_packed=off), bias, None, res, gs)
    lead3 = engine.linear_int4(x.view(1, M, 1, C), rec, bias=bias, residual=res.view(1, M, 1, R), group_size=gs)
    assert lead3.shape == (1, M, 1, R) and torch.equal(lead3.view(M, R), want)


def test_empty_and_group_size_rules(hip):
    x, rec, bias, res = _inputs(4, 256, 24, 64)
    assert engine.linear_int4(x[:0], rec).shape == (0, 24)
    assert engine.linear_int4(x[0], rec).shape == (24,)
    assert torch.equal(engine.linear_int4(x, rec), engine.linear_int4(x, rec, group_size=64))


@pytest.mark.parametrize("M", [1, 16, 40, 300])
def test_special_values(hip, M):
    """an infinity or NaN of x reaches its own row and no other; columns behind C are never read"""
    C, R, gs = 384, 48, 128
    x, rec, _, _ = _inputs(M, C, R, gs)
    clean = engine.linear_int4(x, rec, group_size=gs)
    if M > 1:
        x2 = x.clone()
        x2[0, 5] = float("nan")
        y = engine.linear_int4(x2, rec, group_size=gs)
        assert torch.isnan(y[0]).all() and torch.equal(y[1:], clean[1:])
    x2 = x.clone()
    x2[-1, 200] = float("inf")
    y = engine.linear_int4(x2, rec, group_size=gs)
    q = unpack_int4(rec["weight_packed"], C)[:, 200]
    want = torch.where(q > 0, float("inf"), torch.where(q < 0, float("-inf"), float("nan"))).to(y.device)
    assert torch.equal(torch.isnan(y[-1]), torch.isnan(want))
    assert torch.equal(y[-1][q != 0].float(), want[q != 0].float())
    wide = torch.full((M, C + 64), float("nan"), device=DEV).bfloat16()
    wide[:, :C] = x
    assert torch.equal(engine.linear_int4(wide[:, :C], rec, group_size=gs), clean)


@pytest.mark.parametrize("sym", [True, False])
def test_follows_the_solve(hip, sym):
    """quantise a layer, pack it, and multiply by the packed words: the product with the layer's own
    dequantised weights (zero points inside the nibbles' range)"""
    from forge.gptq import GPTQ
    g = torch.Generator().manual_seed(2)
    R, C, n = 96, 384, 500
    layer = torch.nn.Linear(C, R, bias=False)
    layer.weight.data = 0.02 * torch.randn(R, C, generator=g)
    q = GPTQ(layer.to(DEV), bits=4, group_size=128, symmetric=sym, device=DEV)
    q.update(torch.randn(n, C, generator=g).to(DEV))
    codes, scales, zeros = q.quantize()
    rec = export.pack_weight(export.layer_record(codes, scales, zeros, 128, 4, (R, C)), 4, sym, 128)
    x = torch.randn(50, C, generator=g).bfloat16().to(DEV)
    y = engine.linear_int4(x, rec, group_size=128)
    want, bound = int4_64(x, rec["weight_packed"], rec["weight_scale"], 128, None, None, None)
    within(y, want, bound)
    shifted = (codes.double().view(R, 3, 128) - zeros.double().view(R, 3, 1))
    fits = ((shifted >= -8) & (shifted <= 7)).view(R, C).all(1)
    W = engine.dequantize_forge_full(torch.float32, codes, scales, zeros, 128, DEV).double()
    dense = x.double() @ W.T
    assert fits.any()
    assert ((dense - want).abs()[:, fits] <= 1e-6 * (x.double().abs() @ W.abs().T)[:, fits] + 1e-12).all()


def test_same_bits_every_time_and_in_a_graph(hip):
    for M in (1, 16, 40, 300):
        x, rec, bias, res = _inputs(M, 2048, 272, 128)
        f = lambda: engine.linear_int4(x, rec, bias=bias, activation="gelu", residual=res)   # noqa: E731,B023
        want = f()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            a = f()
        b = f()
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(want, a) and torch.equal(want, b)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f()
        keep = x.clone()
        for k in range(3):
            x.copy_(keep * (k + 1))
            graph.replay()
            torch.cuda.synchronize()
            got = out.clone()
            assert torch.equal(got, f())
            torch.randn(500, 500, device=DEV).sum().item()
