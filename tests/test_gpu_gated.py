"""expert_gated_rows and its gradients against their float64 forms (tests/block_ref.py)."""
import pytest
import torch

from block_ref import gated64, within
from forge import engine

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _inputs(counts, H, I, seed=0, lead=0, tail=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    E = len(counts)
    offs = [lead]
    for c in counts:
        offs.append(offs[-1] + c)
    N = offs[-1] + tail
    mk = lambda s, *sh: (s * torch.randn(*sh, generator=g, device=DEV)).bfloat16()   # noqa: E731
    return mk(1.0, N, H), offs, mk(H ** -0.5, E, I, H), mk(H ** -0.5, E, I, H), mk(1.0, N, I)


def _run(rows, offs, wg, wu, dh, act):
    rows, wg, wu = (t.detach().requires_grad_(True) for t in (rows, wg, wu))
    h = engine.expert_gated_rows(rows, offs, wg, wu, activation=act)
    return h.detach(), torch.autograd.grad(h, (rows, wg, wu), dh)


def _check(rows, offs, wg, wu, dh, act):
    h, grads = _run(rows, offs, wg, wu, dh, act)
    (want, bound), wants = gated64(rows, offs, wg, wu, act, dh)
    within(h, want, bound)
    for got, (w, b) in zip(grads, wants):
        within(got, w, b)
    with torch.no_grad():
        assert torch.equal(engine.expert_gated_rows(rows, offs, wg, wu, activation=act), h)
    return h, grads


CASES = [
    # rows per expert, H, I
    ([1], 8, 8), ([1], 1, 1), ([3], 7, 5), ([64], 64, 64), ([65], 72, 136), ([0], 16, 16),
    ([0, 0, 5, 0], 40, 24), ([1, 0, 2, 31, 32, 33], 128, 128), ([300, 1, 0, 129], 256, 192),
    ([257, 255, 256], 320, 128), ([5, 70], 130, 258), ([13, 600], 2048, 768), ([40], 104, 1000),
    ([2] * 70, 64, 32), ([0] * 100 + [9] + [0] * 29 + [600], 136, 72), ([1000], 136, 24), ([37, 0, 65], 513, 127),
]


@pytest.mark.parametrize("counts,H,I", CASES, ids=[f"{sum(c)}rows-{len(c)}experts-{h}x{i}" for c, h, i in CASES])
def test_gated_rows_and_gradients(hip, counts, H, I):
    _check(*_inputs(counts, H, I, seed=H + I), "silu")


@pytest.mark.parametrize("act", ["gelu", "relu", None])
@pytest.mark.parametrize("H", [96, 97])
def test_activations(hip, act, H):
    _check(*_inputs([50, 0, 90], H, 80, seed=3), act)


@pytest.mark.parametrize("H,I", [(64, 48), (2048, 256)])
def test_rows_of_no_expert(hip, H, I):
    """rows before the first offset and behind the last get 0, and nothing they hold reaches a
    gradient: NaN there (rows and dh) changes nothing"""
    rows, offs, wg, wu, dh = _inputs([30, 0, 290], H, I, lead=70, tail=300)
    live = torch.zeros(rows.shape[0], dtype=torch.bool, device=DEV)
    live[offs[0]:offs[-1]] = True
    rows[~live] = float("nan")
    dh[~live] = float("nan")
    h, (dx, dwg, dwu) = _run(rows, offs, wg, wu, dh, "silu")
    assert (h[~live] == 0).all() and (dx[~live] == 0).all()
    o2 = [o - offs[0] for o in offs]
    (want, bound), wants = gated64(rows[live], o2, wg, wu, "silu", dh[live])
    within(h[live], want, bound)
    for got, (w, b) in zip((dx[live], dwg, dwu), wants):
        within(got, w, b)
    assert (dwg[1] == 0).all() and (dwu[1] == 0).all()


@pytest.mark.parametrize("H,I", [(64, 40), (1024, 256)])
def test_a_nan_stays_in_its_row_and_expert(hip, H, I):
    rows, offs, wg, wu, dh = _inputs([33, 40, 50], H, I)
    rows[35, 3] = float("nan")
    rows[100, 5] = float("inf")
    h, (dx, dwg, dwu) = _run(rows, offs, wg, wu, dh, "silu")
    bad = torch.zeros(rows.shape[0], dtype=torch.bool, device=DEV)
    bad[35] = bad[100] = True
    assert torch.isnan(h[35]).all() and torch.isfinite(h[~bad]).all() and torch.isfinite(dx[~bad]).all()
    assert torch.isfinite(dwg[0]).all() and torch.isfinite(dwu[0]).all()
    assert torch.isnan(dwg[1]).any() and not torch.isfinite(dwu[2]).all()


def test_offsets_in_every_form(hip):
    rows, offs, wg, wu, _ = _inputs([30, 0, 41], 128, 64)
    want = engine.expert_gated_rows(rows, offs, wg, wu)
    for o in (torch.tensor(offs), torch.tensor(offs, device=DEV), torch.tensor(offs, dtype=torch.int32, device=DEV),
              torch.tensor([x for v in offs for x in (v, 7)], dtype=torch.int32, device=DEV)[::2], tuple(offs)):
        assert torch.equal(engine.expert_gated_rows(rows, o, wg, wu), want)
    dense = engine.expert_gated_rows(rows, None, wg[0], wu[0])
    assert torch.equal(dense, engine.expert_gated_rows(rows, [0, 71], wg[:1], wu[:1]))
    # on the device nothing looks at them: out of range or descending stays in bounds
    for bad in ([0, 500, 71, 90], [-5, 3, 2, 71], [71, 71, 0, 0]):
        o = torch.tensor(bad, dtype=torch.int32, device=DEV)
        out, g, u = hip.gated_rows(rows, o, wg, wu, "silu", keep=True)
        hip.gated_rows_backward(out, torch.zeros_like(g), torch.zeros_like(u), rows, o, wg, wu, "silu")
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="int32 or int64"):
        engine.expert_gated_rows(rows, torch.zeros(3, device=DEV, dtype=torch.int32), wg, wu)


@pytest.mark.parametrize("H", [96, 256])
def test_strides(hip, H):
    """rows of a wider tensor; weights that are a slice of a fused [E, 2I, H + pad] tensor; transposed
    weights and an expanded gradient are copied"""
    counts, I = [20, 0, 77], 64
    rows, offs, wg, wu, dh = _inputs(counts, H, I)
    wide = torch.full((rows.shape[0], H + 24), float("nan"), device=DEV).bfloat16()
    wide[:, 8:8 + H] = rows
    fused = torch.full((3, 2 * I + 3, H + 16), float("nan"), device=DEV).bfloat16()
    fused[:, :I, :H], fused[:, I:2 * I, :H] = wg, wu
    want, grads = _run(rows, offs, wg, wu, dh, "silu")
    r, g, u = wide[:, 8:8 + H], fused[:, :I, :H], fused[:, I:2 * I, :H]
    got, grads2 = _run(r, offs, g, u, dh, "silu")
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(grads, grads2))
    odd = torch.full((rows.shape[0], H + 3), float("nan"), device=DEV).bfloat16()     # off the 16-byte grid
    odd[:, 1:1 + H] = rows
    got, grads3 = _run(odd[:, 1:1 + H], offs, wg, wu, dh, "silu")
    (w64, b64), wants = gated64(rows, offs, wg, wu, "silu", dh)
    within(got, w64, b64)
    for a, (w, b) in zip(grads3, wants):
        within(a, w, b)
    t = wg.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(engine.expert_gated_rows(rows, offs, t, wu), want)
    one = torch.ones(1, 1, device=DEV).bfloat16().expand(rows.shape[0], I)
    a = _run(rows, offs, wg, wu, one, "silu")[1]
    b = _run(rows, offs, wg, wu, one.contiguous(), "silu")[1]
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_only_the_gradients_asked_for(hip):
    rows, offs, wg, wu, dh = _inputs([20, 50], 128, 64)
    full = _run(rows, offs, wg, wu, dh, "silu")[1]
    for i in range(3):
        t = [rows.clone(), wg.clone(), wu.clone()]
        t[i].requires_grad_(True)
        h = engine.expert_gated_rows(t[0], offs, t[1], t[2])
        h.backward(dh)
        assert torch.equal(t[i].grad, full[i])
        assert all(x.grad is None for j, x in enumerate(t) if j != i)
    # no rows at all: zero weight gradients
    e = _run(rows[:0], [0, 0, 0], wg, wu, dh[:0], "silu")
    assert e[0].shape == (0, 64) and e[1][0].shape == (0, 128)
    assert (e[1][1] == 0).all() and (e[1][2] == 0).all()


def test_gradients_against_differences(hip):
    """central differences of a float64 loss along random directions, taken on the float64 form;
    the kernel's gradient along the same direction within what its elements may be off"""
    rows, offs, wg, wu, dh = _inputs([40, 0, 25], 96, 64, seed=9)
    _, grads = _run(rows, offs, wg, wu, dh, "silu")
    (_, _), wants = gated64(rows, offs, wg, wu, "silu", dh)
    g = torch.Generator(device=DEV).manual_seed(1)

    def loss(x, a, b):
        return (gated64(x, offs, a, b, "silu")[0] * dh.double()).sum()

    base = [t.double() for t in (rows, wg, wu)]
    for k in range(3):
        d = torch.randn(base[k].shape, generator=g, device=DEV, dtype=torch.float64)
        eps = 1e-5
        up = loss(*[t + eps * d if j == k else t for j, t in enumerate(base)])
        dn = loss(*[t - eps * d if j == k else t for j, t in enumerate(base)])
        num = ((up - dn) / (2 * eps)).item()
        got = (grads[k].double() * d).sum().item()
        allowed = (wants[k][1] * d.abs()).sum().item() + 1e-6 * abs(num) + 1e-6
        assert abs(got - num) <= allowed, (k, got, num, allowed)


def test_same_bits_every_time_and_beside_other_work(hip):
    """two calls, two streams at once, and a replayed graph give the same bits"""
    rows, offs, wg, wu, dh = _inputs([300, 0, 33, 511], 512, 256, seed=4)
    o = torch.tensor(offs, dtype=torch.int32, device=DEV)

    def step():
        h, g, u = hip.gated_rows(rows, o, wg, wu, "silu", keep=True)
        return (h, *hip.gated_rows_backward(dh, g, u, rows, o, wg, wu, "silu"))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = step()
    b = step()
    torch.cuda.current_stream().wait_stream(side)
    for x, y, z in zip(want, a, b):
        assert torch.equal(x, y) and torch.equal(x, z)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    first = (rows.clone(), dh.clone(), o.clone())
    for k in range(3):
        if k:
            rows.copy_(first[0].flip(0)), dh.copy_(first[1] * k), o.copy_(first[2].clamp_max(400 * k))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for x, y in zip(step(), got):
            assert torch.equal(x, y)
        torch.randn(1000, 1000, device=DEV).sum().item()
