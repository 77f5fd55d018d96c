"""Float64 forms of the operators around the solve (norm, gated rows and their gradients, packed
int4 product) and how far a correct f32 kernel with one rounding at the end can be from them.
Written from the formulas; runs on whatever device its inputs are on.

Error model: an f32 sum of n exact products is off by at most n * 2^-23 * sum |terms| whatever its
order (2^-24 per addition if each is rounded to nearest, twice that if the matrix instruction rounds
otherwise); a rounding to a type by half a step, torch.finfo(t).eps / 2 of the value; exp and the
reciprocal inside an activation by 2^-20 of its value."""
import math

import torch

U = 2.0 ** -23
ACT = 2.0 ** -20
# |act'| <= L1, |act''| <= L2 (silu' <= 1.1, silu'' <= 1/2; gelu' <= 1.13, gelu'' <= 0.8)
L1 = {"silu": 1.1, "gelu": 1.14, "relu": 1.0, None: 1.0}
L2 = {"silu": 0.51, "gelu": 0.9, "relu": 0.0, None: 0.0}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def act64(name, v):
    if name == "silu":
        return v / (1 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    if name == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    return v


def dact64(name, v):
    if name == "silu":
        p = 1 / (1 + torch.exp(-v))
        return p * (1 + v * (1 - p))
    if name == "gelu":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (v + 0.044715 * v ** 3))
        return 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * c * (1 + 3 * 0.044715 * v * v)
    if name == "relu":
        return (v > 0).to(v.dtype)
    return torch.ones_like(v)


def norm64(x, w, eps, residual=None):
    s = x.double() if residual is None else x.double() + residual.double()
    y = s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps) * w.double()
    return y, s


# f32 chain of the norm: the sum of squares is off by at most (longest chain + tree) * 2^-23, half of
# which reaches the root: chains of 128 terms at most at the tested sizes (32768 columns over 256 lanes)
NORM_F32 = (128 + 16) * U / 2 + 8 * U


def gated64(rows, offsets, wg, wu, act, dh=None):
    """-> (h, bound of h) and, with dh, [(dx, bound), (dwg, bound), (dwu, bound)]; offsets a list."""
    N, (E, I, H) = rows.shape[0], wg.shape
    z = lambda *s: torch.zeros(*s, dtype=torch.float64, device=rows.device)   # noqa: E731
    h, hb = z(N, I), z(N, I)
    dx, dxb = z(N, H), z(N, H)
    dw, dwb = [z(E, I, H), z(E, I, H)], [z(E, I, H), z(E, I, H)]
    r = half_step(torch.bfloat16)
    for e in range(E):
        a, b = offsets[e], offsets[e + 1]
        if a == b:
            continue
        x, G, Uw = rows[a:b].double(), wg[e].double(), wu[e].double()
        g, u = x @ G.T, x @ Uw.T
        eg, eu = H * U * (x.abs() @ G.abs().T), H * U * (x.abs() @ Uw.abs().T)
        ag = act64(act, g)
        h[a:b] = ag * u
        hb[a:b] = (L1[act] * eg * (u.abs() + eu) + ag.abs() * eu) * (1 + r) + (r + 4 * ACT) * (ag * u).abs()
        if dh is None:
            continue
        d = dh[a:b].double()
        dag = dact64(act, g)
        dg, du = d * u * dag, d * ag
        e_dag = L2[act] * eg + ACT * (1 + dag.abs())
        if act == "relu":                      # a sign of g that the f32 sum may take either way
            e_dag = e_dag + (g.abs() <= eg).double()
        edg = r * dg.abs() + (1 + r) * d.abs() * (eu * (dag.abs() + e_dag) + u.abs() * e_dag)
        edu = r * du.abs() + (1 + r) * d.abs() * (L1[act] * eg + ACT * ag.abs())
        v = dg @ G + du @ Uw
        dx[a:b] = v
        A = dg.abs() + edg
        B = du.abs() + edu
        dxb[a:b] = (edg @ G.abs() + edu @ Uw.abs() + 2 * I * U * (A @ G.abs() + B @ Uw.abs())) * (1 + r) + r * v.abs()
        for k, (t, et, m) in enumerate(((dg, edg, A), (du, edu, B))):
            v = t.T @ x
            dw[k][e] = v
            dwb[k][e] = (et.T @ x.abs() + (b - a) * U * (m.T @ x.abs())) * (1 + r) + r * v.abs()
    if dh is None:
        return h, hb
    return (h, hb), [(dx, dxb), (dw[0], dwb[0]), (dw[1], dwb[1])]


def unpack_int4(packed, C):
    """[R, words] int32 -> integers -8 .. 7 [R, C], lowest nibble first"""
    w = packed.to(torch.int64) & 0xFFFFFFFF
    q = torch.stack([(w >> (4 * k)) & 15 for k in range(8)], -1).reshape(packed.shape[0], -1)
    return q[:, :C] - 8


def int4_64(x, packed, scale, gs, bias, act, residual):
    C = x.shape[1]
    col = torch.arange(C, device=x.device) // gs
    W = unpack_int4(packed, C).double() * scale.double()[:, col]
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


# values under the type's smallest normal number are rounded to a step of its own
TINY = {torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -149}


def within(got, want, bound):
    """every element within its bound; the message says where it is worst"""
    tiny = TINY[got.dtype]
    got = got.double()
    assert got.shape == want.shape, (got.shape, want.shape)
    assert torch.isfinite(got).all(), "not finite"
    if not got.numel():
        return
    over = (got - want).abs() - bound - tiny
    worst = int(over.argmax())
    assert over.flatten()[worst] <= 0, (f"element {worst} of {tuple(got.shape)}: {got.flatten()[worst]} for "
                                        f"{want.flatten()[worst]}, allowed off by {bound.flatten()[worst]}")
