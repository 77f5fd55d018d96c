"""What is measured of the operators around the solve: the root-mean-square norm with the residual's
addition (plain and with 8-bit output), the experts' gated feed-forward rows with their gradients, and
the product with packed int4 weights and its epilogue.

``own`` false: the operators in elementary torch operations, in float32.  ``own`` true: the
framework's entry points (``forge.engine``).  Sizes are those of the Qwen3-style and DeepSeek-V3-style
layers of ``forge.synth`` (2048 x 768, 128 experts; 7168 x 2048, top-8 routing with Zipf popularity),
and generic odd ones.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
EPS = 1e-6
FP8_MAX = 448.0          # largest e4m3 value
FP8_GROUP = 128          # columns that share an 8-bit scale


def _engine():
    pkg = str(Path(__file__).resolve().parents[1] / "4bit-forge_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from forge import engine
    return engine


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one token's hidden state, as in decoding: latency
        dict(name="norm-token", op="norm", T=1, C=7168, dtype="bf16", residual=True),
        # the calibration tokens of one DeepSeek-V3-style layer
        dict(name="norm-rows", op="norm", T=8192, C=7168, dtype="bf16", residual=True),
        # a ragged prompt, 8-bit rows for an fp8 product
        dict(name="norm-fp8", op="norm_fp8", T=4099, C=2048, dtype="bf16", residual=True),
        # one token routed to 8 of a GPU's 32 experts: the weights of 8 experts stream through
        dict(name="gated-token", op="gated", tokens=1, topk=8, E=32, H=7168, I=2048, train=False),
        # the Qwen3-style layer's calibration pass
        dict(name="gated-qwen3", op="gated", tokens=4096, topk=8, E=128, H=2048, I=768, train=False),
        # a GPU's share of the DeepSeek-V3-style layer: 16 experts
        dict(name="gated-deepseek", op="gated", tokens=2048, topk=8, E=16, H=7168, I=2048, train=False),
        # gradients of a small odd batch
        dict(name="train-small", op="gated", tokens=129, topk=2, E=8, H=2048, I=768, train=True),
        # gradients at the DeepSeek-V3-style sizes
        dict(name="train-deepseek", op="gated", tokens=1021, topk=8, E=16, H=7168, I=2048, train=True),
        # one token through a packed down projection, residual added: latency
        dict(name="int4-token", op="int4", M=1, C=2048, R=7168, gs=128, bias=False, act="none", residual=True),
        # a decoding batch through packed gate and up rows
        dict(name="int4-batch", op="int4", M=16, C=7168, R=4096, gs=128, bias=False, act="none", residual=False),
        # a few odd rows, bias and activation, groups of 64
        dict(name="int4-odd", op="int4", M=77, C=2048, R=1000, gs=64, bias=True, act="silu", residual=False),
        # the calibration tokens through packed rows once more, as after the solve
        dict(name="int4-rows", op="int4", M=8192, C=7168, R=4096, gs=128, bias=True, act="silu", residual=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm_fp8", "gated", "train", "int4"])
    if op in ("norm", "norm_fp8"):
        T, C = _log_int(rng, 1, 8192), _log_int(rng, 256, 7168)
        if rng.random() < 0.6:
            C = max(8, C // 8 * 8)
        return dict(op=op, T=T, C=C, dtype=rng.choice(["bf16", "bf16", "f32"]), residual=rng.random() < 0.7)
    if op in ("gated", "train"):
        H, I = _log_int(rng, 256, 7168), _log_int(rng, 128, 2048)
        if rng.random() < 0.7:
            H, I = max(8, H // 8 * 8), max(8, I // 8 * 8)
        E, topk = rng.choice([1, 4, 8, 16, 32]), rng.choice([1, 2, 4, 8])
        return dict(op="gated", tokens=_log_int(rng, 1, 1024), topk=min(topk, E), E=E, H=H, I=I, train=op == "train")
    M, C, R = _log_int(rng, 1, 4096), _log_int(rng, 256, 7168), _log_int(rng, 64, 4096)
    if rng.random() < 0.7:
        C, R = C // 32 * 32, max(8, R // 8 * 8)
    return dict(op="int4", M=M, C=C, R=R, gs=rng.choice([32, 64, 128, 128]), bias=rng.random() < 0.5,
                act=rng.choice(["none", "silu", "gelu", "relu"]), residual=rng.random() < 0.5)


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape, scale=1.0, dtype=torch.bfloat16):
    return (scale * torch.randn(*shape, generator=g, device=DEV)).to(dtype)


def _route(tokens, E, topk, g):
    """Rows per expert and which token each row is, popularity ~ rank^-1.1 over a random order."""
    pop = torch.empty(E, device=DEV)
    pop[torch.randperm(E, generator=g, device=DEV)] = torch.arange(1, E + 1, device=DEV).float() ** -1.1
    logits = torch.randn(tokens, E, generator=g, device=DEV) + pop.log()
    expert = logits.topk(topk, dim=-1).indices.reshape(-1)
    order = torch.argsort(expert, stable=True)
    return order // topk, torch.bincount(expert, minlength=E)


def _draw_inputs(case, seed):
    """The tensors alone, from the seed alone."""
    g = _gen(seed)
    if case["op"] in ("norm", "norm_fp8"):
        dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        T, C = case["T"], case["C"]
        return dict(x=_randn(g, T, C, dtype=dt),
                    r=_randn(g, T, C, scale=3.0, dtype=dt) if case["residual"] else None,
                    w=(1.0 + 0.1 * torch.randn(C, generator=g, device=DEV)).to(dt))
    if case["op"] == "gated":
        E, H, I = case["E"], case["H"], case["I"]
        tok, counts = _route(case["tokens"], E, case["topk"], g)
        rows = _randn(g, case["tokens"], H)[tok].contiguous()
        s = dict(rows=rows, counts=counts, wg=_randn(g, E, I, H, scale=0.02), wu=_randn(g, E, I, H, scale=0.02))
        if case["train"]:
            s["dh"] = _randn(g, rows.shape[0], I)
        return s
    M, C, R, gs = case["M"], case["C"], case["R"], case["gs"]
    G, words = -(-C // gs), -(-C // 8)
    return dict(x=_randn(g, M, C),
                packed=torch.randint(-2 ** 31, 2 ** 31, (R, words), generator=g, device=DEV, dtype=torch.int64).to(torch.int32),
                scale=0.002 + 0.004 * torch.rand(R, G, generator=g, device=DEV),
                bias=_randn(g, R) if case["bias"] else None,
                residual=_randn(g, M, R) if case["residual"] else None)


def prepare(case, seed):
    s = _draw_inputs(case, seed)
    s["case"] = case
    if case["op"] == "gated":
        counts = s.pop("counts")
        s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        s["longest"] = int(counts.max())
        if case["train"]:
            for k in ("rows", "wg", "wu"):
                s[k].requires_grad_(True)
    if case["op"] == "int4":
        s["record"] = dict(weight_packed=s.pop("packed"), weight_scale=s.pop("scale"),
                           weight_shape=torch.tensor([case["R"], case["C"]], dtype=torch.int64))
    return s


# ------------------------------------------------------------------ plain forms
def _norm_plain(s):
    x = s["x"].float()
    if s["r"] is not None:
        x = x + s["r"].float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["w"].float()
    res = [] if s["r"] is None else [x.to(s["x"].dtype)]
    if s["case"]["op"] == "norm":
        return [y.to(s["x"].dtype)] + res
    T, C = y.shape
    G = -(-C // FP8_GROUP)
    yg = torch.nn.functional.pad(y, (0, G * FP8_GROUP - C)).view(T, G, FP8_GROUP)
    scale = yg.abs().amax(-1).clamp_min(1e-12) / FP8_MAX
    codes = (yg / scale[..., None]).to(torch.float8_e4m3fn).view(T, G * FP8_GROUP)[:, :C].contiguous()
    return [codes, scale] + res


def _act(name, v):
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    if name == "relu":
        return v.clamp_min(0)
    return v


def _padded(v, offsets, longest):
    """[E, longest, .] float32: each expert's rows, zeros behind them."""
    j = torch.arange(longest, device=DEV)
    at = offsets[:-1, None].long() + j
    live = at < offsets[1:, None]
    return v[at.clamp_max(v.shape[0] - 1)].float() * live[..., None]


def _flat(p, offsets, n):
    i = torch.arange(n, device=DEV, dtype=offsets.dtype)
    e = torch.searchsorted(offsets[1:].contiguous(), i, right=True)
    return p[e, i.long() - offsets[e].long()]


@torch.no_grad()
def _gated_plain(s):
    off, n = s["offsets"], s["rows"].shape[0]
    x = _padded(s["rows"], off, s["longest"])
    wg, wu = s["wg"].float(), s["wu"].float()
    g, u = torch.bmm(x, wg.transpose(1, 2)), torch.bmm(x, wu.transpose(1, 2))
    sig = torch.sigmoid(g)
    h = _flat(g * sig * u, off, n).bfloat16()
    if not s["case"]["train"]:
        return [h]
    dh = _padded(s["dh"], off, s["longest"])
    du = dh * g * sig
    dg = dh * u * (sig * (1.0 + g * (1.0 - sig)))
    dx = torch.bmm(dg, wg) + torch.bmm(du, wu)
    return [h, _flat(dx, off, n).bfloat16(), torch.bmm(dg.transpose(1, 2), x).bfloat16(),
            torch.bmm(du.transpose(1, 2), x).bfloat16()]


def _int4_plain(s):
    c, rec = s["case"], s["record"]
    shifts = torch.arange(0, 32, 4, device=DEV, dtype=torch.int32)
    q = ((rec["weight_packed"][..., None] >> shifts) & 15).view(c["R"], -1)[:, : c["C"]]
    group = torch.arange(c["C"], device=DEV) // c["gs"]
    w = (q - 8).float() * rec["weight_scale"][:, group]
    y = s["x"].float() @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = _act(c["act"], y)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return [y.bfloat16()]


# ------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if not own:
        return _norm_plain(state) if op in ("norm", "norm_fp8") else _gated_plain(state) if op == "gated" else _int4_plain(state)
    engine = _engine()
    if op == "norm":
        out = engine.rms_norm(state["x"], state["w"], EPS, residual=state["r"])
        return list(out) if state["r"] is not None else [out]
    if op == "norm_fp8":
        return list(engine.rms_norm_fp8(state["x"], state["w"], EPS, residual=state["r"]))
    if op == "gated":
        h = engine.expert_gated_rows(state["rows"], state["offsets"], state["wg"], state["wu"], activation="silu")
        if not state["case"]["train"]:
            return [h]
        return [h.detach(), *torch.autograd.grad(h, (state["rows"], state["wg"], state["wu"]), state["dh"])]
    act = None if state["case"]["act"] == "none" else state["case"]["act"]
    return [engine.linear_int4(state["x"], state["record"], bias=state["bias"], activation=act,
                               residual=state["residual"], group_size=state["case"]["gs"])]


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = _draw_inputs(case, seed)
    f64 = torch.float64
    if case["op"] in ("norm", "norm_fp8"):
        v = s["x"].to(f64) if s["r"] is None else s["x"].to(f64) + s["r"].to(f64)
        y = v / (v.square().sum(-1, keepdim=True) / case["C"] + EPS).sqrt() * s["w"].to(f64)
        tail = [] if s["r"] is None else [v]
        if case["op"] == "norm":
            return [y] + tail
        codes, scales = torch.empty_like(y), []
        for c0 in range(0, case["C"], FP8_GROUP):
            part = y[:, c0:c0 + FP8_GROUP]
            m = part.abs().max(dim=-1, keepdim=True).values.clamp(min=1e-12) / FP8_MAX
            codes[:, c0:c0 + FP8_GROUP] = part / m
            scales.append(m)
        return [codes, torch.cat(scales, 1)] + tail
    if case["op"] == "gated":
        # expert by expert
        n = s["rows"].shape[0]
        h = torch.zeros(n, case["I"], dtype=f64, device=DEV)
        if case["train"]:
            dx = torch.zeros(n, case["H"], dtype=f64, device=DEV)
            dwg, dwu = (torch.zeros(case["E"], case["I"], case["H"], dtype=f64, device=DEV) for _ in range(2))
        a = 0
        for e, k in enumerate(s["counts"].tolist()):
            if k:
                x, wg, wu = s["rows"][a:a + k].to(f64), s["wg"][e].to(f64), s["wu"][e].to(f64)
                g, u = x.mm(wg.t()), x.mm(wu.t())
                p = 1.0 / (1.0 + torch.exp(-g))
                h[a:a + k] = g * p * u
                if case["train"]:
                    dh = s["dh"][a:a + k].to(f64)
                    dg, du = dh * u * (p + g * p * (1.0 - p)), dh * (g * p)
                    dx[a:a + k] = dg.mm(wg) + du.mm(wu)
                    dwg[e], dwu[e] = dg.t().mm(x), du.t().mm(x)
            a += k
        return [h, dx, dwg, dwu] if case["train"] else [h]
    R, C, gs = case["R"], case["C"], case["gs"]
    w = torch.empty(R, C, dtype=f64, device=DEV)
    for k in range(8):                                   # nibble k of every word: columns k, k + 8, ...
        cols = torch.arange(k, C, 8, device=DEV)
        nib = torch.div(s["packed"].long() & 0xFFFFFFFF, 16 ** k, rounding_mode="floor") % 16
        w[:, cols] = (nib[:, : cols.numel()].to(f64) - 8.0) * s["scale"].to(f64)[:, cols // gs]
    y = s["x"].to(f64).mm(w.t())
    if s["bias"] is not None:
        y += s["bias"].to(f64)
    if case["act"] == "silu":
        y = y / (1.0 + torch.exp(-y))
    elif case["act"] == "gelu":
        y = y / (1.0 + torch.exp(-2.0 * (2.0 / math.pi) ** 0.5 * (y + 0.044715 * y ** 3)))
    elif case["act"] == "relu":
        y = torch.where(y > 0, y, torch.zeros_like(y))
    if s["residual"] is not None:
        y = y + s["residual"].to(f64)
    return [y]


# ------------------------------------------------------------------ what a pass cannot do without
def _live_experts(case):
    """Experts that a batch reaches: all of them once it is large, one per row where it is small."""
    return min(case["E"], case["tokens"] * case["topk"])


def work(case):
    if case["op"] in ("norm", "norm_fp8"):
        n, size = case["T"] * case["C"], 2 if case["dtype"] == "bf16" else 4
        b = n * size * (3 if case["residual"] else 1) + case["C"] * size
        b += n * size if case["op"] == "norm" else n + 4 * case["T"] * -(-case["C"] // FP8_GROUP)
        return {"bytes": b, "flops": 6 * n}
    if case["op"] == "gated":
        n, H, I = case["tokens"] * case["topk"], case["H"], case["I"]
        w = 2 * 2 * _live_experts(case) * I * H
        b = 2 * n * H + w + 2 * n * I
        if case["train"]:
            return {"bytes": b + 2 * n * I + 2 * n * H + 2 * 2 * case["E"] * I * H, "flops": 12 * n * H * I}
        return {"bytes": b, "flops": 4 * n * H * I}
    M, R, C = case["M"], case["R"], case["C"]
    b = 4 * R * -(-C // 8) + 4 * R * -(-C // case["gs"]) + 2 * M * C + 2 * M * R
    b += (2 * R if case["bias"] else 0) + (2 * M * R if case["residual"] else 0)
    return {"bytes": b, "flops": 2 * M * R * C}
