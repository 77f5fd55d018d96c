"""Callers either side of the solve (forge/utils/engine.py, forge/utils/quant.py of the
reference): the dequantised weight that is written back into the layer before the block is
run again, the routed-row gather in front of the per-expert Hessian update, and the block's own
arithmetic around both: the norm in front of the router (``rms_norm``, ``rms_norm_fp8``), the
experts' gated rows that the down projection's Hessian takes (``expert_gated_rows``, with
gradients) and the product with the packed result of the solve (``linear_int4``)."""
from __future__ import annotations

from typing import Dict, Optional, Sequence, Tuple, Union

import torch
from torch.autograd import forward_ad

from forge.backend.hip import kernels, _need_one_device, _unit_rows, ACTIVATIONS


@torch.no_grad()
def dequantize_forge_full(dtype, qweight, scales, qzeros, group_size, device):
    """Same call as forge/utils/engine.py:71-97: (q - q0) * s with flat [R*G] per-group
    meta, computed in f32 and rounded to `dtype`; qweight [R, C] unpacked codes."""
    if qweight.dim() != 2:
        raise ValueError(f"Expected qweight (R,C) unpacked, got shape={tuple(qweight.shape)}")
    R, C = qweight.shape
    G = (C + group_size - 1) // group_size
    scales = scales.reshape(-1)
    qzeros = qzeros.reshape(-1)
    if scales.numel() != R * G or qzeros.numel() != R * G:
        raise ValueError(f"Expected scales/qzeros numel == R*G ({R * G}), "
                         f"got scales={scales.numel()}, qzeros={qzeros.numel()}")
    dev = torch.device(device)
    return kernels.dequantize_groups(qweight.to(dev).to(torch.uint8), scales.to(dev),
                                     qzeros.to(dev), group_size, dtype)


@torch.no_grad()
def routed_rows(x: torch.Tensor, router_indices: torch.Tensor,
                routing_weights: Optional[torch.Tensor], num_experts: int
                ) -> Tuple[torch.Tensor, list]:
    """What the fused-expert hook of forge/utils/engine.py:210-238 feeds to the per-expert
    handles, for all experts at once: the rows of `x` [tokens, H] routed to each expert,
    scaled by their routing weight, grouped by expert in ascending token order.
    router_indices / routing_weights: [tokens, top_k].  Returns (rows [N, H], offsets
    [num_experts + 1]) as ExpertGroupGPTQ.update takes them.  Entries with an expert id
    outside [0, num_experts) are dropped, as the hook skips them."""
    ri = router_indices.reshape(router_indices.shape[0], -1).to(x.device)
    tok = torch.arange(ri.shape[0], device=x.device).unsqueeze(1).expand_as(ri).reshape(-1)
    exp = ri.reshape(-1).to(torch.int64)
    ok = (exp >= 0) & (exp < num_experts)
    # stable sort by expert keeps (token, k) order inside an expert, as nonzero() yields it
    order = torch.argsort(torch.where(ok, exp, torch.full_like(exp, num_experts)), stable=True)
    n_ok = int(ok.sum())
    order = order[:n_ok]
    counts = torch.bincount(exp[order], minlength=num_experts).cpu().tolist()
    offsets = [0]
    for c in counts:
        offsets.append(offsets[-1] + int(c))
    w = None
    if routing_weights is not None:
        w = routing_weights.reshape(ri.shape[0], -1).to(x.device).reshape(-1)[order].to(x.dtype)
    x2 = x if x.stride(-1) == 1 else x.contiguous()
    rows = kernels.gather_scaled_rows(x2, tok[order].contiguous(), w)
    return rows, offsets


def _no_tangent(name: str, *tensors):
    # (a dual tensor asks for no gradient; the level is looked at first because it costs nothing)
    if getattr(forward_ad, "_current_level", 0) < 0:
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{name} has no forward-mode derivative: call it on the primal tensors")


def _no_gradient(name: str, *tensors):
    _no_tangent(name, *tensors)
    if not torch.is_grad_enabled():
        return
    for t in tensors:
        if t is None or not t.requires_grad:
            continue
        raise RuntimeError(f"{name} has no backward pass: call it under torch.no_grad() or on detached "
                           "tensors")


def _rows_of(t: torch.Tensor) -> torch.Tensor:
    """[..., C] as [rows, C] with unit column stride"""
    return _unit_rows(t if t.dim() == 2 else t.reshape(-1, t.shape[-1]))


def _norm_arguments(name, x, weight, eps, residual):
    _no_gradient(name, x, weight, residual)
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"{name}: x is {x.dtype}, expected float32 or bfloat16")
    if weight.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"{name}: weight is {weight.dtype}, expected float32 or bfloat16")
    if x.dim() < 1 or x.shape[-1] == 0 or weight.dim() != 1 or weight.shape[0] != x.shape[-1]:
        raise ValueError(f"{name}: weight {tuple(weight.shape)} does not fit rows of x {tuple(x.shape)}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"{name}: residual {tuple(residual.shape)} {residual.dtype}, "
                         f"x {tuple(x.shape)} {x.dtype}")
    if not eps >= 0:
        raise ValueError(f"{name}: eps={eps}")
    return _rows_of(x), weight.contiguous(), None if residual is None else _rows_of(residual)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
             residual: Optional[torch.Tensor] = None):
    """Root-mean-square norm over the last dimension of x [..., C] (bf16 or f32), the residual
    added first:  s = x + residual,  y = s * rsqrt(mean(s^2) + eps) * weight.  Returns y, or
    (y, s) with a residual (s is the residual stream for the next addition), in x's dtype.
    Everything in f32 with one rounding at the end; the statistics come from the unrounded s.
    weight [C] bf16 or f32.  New tensors; no backward pass (refused where one is asked for)."""
    x2, w, r2 = _norm_arguments("rms_norm", x, weight, eps, residual)
    y, out = kernels.rms_norm_of_checked(x2, w, eps, r2)
    if x.dim() != 2:
        y, out = y.view(x.shape), None if out is None else out.view(x.shape)
    return y if residual is None else (y, out)


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                 residual: Optional[torch.Tensor] = None):
    """rms_norm with y in 8 bits: (codes [..., C] float8_e4m3fn, scale_inv [..., ceil(C/128)] f32
    [, s]), one scale = max(max |y|, 1e-12) / 448 per 128 columns, so that y = codes * scale_inv as
    ``kernels.fp8_block_dequant`` reads block-scaled weights."""
    x2, w, r2 = _norm_arguments("rms_norm_fp8", x, weight, eps, residual)
    codes, scale_inv, out = kernels.rms_norm_fp8_of_checked(x2, w, eps, r2)
    if x.dim() != 2:
        codes, scale_inv = codes.view(x.shape), scale_inv.view(*x.shape[:-1], scale_inv.shape[1])
        out = None if out is None else out.view(x.shape)
    return (codes, scale_inv) if residual is None else (codes, scale_inv, out)


class _GatedRows(torch.autograd.Function):
    """expert_gated_rows under autograd: keeps g and u in f32 (8 bytes per row and feature), which
    costs less than forming them again (two of the backward pass's four products)."""

    @staticmethod
    def forward(ctx, rows, offsets, w_gate, w_up, activation):
        I, H = w_gate.shape[1:]
        dev = _need_one_device(rows, offsets, w_gate, w_up)
        # odd sizes: the padded copies are kept, so that the backward pass need not make them again
        rows, w_gate, w_up = kernels.gated_operands(rows, offsets, w_gate, w_up)
        act = ACTIVATIONS[activation]
        h, g, u = kernels.gated_rows_of_operands(dev, rows, offsets, w_gate, w_up, act, True)
        ctx.save_for_backward(rows, offsets, w_gate, w_up, g, u)
        ctx.sizes = dev, act, H, I
        return h if h.shape[1] == I else h[:, :I].contiguous()

    @staticmethod
    def backward(ctx, dh):
        if torch.is_grad_enabled():
            # (once_differentiable would let a graph pass whose saved tensors alone ask for gradients)
            raise RuntimeError("expert_gated_rows has no gradients of its gradients (create_graph=True)")
        rows, offsets, w_gate, w_up, g, u = ctx.saved_tensors
        dev, act, H, I = ctx.sizes
        need = ctx.needs_input_grad
        if g.shape[1] != I:
            dh = kernels.pad_rows(_unit_rows(dh))
        dx, dwg, dwu = kernels.gated_gradients_of_operands(dev, dh, g, u, rows, offsets, w_gate, w_up, act,
                                                           (need[0], need[2], need[3]))
        if rows.shape[1] != H or g.shape[1] != I:
            dx = None if dx is None else dx[:, :H]
            dwg, dwu = (None if d is None else d[:, :I, :H] for d in (dwg, dwu))
        return dx, None, dwg, dwu, None


def expert_gated_rows(rows: torch.Tensor, offsets: Union[torch.Tensor, Sequence[int], None],
                      w_gate: torch.Tensor, w_up: torch.Tensor, activation: Optional[str] = "silu"
                      ) -> torch.Tensor:
    """The rows that reach each expert's down projection, for all experts at once:
    h_i = act(w_gate[e] x_i) * (w_up[e] x_i) for the rows x_i of expert e, i.e. what
    ``ExpertGroupGPTQ.update`` of the down projections takes.  rows [N, H] bf16 grouped by expert
    and offsets [E + 1] as ``routed_rows`` returns them (a list: copied to the device, which waits for the work
    queued there, and refused in a capture); offsets may also be an int32 or int64 tensor on
    the rows' device, which is taken without looking at it on the host (ascending within [0, N] is
    then the caller's duty; values outside are clamped).  w_gate, w_up [E, I, H] bf16, or [I, H]
    for a dense layer (offsets None: all rows are its own).  Rows of no expert (before offsets[0],
    from offsets[E] on) get 0.  activation: "silu", "gelu" (tanh form), "relu" or None.
    Sums in f32, h [N, I] bf16 rounded once.

    Differentiable in rows, w_gate and w_up (once: create_graph and forward mode are refused); gradients are bf16, with dg and du rounded to
    bf16 between the products.  A HIP graph of a training step captures ``kernels.gated_rows(...,
    keep=True)`` and ``kernels.gated_rows_backward`` directly; under autograd a capture is refused, and the backward pass of an
    eager call is not one to capture either: autograd runs it on that call's stream."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"expert_gated_rows: unknown activation {activation!r} (one of {list(ACTIVATIONS)})")
    for n, t in (("rows", rows), ("w_gate", w_gate), ("w_up", w_up)):
        if t.dtype != torch.bfloat16:
            raise ValueError(f"expert_gated_rows: {n} is {t.dtype}, expected bfloat16")
    if w_gate.shape != w_up.shape or w_gate.dim() not in (2, 3):
        raise ValueError(f"expert_gated_rows: w_gate {tuple(w_gate.shape)}, w_up {tuple(w_up.shape)}: "
                         "expected one [E, I, H] or [I, H] for both")
    if rows.dim() != 2 or rows.shape[1] != w_gate.shape[-1]:
        raise ValueError(f"expert_gated_rows: rows {tuple(rows.shape)} do not fit weights {tuple(w_gate.shape)}")
    if 0 in w_gate.shape:
        raise ValueError(f"expert_gated_rows: empty weights {tuple(w_gate.shape)}")
    if w_gate.dim() == 2:
        w_gate, w_up = w_gate.unsqueeze(0), w_up.unsqueeze(0)
    E, N = w_gate.shape[0], rows.shape[0]
    if offsets is None:
        if E != 1:
            raise ValueError(f"expert_gated_rows: {E} experts need offsets")
        # made on the device where the rows are on one: nothing to copy, nothing to wait for
        offsets = torch.arange(0, N + 1, N, dtype=torch.int32, device=rows.device) if rows.is_cuda and N else [0, N]
    if isinstance(offsets, torch.Tensor) and offsets.is_cuda:
        if offsets.dtype not in (torch.int32, torch.int64) or tuple(offsets.shape) != (E + 1,):
            raise ValueError(f"expert_gated_rows: offsets {tuple(offsets.shape)} {offsets.dtype}, expected "
                             f"[{E + 1}] int32 or int64")
        # (clamped while they are wide: behind 2^31 they would come back as others within [0, N])
        off = (offsets.clamp(0, N) if offsets.dtype == torch.int64 else offsets).to(torch.int32).contiguous()
    else:
        off = [int(v) for v in offsets]
        if len(off) != E + 1 or off[0] < 0 or off[-1] > N or any(a > b for a, b in zip(off, off[1:])):
            raise ValueError(f"expert_gated_rows: offsets must be {E + 1} ascending numbers within "
                             f"[0, {N}]")
        if rows.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("expert_gated_rows: offsets on the host cannot be captured (the copy waits for the GPU): "
                               "pass them as an int32 tensor on the rows' device")
        off = torch.tensor(off, dtype=torch.int32).to(rows.device)
    _no_tangent("expert_gated_rows", rows, w_gate, w_up)
    rows, w_gate, w_up = _unit_rows(rows), _unit_rows(w_gate), _unit_rows(w_up)
    if torch.is_grad_enabled() and (rows.requires_grad or w_gate.requires_grad or w_up.requires_grad):
        if torch.cuda.is_current_stream_capturing():
            # its engine waits for the streams that leaves were used on before: the capture would fail in
            # one of its threads, and the process with it
            raise RuntimeError("expert_gated_rows under autograd cannot be captured: capture kernels.gated_rows(..., "
                               "keep=True) and kernels.gated_rows_backward")
        return _GatedRows.apply(rows, off, w_gate, w_up, activation)
    return kernels.gated_rows(rows, off, w_gate, w_up, activation).contiguous()


def linear_int4(x: torch.Tensor, packed: Dict[str, torch.Tensor], bias: Optional[torch.Tensor] = None,
                activation: Optional[str] = None, residual: Optional[torch.Tensor] = None,
                group_size: Optional[int] = None) -> torch.Tensor:
    """A layer's product with its packed weights, as ``export.pack_weight`` returns them:
    act(x W^T + bias) + residual with W[r, c] = (code - zero) * weight_scale[r, c / group_size], the layer's
    dequantised weight.  The record's nibbles are code - zero + 8 modulo 16: with a ``weight_zero_point`` (whole
    numbers of an integer type, one per group; 0 .. 15 on the solver's grids, -240 .. 255 are exact) the codes are formed from both, without one every zero
    is 8 (symmetric records).  x [..., C] bf16, bias [R] bf16, residual [..., R] bf16;
    activation "silu", "gelu" (tanh form), "relu" or None; result [..., R] bf16, rounded once.
    group_size may be left out when the groups divide C evenly (or there is one) and no power of two gives as
    many groups, the last one shorter.  The weights stay
    4 bits wide in memory; no layout of them is kept.  No backward pass (refused where one is asked
    for)."""
    w, scale = packed["weight_packed"], packed["weight_scale"]
    _no_gradient("linear_int4", x, scale, bias, residual)
    R, C = packed["weight_shape"].tolist()
    if activation not in ACTIVATIONS:
        raise ValueError(f"linear_int4: unknown activation {activation!r} (one of {list(ACTIVATIONS)})")
    if x.dtype != torch.bfloat16:
        raise ValueError(f"linear_int4: x is {x.dtype}, expected bfloat16")
    if x.dim() < 1 or x.shape[-1] != C:
        raise ValueError(f"linear_int4: x {tuple(x.shape)} does not fit a weight of {R} x {C}")
    if w.dtype != torch.int32 or w.shape != (R, (C + 7) // 8):
        raise ValueError(f"linear_int4: weight_packed {tuple(w.shape)} {w.dtype}, expected "
                         f"[{R}, {(C + 7) // 8}] int32")
    if scale.dim() != 2 or scale.shape[0] != R or not 1 <= scale.shape[1] <= C:
        raise ValueError(f"linear_int4: weight_scale {tuple(scale.shape)}, expected [{R}, groups]")
    G = scale.shape[1]
    if group_size is None:
        if C % G:
            raise ValueError(f"linear_int4: {G} groups do not divide {C} columns evenly: pass group_size")
        group_size = C // G
        # another usual size may give as many groups, the last one shorter: 2 of 192 columns are 96 + 96 or 128 + 64
        usual = 1 << (group_size - 1).bit_length()
        if G > 1 and usual != group_size and (C + usual - 1) // usual == G:
            raise ValueError(f"linear_int4: {G} groups of {C} columns may be of {group_size} or of {usual}: pass group_size")
    if group_size < 1 or (C + group_size - 1) // group_size != G:
        raise ValueError(f"linear_int4: group_size={group_size} does not give {G} groups of {C} columns")
    zero = packed.get("weight_zero_point")
    if zero is not None:
        if zero.dtype.is_floating_point or zero.dtype.is_complex or zero.dtype == torch.bool:
            raise ValueError(f"linear_int4: weight_zero_point is {zero.dtype}, expected an integer type")
        if zero.shape != scale.shape:
            raise ValueError(f"linear_int4: weight_zero_point {tuple(zero.shape)}, weight_scale {tuple(scale.shape)}")
        zero = zero.to(torch.int32).contiguous()
    if bias is not None and (bias.dtype != torch.bfloat16 or bias.shape != (R,)):
        raise ValueError(f"linear_int4: bias {tuple(bias.shape)} {bias.dtype}, expected [{R}] bfloat16")
    shape = (*x.shape[:-1], R)
    if residual is not None and (residual.dtype != torch.bfloat16 or residual.shape != shape):
        raise ValueError(f"linear_int4: residual {tuple(residual.shape)} {residual.dtype}, expected "
                         f"{shape} bfloat16")
    y = kernels.linear_int4_of_checked(_rows_of(x), w.contiguous(), scale.float().contiguous(), zero, int(group_size),
                                       None if bias is None else bias.contiguous(), ACTIVATIONS[activation],
                                       None if residual is None else _rows_of(residual))
    return y if len(shape) == 2 else y.view(shape)
