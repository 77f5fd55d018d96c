"""Tensors with a tangent (forward-mode differentiation) ask for no gradient and would lose it behind a raw
pointer: every operator refuses them, before anything reaches a GPU."""
import pytest
import torch
from torch.autograd import forward_ad

from forge import engine


def _calls():
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)   # noqa: E731
    rec = lambda scale: dict(weight_packed=torch.zeros(8, 2, dtype=torch.int32), weight_scale=scale,   # noqa: E731
                             weight_shape=torch.tensor([8, 16]))
    one = torch.ones(8, 1)
    return [
        (lambda x: engine.rms_norm(x, bf(16)), bf(4, 16)),
        (lambda w: engine.rms_norm(bf(4, 16), w), bf(16)),
        (lambda r: engine.rms_norm(bf(4, 16), bf(16), residual=r), bf(4, 16)),
        (lambda x: engine.rms_norm_fp8(x, bf(16)), bf(4, 16)),
        (lambda x: engine.expert_gated_rows(x, [0, 2, 4], bf(2, 8, 16), bf(2, 8, 16)), bf(4, 16)),
        (lambda w: engine.expert_gated_rows(bf(4, 16), [0, 2, 4], w, bf(2, 8, 16)), bf(2, 8, 16)),
        (lambda w: engine.expert_gated_rows(bf(4, 16), [0, 2, 4], bf(2, 8, 16), w), bf(2, 8, 16)),
        (lambda x: engine.linear_int4(x, rec(one)), bf(4, 16)),
        (lambda s: engine.linear_int4(bf(4, 16), rec(s)), one),
        (lambda b: engine.linear_int4(bf(4, 16), rec(one), bias=b), bf(8)),
        (lambda r: engine.linear_int4(bf(4, 16), rec(one), residual=r), bf(4, 8)),
    ]


@pytest.mark.parametrize("i", range(11))
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(i, grad):
    f, t = _calls()[i]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(t, torch.ones_like(t))
        with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
            f(dual)
        if not torch.cuda.is_available():                 # none of the arguments has one: as always
            with pytest.raises(RuntimeError) as e:
                f(t)
            assert "forward-mode" not in str(e.value)
    with pytest.raises(RuntimeError):
        torch.func.jvp(f, (t,), (torch.ones_like(t),))
