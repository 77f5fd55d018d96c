"""A block with the solver's default (asymmetric) grids, from the residual's addition to the sum of the experts'
results: every token's result against the same sum in float64 on the weights that are written back into the layer."""
import pytest
import torch

from block_ref import U, gated64, half_step, within
from forge import engine, export
from forge.moe import ExpertGroupGPTQ

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("group_size", [128, 64])
def test_tokens_results(hip, group_size):
    g = torch.Generator(device=DEV).manual_seed(group_size)
    mk = lambda s, *sh: (s * torch.randn(*sh, generator=g, device=DEV)).bfloat16()   # noqa: E731
    T, H, I, E, K = 230, 256, 192, 6, 2
    hidden, attn, w, router = mk(1.0, T, H), mk(0.5, T, H), mk(1.0, H), mk(0.1, E, H)
    wg, wu, wd = mk(0.06, E, I, H), mk(0.06, E, I, H), mk(0.06, E, H, I)
    normed, stream = engine.rms_norm(attn, w, residual=hidden)
    logits = normed.float() @ router.float().T
    logits[:, 4] = -1e9                                            # an expert without rows
    rw, ri = torch.softmax(logits, -1).topk(K, dim=-1)
    rows, offs = engine.routed_rows(normed, ri, None, E)
    h = engine.expert_gated_rows(rows, offs, wg, wu)
    within(h, *gated64(rows, offs, wg, wu, "silu"))

    group = ExpertGroupGPTQ([wd], bits=4, group_size=group_size, symmetric=False, device=DEV)
    group.update(h, offs)
    (codes, scales, zeros), = group.quantize()
    token = torch.argsort(ri.reshape(-1), stable=True) // K        # routed_rows' order: by expert, then by token
    assert torch.equal(rows, normed[token])
    weight = rw.reshape(-1)[torch.argsort(ri.reshape(-1), stable=True)].double()

    out = stream.double()
    want, bound = stream.double(), torch.zeros(T, H, dtype=torch.float64, device=DEV)
    r = half_step(torch.bfloat16)
    for e in range(E):
        a, b = offs[e], offs[e + 1]
        rec = export.pack_weight(export.layer_record(codes[e], scales[e], zeros[e], group_size, 4, (H, I)), 4, False,
                                 group_size)
        y = engine.linear_int4(h[a:b], rec, group_size=group_size)
        W = engine.dequantize_forge_full(torch.float32, codes[e], scales[e], zeros[e], group_size, DEV).double()
        y64, size = h[a:b].double() @ W.T, h[a:b].double().abs() @ W.abs().T
        # f32 sums (a written-back weight is rounded once more), rounded to bf16
        off = (I + 2 * (I // group_size + 1) + 9) * U * size * (1 + r) + r * y64.abs()
        out.index_add_(0, token[a:b], weight[a:b, None] * y.double())
        want.index_add_(0, token[a:b], weight[a:b, None] * y64)
        bound.index_add_(0, token[a:b], weight[a:b, None] * off)
    # (the sums over experts are in 64 bits on both sides)
    assert ((out - want).abs() <= bound + 1e-12).all()
    assert (out - stream.double()).abs().amax(1).min() > 0         # every token got something


def test_two_threads_on_streams_of_their_own(hip):
    """every operator from two threads at once, odd sizes (padded copies) among them: the bits of one after the other"""
    import threading
    g = torch.Generator(device=DEV).manual_seed(3)
    mk = lambda s, *sh: (s * torch.randn(*sh, generator=g, device=DEV)).bfloat16()   # noqa: E731

    def job(H, I):
        x, w = mk(1.0, 500, H), mk(1.0, H)
        leaves = [mk(1.0, 500, H), mk(0.05, 3, I, H), mk(0.05, 3, I, H)]
        dh, offs = mk(1.0, 500, I), torch.tensor([0, 130, 130, 500], dtype=torch.int32, device=DEV)
        codes = torch.randint(0, 16, (H, I), generator=g, device=DEV, dtype=torch.uint8)
        scale = torch.rand(H, -(-I // 64), generator=g, device=DEV)
        zero = torch.randint(0, 16, scale.shape, generator=g, device=DEV)
        rec = export.pack_weight({"qweight": codes, "scale": scale, "zero": zero}, 4, False, 64)

        def run():
            y, s = engine.rms_norm(x, w, residual=leaves[0])
            c, sc, _ = engine.rms_norm_fp8(x, w, residual=leaves[0])
            t = [v.detach().requires_grad_(True) for v in leaves]
            h = engine.expert_gated_rows(t[0], offs, t[1], t[2])
            grads = torch.autograd.grad(h, t, dh)
            out = engine.linear_int4(h.detach(), rec, residual=s, group_size=64)
            return [y, s, c.view(torch.uint8), sc, h.detach(), *grads, out]
        return run

    jobs = [job(256, 192), job(131, 77)]
    want = [j() for j in jobs]
    got, errors = [[], []], []
    torch.cuda.synchronize()

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got[i].append(jobs[i]())
                stream.synchronize()
        except Exception as e:                                     # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for i in range(2):
        assert len(got[i]) == 20
        for res in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(res, want[i]))
