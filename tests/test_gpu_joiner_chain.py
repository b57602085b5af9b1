"""The joiner's operators run together, as they are used: norms of the encoder's and the predictor's outputs, the joint
layer norm, an output layer, the adjustment of the logits, the loss (training, padded and packed), and a greedy
decoder's loop (one frame and one context per step)."""
import numpy as np
import pytest
import torch

from joiner_ref import U, check, norm_reference, valid_rows
from test_gpu_logits import oracle_from_logits

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def W():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import warp_ctct_b200
    from warp_ctct_b200 import _lib
    _lib.lib()
    return warp_ctct_b200


def _inputs(W, N, T, U1, H, V):
    g = torch.Generator(device=DEV)
    g.manual_seed(N + T)
    r = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    p = {"f": r(N, T, H), "g": r(N, U1, H), "w": 1 + 0.2 * r(H), "b": 0.2 * r(H), "out": r(H, V) / H ** 0.5, "bias": 0.3 * r(V)}
    labels = torch.randint(1, 9, (N, U1 - 1), generator=g, device=DEV, dtype=torch.int32)
    lx = torch.randint(2 * U1, T + 1, (N,), generator=g, device=DEV, dtype=torch.int32)
    ly = torch.randint(1, U1, (N,), generator=g, device=DEV, dtype=torch.int32)
    ok = torch.rand((N, U1, V), generator=g, device=DEV) < 0.8
    ok[..., :9] = True      # the blank and the tokens that occur stay possible
    return p, labels, lx, ly, ok


def _train(W, p, labels, lx, ly, words, packed):
    q = {k: v.detach().requires_grad_(True) for k, v in p.items()}
    how = dict(bias=q["bias"], allowed=words, repetition_penalty=1.2, presence_penalty=0.25, frequency_penalty=0.1)
    T = p["f"].size(1)
    if packed:
        rows = int((lx.long() * (ly.long() + 1)).sum())
        h = W.joint_layer_norm_packed(q["f"], q["g"], lx, ly, q["w"], q["b"], rows=rows)
        z = W.adjust_joint_logits_packed(h @ q["out"], labels, lx, ly, max_frames=T, **how)
        loss = W.ctct_loss_packed(z, labels, lx, ly, max_frames=T, from_logits=True)
    else:
        h = W.joint_layer_norm(q["f"], q["g"], lx, ly, q["w"], q["b"])
        z = W.adjust_joint_logits(h @ q["out"], labels, lx, ly, **how)
        loss = W.ctct_loss_from_logits(z, labels, lx, ly)
    dz, = torch.autograd.grad(loss, [z], retain_graph=True)
    return loss.detach(), z.detach(), dz, dict(zip(q, torch.autograd.grad(loss, list(q.values()))))


def test_training_step(W):
    N, T, U1, H, V = 4, 36, 9, 96, 40
    p, labels, lx, ly, ok = _inputs(W, N, T, U1, H, V)
    words = W.pack_token_mask(ok)
    valid = valid_rows(lx, ly, N, T, U1, DEV)
    loss, z, dz, grads = _train(W, p, labels, lx, ly, words, False)
    loss_p, z_p, dz_p, grads_p = _train(W, p, labels, lx, ly, words, True)
    # the loss of these logits is the oracle's
    costs, _ = oracle_from_logits(z.cpu().numpy(), labels.cpu().numpy(), lx.cpu().numpy(), ly.cpu().numpy(), np.full(N, 1.0 / N))
    assert np.isfinite(costs).all()
    for v in (loss, loss_p):
        assert abs(v.item() - costs.mean()) <= 1e-5 * costs.mean() + 40 * U * np.abs(costs).max()
    # every gradient is the 64-bit chain's on the same gradient of the logits
    d = {k: v.double() for k, v in p.items()}
    s = (d["f"].unsqueeze(2) + d["g"].unsqueeze(1))[valid]
    counts = torch.cat([torch.zeros((N, 1, V), device=DEV, dtype=torch.float64),
                        (labels.long().unsqueeze(-1) == torch.arange(V, device=DEV)).double().cumsum(1)], 1)
    per_row = lambda t: t.unsqueeze(1).expand(N, T, U1, V)[valid]  # noqa: E731
    for dzv, got in ((dz[valid], grads), (dz_p, grads_p)):
        dzv = dzv.double()
        sn = s - s.mean(-1, keepdim=True)
        h = sn * (sn.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * d["w"] + d["b"]
        x = h @ d["out"]
        hit = per_row(counts) > 0
        near = x.abs() < 200 * U * (h.abs() @ d["out"].abs())   # a logit whose sign float32 may see otherwise
        assert not bool((near & hit).any())
        dx = torch.where(per_row(ok), dzv * torch.where(hit, torch.where(x > 0, 1 / 1.2, 1.2), 1.0), 0.0)
        dh, e_h = dx @ d["out"].T, (V + 8) * U * (dx.abs() @ d["out"].abs().T)   # V products in float32
        amax = (p["f"].abs().amax(-1).unsqueeze(2) + p["g"].abs().amax(-1).unsqueeze(1))[valid].unsqueeze(-1).double()
        mag = lambda t: (t.double() - t.double().mean(-1, keepdim=True)).abs()  # noqa: E731
        parts = (mag(p["f"]).unsqueeze(2) + mag(p["g"]).unsqueeze(1))[valid]
        val, tol = norm_reference(s, p["w"], p["b"], 1e-5, dh, amax, 80, s.size(0) + 64, torch.float32, torch.float32, parts)
        r = (sn.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
        xh, we = (sn * r).abs(), d["w"].abs() * e_h
        e_ds = tol["ds"] + r * (we + we.mean(-1, keepdim=True) + xh * (we * xh).mean(-1, keepdim=True))
        full = torch.zeros((N, T, U1, H), device=DEV, dtype=torch.float64)
        ds, e, terms = full.clone(), full.clone(), full.clone()
        ds[valid], e[valid], terms[valid] = val["ds"], e_ds, val["terms"]
        check("df", got["f"], ds.sum(2), e.sum(2) + 80 * U * terms.sum(2))
        check("dg", got["g"], ds.sum(1), e.sum(1) + 80 * U * terms.sum(1))
        check("dw", got["w"], val["dw"], tol["dw"] + (e_h * xh).sum(0))
        check("db", got["b"], val["db"], tol["db"] + e_h.sum(0))
        want = torch.where(per_row(ok), dzv, 0.0).sum(0)
        check("dbias", got["bias"], want, (s.size(0) + 8) * U * dzv.abs().sum(0))
        want = h.T @ dx
        check("dout", got["out"], want, (s.size(0) + 200) * U * (h.abs().T @ dx.abs()))


def test_greedy_decoder(W):
    """Frame by frame, one hypothesis per stream: the tokens are those of the 64-bit forms."""
    R, T, H, V, L = 5, 24, 64, 130, 24
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    r = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    enc, emb, w, b, out, bias = r(R, T, H), r(V, H), 1 + 0.2 * r(H), 0.2 * r(H), r(H, V) / 4, 0.5 * r(V)
    ok = torch.rand((R, V), generator=g, device=DEV) < 0.7
    ok[:, 0] = True
    words = W.pack_token_mask(ok)
    tokens, lens = torch.full((R, L), -1, dtype=torch.int32, device=DEV), torch.zeros(R, dtype=torch.int32, device=DEV)
    last = torch.zeros(R, dtype=torch.int64, device=DEV)
    for t in range(T):
        pred = W.layer_norm(emb[last], w, b)
        h = W.joint_layer_norm(enc[:, t:t + 1], pred.unsqueeze(1), None, None, w, b)
        z = W.adjust_logits(h.view(R, H) @ out, tokens, lens, bias, words, 1.3, 0.2, 0.1)
        best = z.argmax(-1)
        # the same step in 64 bits
        ln = lambda x: (x - x.mean(-1, keepdim=True)) / (x.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt() * w.double() + b.double()  # noqa: E731
        z64 = ln(enc[:, t].double() + ln(emb[last].double())) @ out.double()
        seen = torch.arange(L, device=DEV) < lens.view(-1, 1)
        c = ((tokens.long().unsqueeze(-1) == torch.arange(V, device=DEV)) & seen.unsqueeze(-1)).sum(1).double()
        z64 = torch.where(c > 0, torch.where(z64 > 0, z64 / 1.3, z64 * 1.3), z64) - 0.2 * (c > 0) - 0.1 * c + bias.double()
        z64 = torch.where(ok, z64, float("-inf"))
        top = z64.topk(2, -1).values
        clear = top[:, 0] - top[:, 1] > 1e-4     # far above float32's error of a sum of 64 terms near 10
        assert bool((best == z64.argmax(-1))[clear].all())
        emit = best != 0
        rows = torch.arange(R, device=DEV)[emit]
        tokens[rows, lens[emit].long()] = best[emit].int()
        lens += emit.int()
        last = torch.where(emit, best, last)
    assert int(lens.max()) > 0
