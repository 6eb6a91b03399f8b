"""The operators around the recurrence run together, as a state-space block uses them: residual norm, projection, short
convolution, scan, gated norm -- forward and backward against the same block in 64 bits, and token by token from a prompt."""
import pytest
import torch
import torch.nn.functional as F

from oracle import block_oracle as bo

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def params(seed, C, H, Hq, K, V, W):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    conv = H * V + 2 * Hq * K
    return dict(norm=1 + 0.1 * r(C), w_in=r(2 * H * V + 2 * Hq * K + H, C) / C ** 0.5, conv_w=r(conv, W) / W ** 0.5, conv_b=0.1 * r(conv),
                gt_bias=-2 + 0.3 * r(H), g=0.5 + r(H).abs(), D=1 + 0.1 * r(H), o_norm=1 + 0.1 * r(V), w_out=r(C, H * V) / (H * V) ** 0.5)


def block(p, x, res, dims, state=None, conv_state=None, cu=None, decode=False):
    """One block on (x, res): returns (output of the mixer, new residual, final state, final convolution state)."""
    from palimpsa_b200.layers import add_rms_norm, layer_epilogue, short_conv, short_conv_step
    from palimpsa_b200.ops import chunk_ssm, ssm_step
    H, Hq, K, V = dims
    y, z = add_rms_norm(x, p["norm"], residual=res)
    gate, xbc, gt = (y @ p["w_in"].T.to(y.dtype)).split([H * V, H * V + 2 * Hq * K, H], -1)
    if decode:
        xbc = short_conv_step(xbc, p["conv_w"], conv_state, p["conv_b"])
    else:
        xbc, conv_state = short_conv(xbc, p["conv_w"], p["conv_b"], initial_state=conv_state, output_final_state=True, cu_seqlens=cu)
    v, k, q = xbc.split([H * V, Hq * K, Hq * K], -1)
    q, k, v = q.unflatten(-1, (Hq, K)), k.unflatten(-1, (Hq, K)), v.unflatten(-1, (H, V))
    if decode:
        o = ssm_step(q, k, v, gt, p["g"], state, D=p["D"], gt_bias=p["gt_bias"], gt_softplus=True)
    else:
        o, state = chunk_ssm(q, k, v, gt, p["g"], D=p["D"], gt_bias=p["gt_bias"], gt_softplus=True, initial_state=state,
                             output_final_state=True, cu_seqlens=cu)
    o = layer_epilogue(o, None, None, p["o_norm"], gate.unflatten(-1, (H, V)))
    return o.flatten(-2) @ p["w_out"].T.to(o.dtype), z, state, conv_state


def block64(p, x, res, dims):
    """The same in 64 bits, differentiable."""
    H, Hq, K, V = dims
    B, T, _ = x.shape
    z = x + res
    y = bo.rms_norm(z, p["norm"], 1e-5)
    gate, xbc, gt = (y @ p["w_in"].T).split([H * V, H * V + 2 * Hq * K, H], -1)
    xbc, _ = bo.short_conv(xbc, p["conv_w"], p["conv_b"])
    v, k, q = xbc.split([H * V, Hq * K, Hq * K], -1)
    rep = H // Hq
    q, k = (t.unflatten(-1, (Hq, K)).repeat_interleave(rep, 2) for t in (q, k))
    v = v.unflatten(-1, (H, V))
    dt = F.softplus(gt + p["gt_bias"])
    h, outs = torch.zeros(B, H, V, K, dtype=x.dtype), []
    for t in range(T):
        h = torch.exp(-p["g"] * dt[:, t])[..., None, None] * h + (dt[:, t, :, None] * v[:, t])[..., None] * k[:, t, :, None]
        outs.append((h * q[:, t, :, None]).sum(-1) + p["D"][:, None] * v[:, t])
    o = torch.stack(outs, 1)
    o = bo.rms_norm(o, p["o_norm"], 1e-5) * F.silu(gate.unflatten(-1, (H, V)))
    return o.flatten(-2) @ p["w_out"].T, z


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-4), (torch.bfloat16, 4e-2)])
def test_block_forward_and_gradients(dtype, tol):
    """Relative 2-norms.  float32: the projections' sums (TF32 off) and the chain's condition, some hundred roundings of 2^-24 through
    two norms.  bfloat16: about eight roundings of at most 2^-8 one after the other, forward, and as many back."""
    dims, C, B, T = (4, 2, 32, 16), 48, 2, 150
    p = params(1, C, *dims, 4)
    gen = torch.Generator().manual_seed(2)
    x, res, do, dz = (torch.randn(B, T, C, generator=gen) for _ in range(4))
    x, do = x.to(dtype), do.to(dtype)
    p64 = {n: t.double().requires_grad_(True) for n, t in p.items()}
    x64, r64 = x.double().requires_grad_(True), res.double().requires_grad_(True)
    y, z = block64(p64, x64, r64, dims)
    ref = torch.autograd.grad([y, z], [x64, r64, *p64.values()], [do.double(), dz.double()])
    pg = {n: t.to(DEV).requires_grad_(True) for n, t in p.items()}
    xg, rg = x.to(DEV).requires_grad_(True), res.to(DEV).requires_grad_(True)
    yg, zg, _, _ = block(pg, xg, rg, dims)
    assert zg.dtype == torch.float32 and yg.dtype == dtype
    got = torch.autograd.grad([yg, zg], [xg, rg, *pg.values()], [do.to(DEV), dz.to(DEV)])
    rel = lambda a, b: float((a.detach().cpu().double() - b.detach()).norm() / b.detach().norm())
    errs = {"y": rel(yg, y), **{n: rel(a, b) for n, a, b in zip(("x", "res", *p), got, ref)}}
    assert all(e < tol for e in errs.values()), errs


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_then_tokens(dtype):
    """A packed batch of prompts, then tokens one by one on the states it left: as the same sequences run whole."""
    dims, C, lens, more = (4, 1, 32, 16), 40, (5, 130, 1), 4
    p = {n: t.to(DEV) for n, t in params(3, C, *dims, 4).items()}
    gen = torch.Generator().manual_seed(4)
    seqs = [torch.randn(1, n + more, C, generator=gen).to(DEV, dtype) for n in lens]
    whole = [block(p, s, s.float(), dims)[0][0] for s in seqs]
    packed = torch.cat([s[:, :n] for s, n in zip(seqs, lens)], 1)
    cu = torch.tensor([0, 5, 135, 136], device=DEV)
    out, _, state, conv_state = block(p, packed, packed.float(), dims, cu=cu)
    scale = max(float(w.float().abs().max()) for w in whole)
    close = lambda a, b: float((a.float() - b.float()).abs().max()) <= (3e-5 if dtype == torch.float32 else 4e-2) * scale
    for i, (w, n) in enumerate(zip(whole, lens)):
        assert close(out[0, int(cu[i]):int(cu[i + 1])], w[:n])
    for t in range(more):
        tok = torch.cat([s[:, n + t:n + t + 1] for s, n in zip(seqs, lens)])
        o = block(p, tok, tok.float(), dims, state=state, conv_state=conv_state, decode=True)[0]
        for i, (w, n) in enumerate(zip(whole, lens)):
            assert close(o[i, 0], w[n + t]), (t, i)


def test_quantised_norm_feeds_a_product():
    """q * scale is y to half a step of the 8-bit type: relative 2^-4 (and 2^-10 of the largest below 2^-6), or 1/254 of the largest."""
    from palimpsa_b200.layers import add_rms_norm, add_rms_norm_quant
    gen = torch.Generator().manual_seed(5)
    x, res, w = (torch.randn(70, 512, generator=gen).to(DEV) for _ in range(3))
    y, z = add_rms_norm(x, w[0], residual=res)
    for t in (torch.float8_e4m3fn, torch.int8):
        q, s, zq = add_rms_norm_quant(x, w[0], residual=res, dtype=t, block=128)
        each = s.repeat_interleave(128, -1)
        step = torch.maximum(y.abs() * 2.0 ** -4, each * 2.0 ** -10) if t != torch.int8 else each / 2
        assert torch.equal(z, zq) and ((q.float() * each - y).abs() <= step * (1 + 2.0 ** -18) + 1e-6 * y.abs()).all()
