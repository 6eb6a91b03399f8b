"""Plain 64-bit forms of the operators around the recurrence, on the CPU, and bounds for what rounding may add.

``magnitude=True`` runs the same sums over absolute values: the size of the terms that a result is summed from, which is
what the rounding of terms and partial sums is relative to.
"""
import torch


def softplus_dt(gt, gt_bias, softplus):
    u = gt.double() + (0 if gt_bias is None else gt_bias.double())
    dt = torch.nn.functional.softplus(u, threshold=20) if softplus else u
    return dt, (torch.where(u > 20, torch.ones_like(u), torch.sigmoid(u)) if softplus else torch.ones_like(u))


def ssm(q, k, v, gt, g, D=None, gt_bias=None, softplus=False, h0=None, do=None, dh=None, cu=None, magnitude=False):
    """chunk_ssm token by token; with ``do`` (and ``dh``) the gradients too.  Returns a dict."""
    B, T, H, V = v.shape
    Hq, K = q.shape[2:]
    seqs = [(b, 0, T) for b in range(B)] if cu is None else [(0, int(a), int(e)) for a, e in zip(cu[:-1], cu[1:])]
    size = (lambda x: x.abs()) if magnitude else (lambda x: x)
    rep = H // Hq
    q64, k64 = (size(x.double()).repeat_interleave(rep, 2) for x in (q, k))
    v64 = size(v.double())
    dt_all, slope = softplus_dt(gt, gt_bias, softplus)
    dts = size(dt_all)
    g64 = g.double()
    D64 = torch.zeros(H, dtype=torch.float64) if D is None else size(D.double())
    f_all = torch.exp(-g64 * dt_all)
    out = {"o": torch.zeros(B, T, H, V, dtype=torch.float64), "h": torch.zeros(len(seqs), H, V, K, dtype=torch.float64)}
    if do is not None:
        do64 = size(do.double())
        for n, x in (("dq", q64), ("dk", k64), ("dv", v64), ("dgt", dt_all), ("dlf", dt_all)):
            out[n] = torch.zeros_like(x)
        out["dh0"] = torch.zeros_like(out["h"])
    for n, (b, a, e) in enumerate(seqs):
        h = torch.zeros(H, V, K, dtype=torch.float64) if h0 is None else size(h0[n].double())
        hs = [h]
        for t in range(a, e):
            h = f_all[b, t][:, None, None] * h + dts[b, t][:, None, None] * v64[b, t][:, :, None] * k64[b, t][:, None]
            hs.append(h)
            out["o"][b, t] = torch.einsum("hvk,hk->hv", h, q64[b, t]) + D64[:, None] * v64[b, t]
        out["h"][n] = h
        if do is None:
            continue
        G = torch.zeros_like(h) if dh is None else size(dh[n].double())
        for t in range(e - 1, a - 1, -1):
            G = G + do64[b, t][:, :, None] * q64[b, t][:, None]
            Gk = torch.einsum("hvk,hk->hv", G, k64[b, t])
            out["dq"][b, t] = torch.einsum("hvk,hv->hk", hs[t - a + 1], do64[b, t])
            out["dv"][b, t] = dts[b, t][:, None] * Gk + D64[:, None] * do64[b, t]
            out["dk"][b, t] = dts[b, t][:, None] * torch.einsum("hvk,hv->hk", G, v64[b, t])
            dlf = f_all[b, t] * (G * hs[t - a]).sum((-1, -2))
            out["dlf"][b, t] = dlf
            direct = (v64[b, t] * Gk).sum(-1)
            out["dgt"][b, t] = slope[b, t] * (direct + g64 * dlf if magnitude else direct - g64 * dlf)
            G = f_all[b, t][:, None, None] * G
        out["dh0"][n] = G
    if do is not None:
        fold = lambda x: x.unflatten(2, (Hq, rep)).sum(3)
        out["dq"], out["dk"] = fold(out["dq"]), fold(out["dk"])
        out["dg"] = (dts * out["dlf"]).sum((0, 1)) * (1 if magnitude else -1)
        out["dD"] = (do64 * v64 * _inside(seqs, B, T)[:, :, None, None]).sum((0, 1, 3))
        out["dgt_bias"] = out["dgt"].sum((0, 1))
    return out


def _inside(seqs, B, T):
    m = torch.zeros(B, T, dtype=torch.float64)
    for b, a, e in seqs:
        m[b, a:e] = 1
    return m


def short_conv(x, weight, bias=None, silu=True, state=None, cu=None):
    """Differentiable, in x's own precision (hand in 64 bits).  Returns (y, last)."""
    B, T, D = x.shape
    W = weight.shape[-1]
    seqs = [(b, 0, T) for b in range(B)] if cu is None else [(0, int(a), int(e)) for a, e in zip(cu[:-1], cu[1:])]
    rows = [[torch.zeros(D, dtype=x.dtype)] * T for _ in range(B)]
    last = []
    for n, (b, a, e) in enumerate(seqs):
        front = torch.zeros(W - 1, D, dtype=x.dtype) if state is None else state[n].T
        full = torch.cat([front, x[b, a:e]])
        for t in range(a, e):
            p = (full[t - a:t - a + W] * weight.T).sum(0)
            if bias is not None:
                p = p + bias
            rows[b][t] = p * torch.sigmoid(p) if silu else p
        last.append(full[full.shape[0] - (W - 1):].T)
    y = torch.stack([torch.stack(r) if r else torch.zeros(0, D, dtype=x.dtype) for r in rows]) if B else x.clone()
    return y, torch.stack(last) if last else x.new_zeros(0, D, W - 1)


def rms_norm(z, weight, eps):
    return z * weight / torch.sqrt(z.square().mean(-1, keepdim=True) + eps)


def quantised(y, block, int8):
    """(q as values, scale) of y in 64 bits."""
    D = y.shape[-1]
    top = 127.0 if int8 else 448.0
    b = block or D
    pad = (-D) % b
    a = torch.cat([y.abs(), y.new_zeros(*y.shape[:-1], pad)], -1).unflatten(-1, (-1, b)).amax(-1)
    s = (torch.clamp(a, min=2.0 ** -100) / top).float()
    t = y / s.double().repeat_interleave(b, -1)[..., :D]
    if int8:
        return torch.clamp(torch.round(t), -127, 127), s
    _, e = torch.frexp(t.abs())
    step = torch.ldexp(torch.ones_like(t), torch.clamp(e - 1, min=-6) - 3)
    return torch.clamp(torch.round(t / step) * step, -448, 448), s
