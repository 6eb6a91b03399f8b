"""Cases of the operators that a state-space or Palimpsa block needs around its recurrence, and their plain forms.

``kind`` names the operator and its form:

    scan        ``chunk_ssm``: the selective state space scan over a prompt or a batch (``train``: forward and backward)
    scan_step   ``ssm_step``: one token for each of N running sequences, on the in-place state cache
    conv        ``short_conv``: the causal depthwise convolution in front of the scan (``train``: forward and backward)
    conv_step   ``short_conv_step``: one token for each of N running sequences
    norm        ``add_rms_norm``: residual addition and RMS norm, forward and backward
    norm_quant  ``add_rms_norm_quant``: the same with an output in 8 bits and its scales

With ``own`` the calls go to the package's entry points; without, ``run`` computes the same in elementary torch operations.
Head shapes are those of the shipped configurations (48x96 and 96x192 with 16 heads), of the tests (31x65, 64x64) or
generic (128x64); ``Hq`` is the number of heads of q and k, shared by the ``H`` heads of v.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
Q8 = {"e4m3": (torch.float8_e4m3fn, 448.0), "int8": (torch.int8, 127.0)}
DEV = "cuda"
EPS = 1e-5


def listed():
    return [
        # a short prompt before decoding, 170M heads; its length is no multiple of anything
        dict(name="scan_prompt_short", kind="scan", B=1, T=37, H=16, Hq=1, K=48, V=96, dtype="bf16", train=False, packed=False),
        # prompts of a few thousand tokens, final state handed to the decode cache
        dict(name="scan_prefill", kind="scan", B=2, T=3001, H=32, Hq=1, K=128, V=64, dtype="bf16", train=False, packed=False),
        # a training step of a state-space layer, one q/k head for all value heads
        dict(name="scan_train", kind="scan", B=8, T=2048, H=24, Hq=1, K=128, V=64, dtype="bf16", train=True, packed=False),
        # packed documents, 170M heads with a q/k head each
        dict(name="scan_train_packed", kind="scan", B=1, T=16384, H=16, Hq=16, K=48, V=96, dtype="bf16", train=True, packed=True),
        # the odd shape of the check script in float32
        dict(name="scan_train_fp32_odd", kind="scan", B=2, T=511, H=4, Hq=2, K=31, V=65, dtype="fp32", train=True, packed=False),
        # a server's decode step: 201 MB of state read and written per token
        dict(name="scan_step_serving", kind="scan_step", N=256, H=24, Hq=1, K=128, V=64, dtype="bf16"),
        # the convolution over the concatenated x, B, C channels of the training step above, twice as long
        dict(name="conv_train", kind="conv", B=8, T=4096, D=1792, W=4, dtype="bf16", train=True, packed=False, silu=True),
        # packed documents, odd channel count and width, float32
        dict(name="conv_train_packed", kind="conv", B=1, T=8191, D=777, W=3, dtype="fp32", train=True, packed=True, silu=True),
        # a few users' next token: nothing but latency
        dict(name="conv_step", kind="conv_step", N=3, D=1792, W=4, dtype="bf16"),
        # the block's norm in a training step, float32 residual stream
        dict(name="norm_train", kind="norm", rows=32768, D=768, dtype="bf16", res="fp32"),
        # decode batch: one scale per token
        dict(name="norm_quant_rows", kind="norm_quant", rows=61, D=2048, dtype="bf16", res="bf16", block=0, q8="e4m3"),
        # prefill: one scale per token and 128 channels
        dict(name="norm_quant_blocks", kind="norm_quant", rows=16384, D=2048, dtype="bf16", res="bf16", block=128, q8="e4m3"),
    ]


HEADS = [(48, 48), (48, 96), (96, 192), (64, 64), (128, 64), (128, 128), (31, 65), (16, 32)]
MAX_SCAN = 8 * 2048 * 24 * 128 * 64 / 2   # tokens x heads x state elements of a drawn bf16 scan: half of the largest listed one
MAX_STATE = 256 * 24 * 128 * 64           # state elements of a drawn decode step
MAX_CONV = 8 * 4096 * 1792                # elements of a drawn convolution
MAX_NORM = 32768 * 1024                   # elements of a drawn norm


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["scan", "scan", "scan", "scan_step", "conv", "conv_step", "norm", "norm_quant"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    if kind in ("scan", "scan_step"):
        K, V = rng.choice(HEADS) if rng.random() < 0.75 else (rng.randint(4, 160), rng.randint(4, 200))
        H = rng.choice([1, 2, 4, 6, 8, 12, 16, 24])
        Hq = rng.choice([h for h in (1, 2, H // 2, H) if h and H % h == 0])
        c = dict(kind=kind, H=H, Hq=Hq, K=K, V=V, dtype=dtype)
        if kind == "scan_step":
            c["N"] = _log(rng, 1, max(1, min(512, MAX_STATE // (H * K * V))))
            return c
        top = MAX_SCAN / (H * K * V) / (1 if dtype == "bf16" else 8)
        T = _log(rng, 1, max(1, min(8192, int(top))))
        c.update(train=rng.random() < 0.6, packed=rng.random() < 0.3)
        c.update(B=1 if c["packed"] else _log(rng, 1, max(1, min(32, int(top / T)))), T=T)
        return c
    if kind == "conv":
        D, W = _log(rng, 16, 4096), rng.choice([2, 3, 4, 4, 4])
        T = _log(rng, 1, min(16384, MAX_CONV // D))
        packed = rng.random() < 0.3
        return dict(kind=kind, B=1 if packed else _log(rng, 1, max(1, min(16, MAX_CONV // (D * T)))), T=T, D=D, W=W,
                    dtype=dtype, train=rng.random() < 0.6, packed=packed, silu=rng.random() < 0.8)
    if kind == "conv_step":
        return dict(kind=kind, N=_log(rng, 1, 1024), D=_log(rng, 16, 8192), W=rng.choice([2, 3, 4, 4, 4]), dtype=dtype)
    D = _log(rng, 32, 8192)
    rows = _log(rng, 1, MAX_NORM // D)
    res = rng.choice([dtype, "fp32", ""])
    if kind == "norm":
        return dict(kind=kind, rows=rows, D=D, dtype=dtype, res=res)
    return dict(kind=kind, rows=rows, D=D, dtype=dtype, res=res, block=rng.choice([0, 0, 128]),
                q8=rng.choice(["e4m3", "e4m3", "int8"]))


def _documents(T):
    return max(2, T // 400)


def _offsets(T, gen):
    """A row of T tokens as documents whose lengths differ by factors of up to 256; the first is empty."""
    n = _documents(T)
    weight = torch.exp(torch.rand(n - 1, generator=gen, device=DEV) * math.log(256.0)).tolist()
    ends, total, run_sum = [0, 0], sum(weight), 0.0
    for w in weight:
        run_sum += w
        ends.append(min(T, int(run_sum / total * T)))
    ends[-1] = T
    return torch.tensor(ends, dtype=torch.int32, device=DEV), max(b - a for a, b in zip(ends, ends[1:]))


def _silu(x):
    return x / (1 + torch.exp(-x))


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    io = DTYPES[case["dtype"]]
    kind = case["kind"]

    def randn(*s):
        return torch.randn(*s, generator=gen, device=DEV)

    def rand(*s):
        return torch.rand(*s, generator=gen, device=DEV)

    st = dict(case=case)
    if kind in ("scan", "scan_step"):
        B, T = (case["N"], 1) if kind == "scan_step" else (case["B"], case["T"])
        H, Hq, K, V = case["H"], case["Hq"], case["K"], case["V"]
        # outputs of the convolution and its SiLU, one row per token: x, B and C side by side, as the layer splits them
        xbc = _silu(randn(B, T, H * V + 2 * Hq * K)).to(io)
        v, k, q = xbc.split([H * V, Hq * K, Hq * K], dim=-1)
        st.update(q=q.unflatten(-1, (Hq, K)), k=k.unflatten(-1, (Hq, K)), v=v.unflatten(-1, (H, V)))
        st["gt"] = (0.5 * randn(B, T, H)).to(io)
        dt0 = torch.exp(rand(H) * (math.log(0.1) - math.log(1e-3)) + math.log(1e-3))
        st["gt_bias"] = dt0 + torch.log(-torch.expm1(-dt0))
        st["g"] = 1 + 15 * rand(H)
        st["D"] = 1 + 0.1 * randn(H)
        if kind == "scan_step":
            st["state"] = 0.3 * randn(B, H, V, K)
            return st
        st["cu"], st["longest"] = _offsets(T, gen) if case["packed"] else (None, T)
        n = st["cu"].numel() - 1 if case["packed"] else B
        st["h0"] = 0.3 * randn(n, H, V, K)
        if case["train"]:
            st["do"] = randn(B, T, H, V).to(io)
            st["dh"] = 0.1 * randn(n, H, V, K)
            for name in ("q", "k", "v", "gt", "gt_bias", "g", "D", "h0"):
                st[name] = st[name].detach().requires_grad_(True)
        return st
    if kind == "conv":
        B, T, D, W = case["B"], case["T"], case["D"], case["W"]
        st["x"] = randn(B, T, D).to(io)
        st["weight"] = randn(D, W) / math.sqrt(W)
        st["bias"] = 0.1 * randn(D)
        st["cu"], st["longest"] = _offsets(T, gen) if case["packed"] else (None, T)
        n = st["cu"].numel() - 1 if case["packed"] else B
        st["s0"] = randn(n, D, W - 1).to(io)
        if case["train"]:
            st["dy"] = randn(B, T, D).to(io)
            for name in ("x", "weight", "bias"):
                st[name].requires_grad_(True)
        return st
    if kind == "conv_step":
        N, D, W = case["N"], case["D"], case["W"]
        st.update(x=randn(N, D).to(io), weight=randn(D, W) / math.sqrt(W), bias=0.1 * randn(D), state=randn(N, D, W - 1).to(io))
        return st
    rows, D = case["rows"], case["D"]
    st["x"] = randn(rows, D).to(io)
    st["res"] = (3 * randn(rows, D)).to(DTYPES[case["res"]]) if case["res"] else None
    st["weight"] = 1 + 0.1 * randn(D)
    if kind == "norm":
        st["dy"] = randn(rows, D).to(io)
        st["dz"] = randn(rows, D).to(DTYPES[case["res"]]) if case["res"] else None
        for name in ("x", "weight", "res"):
            if st[name] is not None:
                st[name].requires_grad_(True)
    return st


# ---- plain forms -------------------------------------------------------------------------------------------------
def _pad_index(cu, T, longest):
    """Row of the packed batch for every (sequence, position), and which of them exist."""
    first, last = cu[:-1].long(), cu[1:].long()
    idx = first[:, None] + torch.arange(longest, device=cu.device)[None]
    return idx.clamp(max=T - 1), idx < last[:, None]


def _to_padded(x, idx, live):
    return x[0][idx] * live.reshape(*live.shape, *([1] * (x.dim() - 2))).to(x.dtype)


def _from_padded(x, cu, T):
    row = torch.arange(T, device=x.device)
    seq = torch.searchsorted(cu.long(), row, right=True) - 1
    return x[seq, row - cu.long()[seq]][None]


def _scan_plain(q, k, v, gt, gt_bias, g, D, h0, Q=64):
    """Chunks of Q tokens; log decays are summed in 64 bits, everything else is 32."""
    B, T, H, V = v.shape
    Hq, K = q.shape[2:]
    u = gt + gt_bias
    dt = torch.where(u > 20, u, torch.log1p(torch.exp(torch.clamp(u, max=20.0))))
    return _scan_chunks(q, k, v, dt, g, D, h0, Q)


def _scan_chunks(q, k, v, dt, g, D, h0, Q):
    B, T, H, V = v.shape
    Hq, K = q.shape[2:]
    pad = (-T) % Q
    n = (T + pad) // Q

    def cut(x):
        x = torch.cat([x, x.new_zeros(B, pad, *x.shape[2:])], 1) if pad else x
        return x.reshape(B, n, Q, *x.shape[2:])

    qc, kc, vc, dc = cut(q), cut(k), cut(v), cut(dt)
    L = torch.cumsum((dc * -g).double(), 2)
    low = torch.tril(torch.ones(Q, Q, dtype=torch.bool, device=q.device))[None, None, :, :, None]
    gap = torch.where(low, L[:, :, :, None] - L[:, :, None], torch.zeros((), dtype=L.dtype, device=L.device))
    dec = torch.where(low, torch.exp(gap).float(), torch.zeros((), device=q.device))              # B n Q Q H
    S = torch.einsum("bnihk,bnjhk->bnijh", qc, kc).repeat_interleave(H // Hq, -1)
    o = torch.einsum("bnijh,bnjhv->bnihv", S * dec * dc[:, :, None], vc)
    w = torch.exp(L[:, :, -1:] - L).float() * dc
    kH, qH = kc.repeat_interleave(H // Hq, 3), qc.repeat_interleave(H // Hq, 3)
    local = torch.einsum("bnjhv,bnjhk->bnhvk", vc * w[..., None], kH)
    total = torch.exp(L[:, :, -1]).float()
    h, starts = h0, []
    for c in range(n):
        starts.append(h)
        h = h * total[:, c, :, None, None] + local[:, c]
    inter = torch.einsum("bnihk,bnhvk->bnihv", qH, torch.stack(starts, 1)) if n else o
    o = o + inter * torch.exp(L).float()[..., None] + vc * D[:, None]
    return o.reshape(B, n * Q, H, V)[:, :T], h


def _conv_plain(x, weight, bias, s0, silu):
    """x [B,T,D]; s0 [B,D,W-1]: the inputs in front of the first token."""
    W = weight.shape[1]
    full = torch.cat([s0.transpose(1, 2), x], 1)
    T = x.shape[1]
    y = bias + sum(full[:, w:w + T] * weight[:, w] for w in range(W))
    return _silu(y) if silu else y


def _conv_last(x, s0, lens):
    """The last W-1 inputs of every sequence, [B,D,W-1]; lens [B]."""
    W1 = s0.shape[2]
    full = torch.cat([s0.transpose(1, 2), x], 1)
    idx = lens[:, None] + torch.arange(W1, device=x.device)[None]
    return full[torch.arange(x.shape[0], device=x.device)[:, None], idx].transpose(1, 2)


def _round_8(t, kind):
    """Nearest 8-bit value, ties to even, of a 64-bit t."""
    if kind == "int8":
        return torch.clamp(torch.round(t), -127, 127)
    _, e = torch.frexp(t.abs())
    quantum = torch.ldexp(torch.ones_like(t), torch.clamp(e - 1, min=-6) - 3)
    return torch.clamp(torch.round(t / quantum) * quantum, -448, 448)


def _scales(y, block, top):
    """Per row, or per row and block of channels: the largest value over the type's largest."""
    D = y.shape[1]
    b = block or D
    pad = (-D) % b
    a = y.abs()
    a = torch.cat([a, a.new_zeros(a.shape[0], pad)], 1) if pad else a
    s = (torch.clamp(a.reshape(a.shape[0], -1, b).amax(-1), min=2.0 ** -100) / top).float()
    return s, s.repeat_interleave(b, 1)[:, :D]


def _run_plain(st):
    case = st["case"]
    kind = case["kind"]
    io = DTYPES[case["dtype"]]
    if kind == "scan":
        q, k, v, gt = (st[n].float() for n in ("q", "k", "v", "gt"))
        T = case["T"]
        if case["packed"]:
            idx, live = _pad_index(st["cu"], T, st["longest"])
            q, k, v, gt = (_to_padded(x, idx, live) for x in (q, k, v, gt))
            u = gt + st["gt_bias"]
            dt = torch.where(u > 20, u, torch.log1p(torch.exp(torch.clamp(u, max=20.0)))) * live[..., None]
            o, h = _scan_chunks(q, k, v, dt, st["g"], st["D"], st["h0"], 64)
            o = _from_padded(o, st["cu"], T)
        else:
            o, h = _scan_plain(q, k, v, gt, st["gt_bias"], st["g"], st["D"], st["h0"])
        o = o.to(io)
        if not case["train"]:
            return [o, h]
        leaves = [st[n] for n in ("q", "k", "v", "gt", "gt_bias", "g", "D", "h0")]
        return [o, h, *torch.autograd.grad([o, h], leaves, [st["do"], st["dh"]])]
    if kind == "scan_step":
        q, k, v, gt = (st[n][:, 0].float() for n in ("q", "k", "v", "gt"))
        r = case["H"] // case["Hq"]
        q, k = q.repeat_interleave(r, 1), k.repeat_interleave(r, 1)
        u = gt + st["gt_bias"]
        dt = torch.where(u > 20, u, torch.log1p(torch.exp(torch.clamp(u, max=20.0))))
        f = torch.exp(-st["g"] * dt)
        new = st["state"] * f[..., None, None] + (dt[..., None] * v)[..., None] * k[:, :, None]
        st["state"].copy_(new)
        o = (new * q[:, :, None]).sum(-1) + st["D"][:, None] * v
        return [o[:, None].to(io), st["state"]]
    if kind == "conv":
        x, weight, bias, s0 = st["x"].float(), st["weight"], st["bias"], st["s0"].float()
        B, T = case["B"], case["T"]
        if case["packed"]:
            idx, live = _pad_index(st["cu"], T, st["longest"])
            xp = _to_padded(x, idx, live)
            y = _from_padded(_conv_plain(xp, weight, bias, s0, case["silu"]), st["cu"], T)
            last = _conv_last(xp, s0, live.sum(1))
        else:
            y = _conv_plain(x, weight, bias, s0, case["silu"])
            last = _conv_last(x, s0, torch.full((B,), T, device=x.device))
        y, last = y.to(io), last.detach().to(io)
        if not case["train"]:
            return [y, last]
        return [y, last, *torch.autograd.grad(y, [st["x"], weight, bias], st["dy"])]
    if kind == "conv_step":
        x, state = st["x"].float(), st["state"].float()
        full = torch.cat([state, x[..., None]], -1)
        y = _silu((full * st["weight"]).sum(-1) + st["bias"]).to(io)
        st["state"].copy_(full[..., 1:])
        return [y, st["state"]]
    x, res, weight = st["x"], st["res"], st["weight"]
    if kind == "norm":
        z = x if res is None else (x.float() + res.float()).to(res.dtype)
        zf = z.float()
        y = (zf * torch.rsqrt((zf * zf).mean(-1, keepdim=True) + EPS) * weight).to(io)
        outs, grads = ([y], [st["dy"]]) if res is None else ([y, z], [st["dy"], st["dz"]])
        leaves = [t for t in (x, res, weight) if t is not None]
        return [*outs, *torch.autograd.grad(outs, leaves, grads)]
    # values next to a rounding border: 64 bits until the 8-bit value is known
    top = Q8[case["q8"]][1]
    z = x if res is None else (x.float() + res.float()).to(res.dtype)
    zd = z.double()
    y = zd * weight.double() / torch.sqrt((zd * zd).mean(-1, keepdim=True) + EPS)
    s, each = _scales(y, case["block"], top)
    q8 = _round_8(y / each.double(), case["q8"]).float()
    return [q8 * each, s] if res is None else [q8 * each, s, z]


# ---- the package's calls -----------------------------------------------------------------------------------------
def _run_own(st):
    from palimpsa_b200.layers import add_rms_norm, add_rms_norm_quant, short_conv, short_conv_step
    from palimpsa_b200.ops import chunk_ssm, ssm_step
    case = st["case"]
    kind = case["kind"]
    if kind == "scan":
        o, h = chunk_ssm(st["q"], st["k"], st["v"], st["gt"], st["g"], D=st["D"], gt_bias=st["gt_bias"], gt_softplus=True,
                         initial_state=st["h0"], output_final_state=True, cu_seqlens=st["cu"])
        if not case["train"]:
            return [o, h]
        leaves = [st[n] for n in ("q", "k", "v", "gt", "gt_bias", "g", "D", "h0")]
        return [o, h, *torch.autograd.grad([o, h], leaves, [st["do"], st["dh"]])]
    if kind == "scan_step":
        o = ssm_step(st["q"], st["k"], st["v"], st["gt"], st["g"], st["state"], D=st["D"], gt_bias=st["gt_bias"], gt_softplus=True)
        return [o, st["state"]]
    if kind == "conv":
        y, last = short_conv(st["x"], st["weight"], st["bias"], activation="silu" if case["silu"] else None,
                             initial_state=st["s0"], output_final_state=True, cu_seqlens=st["cu"])
        if not case["train"]:
            return [y, last]
        return [y, last, *torch.autograd.grad(y, [st["x"], st["weight"], st["bias"]], st["dy"])]
    if kind == "conv_step":
        y = short_conv_step(st["x"], st["weight"], st["state"], st["bias"], activation="silu")
        return [y, st["state"]]
    x, res, weight = st["x"], st["res"], st["weight"]
    if kind == "norm":
        y, z = add_rms_norm(x, weight, residual=res, eps=EPS)
        outs, grads = ([y], [st["dy"]]) if res is None else ([y, z], [st["dy"], st["dz"]])
        leaves = [t for t in (x, res, weight) if t is not None]
        return [*outs, *torch.autograd.grad(outs, leaves, grads)]
    q8, s, z = add_rms_norm_quant(x, weight, residual=res, eps=EPS, dtype=Q8[case["q8"]][0], block=case["block"] or None)
    values = q8.float() * s.repeat_interleave(case["block"] or case["D"], 1)[:, :case["D"]]   # what the 8 bits stand for
    return [values, s] if res is None else [values, s, z]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- from the definitions, in 64 bits ------------------------------------------------------------------------------
def _scan_exact(q, k, v, dt, g, D, h0, do=None, dh=None):
    """Token by token.  q, k with a head per value head, all 64 bits.  With do and dh: the gradients of
    (q, k, v, dt, g, D, h0) too, from the adjoint recurrence over states recomputed block by block."""
    T = v.shape[1]
    f = torch.exp(-g * dt)
    step = 32
    h, outs, marks = h0, [], []
    for t in range(T):
        if t % step == 0:
            marks.append(h)
        h = h * f[:, t, :, None, None] + (dt[:, t, :, None] * v[:, t])[..., None] * k[:, t, :, None]
        outs.append((h @ q[:, t, :, :, None])[..., 0] + D[:, None] * v[:, t])
    o = torch.stack(outs, 1) if outs else torch.zeros_like(v)
    if do is None:
        return o, h
    dq, dk, dv, ddt, df = (torch.zeros_like(x) for x in (q, k, v, dt, dt))
    G = dh.clone()
    for b in range(len(marks) - 1, -1, -1):
        states = [marks[b]]
        ts = range(b * step, min(T, (b + 1) * step))
        for t in ts:
            states.append(states[-1] * f[:, t, :, None, None] + (dt[:, t, :, None] * v[:, t])[..., None] * k[:, t, :, None])
        for t in reversed(ts):
            G = G + do[:, t][..., None] * q[:, t, :, None]
            dq[:, t] = (do[:, t][..., None, :] @ states[t - b * step + 1])[..., 0, :]
            Gk = (G @ k[:, t, :, :, None])[..., 0]
            dv[:, t] = dt[:, t, :, None] * Gk + D[:, None] * do[:, t]
            dk[:, t] = dt[:, t, :, None] * (v[:, t][..., None, :] @ G)[..., 0, :]
            ddt[:, t] = (v[:, t] * Gk).sum(-1)
            df[:, t] = (G * states[t - b * step]).sum((-1, -2)) * f[:, t]
            G = G * f[:, t, :, None, None]
    ddt = ddt - g * df
    dg = -(dt * df).sum((0, 1))
    return o, h, dq, dk, dv, ddt, dg, (do * v).sum((0, 1, 3)), G


def exact(case, seed):
    st = prepare(case, seed)
    st = {n: x.detach() if isinstance(x, torch.Tensor) else x for n, x in st.items()}
    kind = case["kind"]
    d = {n: x.double() for n, x in st.items() if isinstance(x, torch.Tensor) and x.is_floating_point()}
    if kind in ("scan", "scan_step"):
        H, Hq = case["H"], case["Hq"]
        r = H // Hq
        q, k, v, gt = d["q"], d["k"], d["v"], d["gt"]
        T = q.shape[1]
        packed = kind == "scan" and case["packed"]
        live = torch.ones(q.shape[:2], dtype=torch.bool, device=DEV)
        idx = None
        if packed:
            idx, live = _pad_index(st["cu"], T, st["longest"])
            if live.numel() * H * case["K"] * case["V"] > 4e11:
                return None
            q, k, v, gt = (_to_padded(x, idx, live) for x in (q, k, v, gt))
        u = gt + d["gt_bias"]
        dt = torch.nn.functional.softplus(u, threshold=1e9) * live[..., None]
        qH, kH = q.repeat_interleave(r, 2), k.repeat_interleave(r, 2)
        if kind == "scan_step":
            o, h = _scan_exact(qH, kH, v, dt, d["g"], d["D"], d["state"])
            return [o, h]
        back = (lambda x: _from_padded(x, st["cu"], T)) if packed else (lambda x: x)
        if not case["train"]:
            o, h = _scan_exact(qH, kH, v, dt, d["g"], d["D"], d["h0"])
            return [back(o), h]
        do = _to_padded(d["do"], idx, live) if packed else d["do"]
        o, h, dq, dk, dv, ddt, dg, dD, dh0 = _scan_exact(qH, kH, v, dt, d["g"], d["D"], d["h0"], do, d["dh"])
        dgt = ddt * torch.sigmoid(u) * live[..., None]
        fold = lambda x: x.unflatten(2, (Hq, r)).sum(3)
        return [back(o), h, back(fold(dq)), back(fold(dk)), back(dv), back(dgt), dgt.sum((0, 1)), dg, dD, dh0]
    if kind in ("conv", "conv_step"):
        W = case["W"]
        weight, bias = d["weight"], d["bias"]
        if kind == "conv_step":
            win = torch.cat([d["state"], d["x"][..., None]], -1)
            pre = torch.einsum("ndw,dw->nd", win, weight) + bias
            return [pre * torch.sigmoid(pre), win[..., 1:]]
        x, T = d["x"], case["T"]
        seqs = [(0, 0, T)] if case["B"] == 1 and not case["packed"] else [(b, 0, T) for b in range(case["B"])]
        if case["packed"]:
            cu = st["cu"].tolist()
            seqs = [(0, a, e) for a, e in zip(cu[:-1], cu[1:])]
        y, last, dx = torch.zeros_like(x), torch.zeros_like(d["s0"]), torch.zeros_like(x)
        dw, db = torch.zeros_like(weight), torch.zeros_like(bias)
        for n, (b, a, e) in enumerate(seqs):
            rows = torch.cat([d["s0"][n].T, x[b, a:e]], 0)
            last[n] = rows[rows.shape[0] - (W - 1):].T
            if e == a:
                continue
            win = rows.unfold(0, W, 1)                                     # tokens, D, W
            pre = torch.einsum("tdw,dw->td", win, weight) + bias
            sg = torch.sigmoid(pre)
            y[b, a:e] = pre * sg if case["silu"] else pre
            if case["train"]:
                dpre = d["dy"][b, a:e] * (sg * (1 + pre * (1 - sg)) if case["silu"] else 1.0)
                dw += torch.einsum("tdw,td->dw", win, dpre)
                db += dpre.sum(0)
                drows = torch.zeros_like(rows)
                for w in range(W):
                    drows[w:w + e - a] += dpre * weight[:, w]
                dx[b, a:e] = drows[W - 1:]
        return [y, last, dx, dw, db] if case["train"] else [y, last]
    x, weight = d["x"], d["weight"]
    z_io = None
    if st["res"] is not None:
        z_io = (st["x"].float() + st["res"].float()).to(st["res"].dtype)
        z = z_io.double()
    else:
        z = x
    D = z.shape[1]
    rms = (z.square().sum(-1, keepdim=True) / D + EPS) ** -0.5
    if kind == "norm":
        y = z * rms * weight
        wdy = weight * d["dy"]
        dz = rms * (wdy - z * rms * rms * (wdy * z).sum(-1, keepdim=True) / D)
        dw = (d["dy"] * z * rms).sum(0)
        if z_io is None:
            return [y, dz, dw]
        dz = dz + d["dz"]
        return [y, x + d["res"], dz, dz, dw]
    return None                                  # rounded to 8 bits from 64: the plain form is the definition itself


# ---- floors ------------------------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    io = 4 if case["dtype"] == "fp32" else 2
    if kind in ("scan", "scan_step"):
        H, Hq, K, V = case["H"], case["Hq"], case["K"], case["V"]
        B, T = (case["N"], 1) if kind == "scan_step" else (case["B"], case["T"])
        n = _documents(T) if case.get("packed") else B
        tok = B * T
        fwd = tok * ((2 * H * V + 2 * Hq * K) * io + H * io) + 8 * n * H * K * V
        ops = 5.0 * tok * H * K * V
        if not case.get("train"):
            return dict(bytes=fwd, flops=ops)
        bwd = tok * ((3 * H * V + 4 * Hq * K) * io + 2 * H * io) + 8 * n * H * K * V
        return dict(bytes=fwd + bwd, flops=ops + 13.0 * tok * H * K * V)
    if kind in ("conv", "conv_step"):
        D, W = case["D"], case["W"]
        if kind == "conv_step":
            return dict(bytes=case["N"] * D * io * (2 + 2 * (W - 1)) + 4 * D * (W + 1), flops=2.0 * case["N"] * D * W)
        e = case["B"] * case["T"] * D
        f = 1 + (1.5 if case["train"] else 0)                     # x, dy read and dx written again
        return dict(bytes=2 * e * io * f + 4 * D * (W + 1), flops=2.0 * e * W * (3 if case["train"] else 1))
    e = case["rows"] * case["D"]
    res = {"": 0, "fp32": 4}.get(case["res"], 2)
    if kind == "norm":
        return dict(bytes=e * (2 * io + 2 * res + io + (io if not res else res) + 2 * res + io), flops=12.0 * e)
    return dict(bytes=e * (io + 2 * res + 1), flops=5.0 * e)
