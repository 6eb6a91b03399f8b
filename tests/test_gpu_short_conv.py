"""short_conv / short_conv_step against the 64-bit form.

Bounds: W + 1 <= 5 products and sums of 2^-24 each relative to the magnitudes, the sigmoid to 2^-20 (16-bit types take it from
approximate instructions, 2^-21 each; float32 from correctly rounded ones), slope of x sigmoid(x) below 1.1; then eps/2 of the
result, 2^-25 in any case in float16, whose steps are 2^-24 below 2^-14 (TINY).  Weight gradients sum n tokens in float32 runs of at most 64 * 4, then one per run: (n / 256 + 300) 2^-24 of the magnitudes,
their terms as exact as dp.
"""
import pytest
import torch

from oracle import block_oracle as bo

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}

TINY = {torch.float32: 1e-30, torch.bfloat16: 1e-30, torch.float16: 2.0 ** -25}


def make(seed, B, T, D, W, dtype, bias=True, state=True, n=None):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    n = B if n is None else n
    return dict(x=r(B, T, D).to(dtype), weight=r(D, W) / 2, bias=r(D) if bias else None,
                state=r(n, D, W - 1).to(dtype) if state else None, dy=r(B, T, D).to(dtype), dlast=r(n, D, W - 1).to(dtype))


def check(d, silu=True, cu=None, dlast=True):
    from palimpsa_b200.layers import short_conv
    dtype = d["x"].dtype
    names = [n for n in ("x", "weight", "bias", "state") if d[n] is not None]
    ref_in = {n: d[n].double().requires_grad_(True) for n in names}
    y, last = bo.short_conv(ref_in["x"], ref_in["weight"], ref_in.get("bias"), silu, ref_in.get("state"), cu)
    loss = (y * d["dy"].double()).sum() + ((last * d["dlast"].double()).sum() if dlast else 0)
    ref = dict(zip(names, torch.autograd.grad(loss, [ref_in[n] for n in names], allow_unused=True, materialize_grads=True)))
    x = {n: d[n].to(DEV).requires_grad_(True) for n in names}
    cut = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=DEV)
    gy, glast = short_conv(x["x"], x["weight"], x.get("bias"), activation="silu" if silu else None, initial_state=x.get("state"),
                           output_final_state=True, cu_seqlens=cut)
    outs, cot = ([gy, glast], [d["dy"].to(DEV), d["dlast"].to(DEV)]) if dlast else ([gy], [d["dy"].to(DEV)])
    got = dict(zip(names, torch.autograd.grad(outs, [x[n] for n in names], cot, allow_unused=True)))
    torch.cuda.synchronize()
    assert gy.dtype == dtype and torch.equal(glast.detach().cpu(), last.detach().to(dtype))
    # magnitudes: the same sums over absolute values, without the activation's slope (below 1.1)
    p_mag = bo.short_conv(d["x"].double().abs(), d["weight"].double().abs(), None if d["bias"] is None else d["bias"].double().abs(), False,
                          None if d["state"] is None else d["state"].double().abs(), cu)[0]
    fine = 16 * 2.0 ** -24 + (2.0 ** -19 if dtype != torch.float32 else 2.0 ** -22)
    half = HALF[dtype]
    assert ((gy.detach().cpu().double() - y).abs() <= fine * (p_mag + 1) + half * y.abs() + TINY[dtype]).all()
    W = d["weight"].shape[1]
    rel = fine * (2 + p_mag.max()) * 4
    for n in names:
        assert got[n].dtype == x[n].dtype and got[n].shape == x[n].shape
        if n in ("x", "state"):
            mag = 1.1 * W * d["dy"].double().abs().max() * d["weight"].double().abs().max() + d["dlast"].double().abs().max()
            bound = rel * mag + half * ref[n].abs() + TINY[dtype]
        else:
            tokens = d["x"].shape[0] * d["x"].shape[1]
            big = max(1.0, float(d["x"].double().abs().max()), float(d["state"].double().abs().max()) if d["state"] is not None else 0)
            mag = 1.1 * d["dy"].double().abs().sum((0, 1)).max() * (big if n == "weight" else 1.0)
            bound = (rel + (tokens / 256 + 300) * 2.0 ** -24) * mag
        err = (got[n].cpu().double() - ref[n]).abs()
        assert (err <= bound + 1e-30).all(), (n, float((err / (bound + 1e-30)).max()))


@pytest.mark.parametrize("shape", [(2, 37, 64, 4), (1, 1, 8, 4), (3, 5, 31, 3), (1, 300, 257, 2), (2, 130, 1792, 4), (1, 2, 40, 4), (1, 70, 1, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_forward_and_backward(shape, dtype):
    check(make(1, *shape, dtype))


@pytest.mark.parametrize("bias,state,silu", [(False, False, True), (True, False, False), (False, True, False)])
def test_optional_parts(bias, state, silu):
    check(make(2, 2, 50, 24, 4, torch.bfloat16, bias=bias, state=state), silu=silu, dlast=state)


@pytest.mark.parametrize("cu", [[0, 1, 1, 3, 40, 100], [0, 0, 0], [7, 30, 90], [0] + list(range(2, 100, 3)) + [100], [0, 100]])
@pytest.mark.parametrize("dtype,D", [(torch.float32, 12), (torch.bfloat16, 64)])
def test_packed(cu, dtype, D):
    d = make(3, 1, 100, D, 4, dtype, n=len(cu) - 1)
    check(d, cu=cu)
    from palimpsa_b200.layers import short_conv
    y = short_conv(d["x"].to(DEV), d["weight"].to(DEV), cu_seqlens=torch.tensor(cu, device=DEV))
    assert not y[0, :cu[0]].any() and not y[0, cu[-1]:].any()


def test_many_sequences_and_long_rows():
    """More sequences than one look-up step tells apart; stretches of several lengths."""
    cu = sorted(torch.randint(0, 4000, (1500,), generator=torch.Generator().manual_seed(4)).tolist())
    cu = [0] + cu + [4000]
    d = make(4, 1, 4000, 8, 3, torch.float32, n=len(cu) - 1)
    check(d, cu=cu)
    check(make(5, 1, 20000, 4, 4, torch.float32, state=False), dlast=False)


def test_rows_apart_and_weight_layouts():
    from palimpsa_b200.layers import short_conv, short_conv_step
    d = {n: t.to(DEV) for n, t in make(6, 2, 40, 48, 4, torch.bfloat16).items()}
    base = short_conv(d["x"], d["weight"], d["bias"], initial_state=d["state"])
    wide = torch.cat([d["x"][..., :8], d["x"], d["x"][..., :3]], -1)
    assert torch.equal(short_conv(wide[..., 8:56], d["weight"], d["bias"], initial_state=d["state"]), base)
    assert torch.equal(short_conv(d["x"].transpose(1, 2).contiguous().transpose(1, 2), d["weight"], d["bias"], initial_state=d["state"]), base)
    assert torch.equal(short_conv(d["x"], d["weight"][:, None], d["bias"], "swish", initial_state=d["state"]), base)
    w16 = d["weight"].bfloat16().requires_grad_(True)
    y = short_conv(d["x"], w16, d["bias"])
    assert torch.autograd.grad(y.sum(), w16)[0].dtype == torch.bfloat16
    state = d["state"].clone()
    y = torch.stack([short_conv_step(wide[:, t, 8:56], d["weight"], state, d["bias"]) for t in range(40)], 1)
    assert torch.equal(y, base)
    assert torch.equal(state, short_conv(d["x"], d["weight"], d["bias"], output_final_state=True)[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,D,W", [(1, 5, 2), (3, 1792, 4), (130, 64, 3)])
def test_single_tokens(N, D, W, dtype):
    from palimpsa_b200.layers import short_conv, short_conv_step
    d = {n: t.to(DEV) for n, t in make(7, N, 3, D, W, dtype).items()}
    want, last = short_conv(d["x"], d["weight"], d["bias"], initial_state=d["state"], output_final_state=True)
    state, version = d["state"].clone(), None
    version = state._version
    for t in range(3):
        y = short_conv_step(d["x"][:, t:t + 1], d["weight"], state, d["bias"])
        assert torch.equal(y[:, 0], want[:, t])
    assert torch.equal(state, last) and state._version > version


def test_graphs_repeats_and_empty_calls():
    from palimpsa_b200.layers import short_conv, short_conv_step
    d = {n: t.to(DEV) for n, t in make(8, 2, 600, 96, 4, torch.bfloat16).items()}
    w = d["weight"].requires_grad_(True)

    def grads():
        y = short_conv(d["x"].detach().requires_grad_(True), w, d["bias"])
        return torch.autograd.grad(y, w, d["dy"])[0]

    ref = grads()
    assert torch.equal(ref, grads())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads()
    torch.cuda.current_stream().wait_stream(side)
    state = d["state"].clone()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        out = grads()
    with torch.cuda.graph(g2):
        y = short_conv_step(d["x"][:, 0], w, state, d["bias"])
    out.zero_()
    g1.replay()
    assert torch.equal(out, ref)
    other = d["state"].clone()
    for _ in range(2):
        g2.replay()
        assert torch.equal(y, short_conv_step(d["x"][:, 0], w, other, d["bias"]))
    assert torch.equal(state, other)
    for shape in ((0, 4, 8), (2, 0, 8)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        wt = torch.ones(8, 4, device=DEV, requires_grad=True)
        st = torch.randn(shape[0], 8, 3, device=DEV, requires_grad=True)
        y, last = short_conv(x, wt, initial_state=st, output_final_state=True)
        assert y.shape == x.shape and torch.equal(last, st if shape[1] == 0 else last)
        gx, gw, gs = torch.autograd.grad([y, last], [x, wt, st], [torch.ones_like(y), torch.ones_like(last)])
        assert gx.shape == x.shape and not gw.any() and torch.equal(gs, torch.ones_like(gs))
    assert short_conv_step(torch.zeros(0, 8, device=DEV), torch.ones(8, 4, device=DEV), torch.zeros(0, 8, 3, device=DEV)).shape == (0, 8)


def test_argument_errors():
    from palimpsa_b200.layers import short_conv, short_conv_step
    x, w = torch.randn(2, 6, 8, device=DEV), torch.randn(8, 4, device=DEV)
    for bad in (dict(weight=w[:7]), dict(weight=torch.randn(8, 5, device=DEV)), dict(weight=torch.randn(8, 1, device=DEV)),
                dict(bias=w[:7, 0]), dict(initial_state=torch.zeros(2, 8, 4, device=DEV)), dict(cu_seqlens=torch.tensor([0, 6], device=DEV)),
                dict(x=x[0])):
        with pytest.raises(ValueError):
            short_conv(**{**dict(x=x, weight=w), **bad})
    with pytest.raises(TypeError):
        short_conv(x.double(), w)
    for state in (torch.zeros(2, 8, 3, device=DEV).bfloat16(), torch.zeros(2, 3, 8, device=DEV).transpose(1, 2), torch.zeros(1, 8, 3, device=DEV)):
        with pytest.raises(ValueError):
            short_conv_step(x[:, 0], w, state)
    with pytest.raises(ValueError, match="one token"):
        short_conv_step(x, w, torch.zeros(2, 8, 3, device=DEV))
    with pytest.raises(RuntimeError, match="second derivatives"):
        w.requires_grad_(True)
        torch.autograd.grad(short_conv(x, w).sum(), w, create_graph=True)
