"""add_rms_norm / add_rms_norm_quant against the 64-bit form.

Bounds: the row's sums are trees over at most 32 values a thread (relative 40 * 2^-24 of sums of magnitudes), r carries half of
that; y and the gradients take 4 more roundings; then eps/2 of the value -- and, in float16, whose steps
are 2^-24 below 2^-14, 2^-25 in any case (TINY).  dw: rows a CTA walks and CTAs, in float32.  The 8-bit values and
scales are compared exactly: they are defined in 64 bits.
"""
import pytest
import torch

from oracle import block_oracle as bo

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-30, torch.bfloat16: 1e-30, torch.float16: 2.0 ** -25}
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
WIDTHS = [1, 8, 31, 200, 256, 260, 512, 768, 1000, 1024, 1032, 2048, 2050, 4096, 5000, 8192, 10000, 16384]


def make(seed, rows, D, dtype, res):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    return dict(x=r(rows, D).to(dtype), res=None if res is None else (3 * r(rows, D)).to(res), weight=1 + 0.3 * r(D),
                dy=r(rows, D).to(dtype), dz=None if res is None else r(rows, D).to(res))


def stored_z(d):
    return d["x"] if d["res"] is None else (d["x"].float() + d["res"].float()).to(d["res"].dtype)


@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("dtype,res", [(BF, FP), (BF, BF), (FP, FP), (HF, None), (BF, None), (HF, FP)])
def test_forward_and_backward(D, dtype, res):
    from palimpsa_b200.layers import add_rms_norm
    d = make(1, 11, D, dtype, res)
    z64 = stored_z(d).double().requires_grad_(True)
    w64 = d["weight"].double().requires_grad_(True)
    y64 = bo.rms_norm(z64, w64, 1e-5)
    loss = (y64 * d["dy"].double()).sum() + (0 if res is None else (z64 * d["dz"].double()).sum())
    dz64, dw64 = torch.autograd.grad(loss, [z64, w64])
    x = {n: None if t is None else t.to(DEV).requires_grad_(n in ("x", "res", "weight")) for n, t in d.items()}
    y, z = add_rms_norm(x["x"], x["weight"], residual=x["res"])
    assert y.dtype == dtype and torch.equal(z.detach().cpu(), stored_z(d))
    outs, cot = ([y], [x["dy"]]) if res is None else ([y, z], [x["dy"], x["dz"]])
    leaves = [x[n] for n in ("x", "res", "weight") if x[n] is not None]
    got = torch.autograd.grad(outs, leaves, cot)
    fine = 80 * 2.0 ** -24
    assert ((y.detach().cpu().double() - y64).abs() <= fine * y64.abs() + HALF[dtype] * y64.abs() + TINY[dtype]).all()
    r = 1 / torch.sqrt(z64.square().mean(-1, keepdim=True) + 1e-5)
    wdy = (w64 * d["dy"].double()).abs()
    mag = r * (wdy + z64.abs() * r * r * (wdy * z64.abs()).mean(-1, keepdim=True)) + (0 if res is None else d["dz"].double().abs())
    for g, leaf in zip(got[:-1], leaves[:-1]):
        assert g.dtype == leaf.dtype
        assert ((g.cpu().double() - dz64).abs() <= 2 * fine * mag + HALF[g.dtype] * dz64.abs() + TINY[g.dtype]).all()
    dw_mag = (d["dy"].double() * z64 * r).abs().sum(0)
    assert ((got[-1].cpu().double() - dw64).abs() <= 2 * fine * dw_mag + 1e-30).all()


@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("dtype,res", [(BF, BF), (FP, FP), (HF, FP), (BF, None)])
@pytest.mark.parametrize("block", [None, 32, 128, 256])
def test_eight_bits(D, dtype, res, block):
    from palimpsa_b200.layers import add_rms_norm_quant
    d = make(2, 13, D, dtype, res)
    d["x"][3] = 0
    if res is not None:
        d["res"][3] = 0
    d["x"][5] *= 1e-3
    z = stored_z(d)
    y64 = bo.rms_norm(z.double(), d["weight"].double(), 1e-5)
    for t in (torch.float8_e4m3fn, torch.int8):
        want, scale = bo.quantised(y64, block, t == torch.int8)
        q, s, zz = add_rms_norm_quant(d["x"].to(DEV), d["weight"].to(DEV), residual=None if res is None else d["res"].to(DEV), dtype=t, block=block)
        assert q.dtype == t and s.shape == scale.shape and torch.equal(zz.cpu(), z)
        assert torch.equal(s.cpu(), scale)
        assert torch.equal(q.cpu().double() if t == torch.int8 else q.cpu().float().double(), want)


def test_values_on_the_border_between_two():
    """Rows made of 8-bit borders: every element lies on the middle between two values or a step of the type beside it."""
    from palimpsa_b200.layers import add_rms_norm_quant
    base = torch.tensor([448.0] + [1.0625, 1.1875, 1.3125, 1.4375, 1.5625, 1.6875, 1.8125, 1.9375, 17.0, 19.0, 0.0009765625, 0.0029296875] * 10)
    x = torch.stack([torch.nextafter(base, base.new_tensor(k)) for k in (0.0, 1000.0)] + [base, -base] + [base * (1 + i * 2.0 ** -23) for i in range(8)])
    w = torch.ones(x.shape[1])
    w[1::7] = 1 + 2.0 ** -23
    y64 = bo.rms_norm(x.double(), w.double(), 1e-5)
    for t in (torch.float8_e4m3fn, torch.int8):
        want, scale = bo.quantised(y64, None, t == torch.int8)
        q, s, _ = add_rms_norm_quant(x.to(DEV), w.to(DEV), dtype=t)
        assert torch.equal(s.cpu(), scale) and torch.equal(q.cpu().float().double(), want)


def test_special_values():
    from palimpsa_b200.layers import add_rms_norm, add_rms_norm_quant
    x = torch.randn(6, 300, device=DEV)
    x[1, 7] = float("nan")
    x[2, 9] = float("inf")
    x[3] = 1e-42
    x[4] = 0
    w = torch.ones(300, device=DEV)
    y, _ = add_rms_norm(x, w)
    assert y[1].isnan().all() and y[2, 9].isnan() and torch.isfinite(y[[0, 3, 4, 5]]).all() and not y[4].any()
    q, s, _ = add_rms_norm_quant(x, w)
    assert s[1].isnan().all() and s[2].isnan().all() and torch.isfinite(s[[0, 3, 4, 5]]).all() and not q[4].float().any()
    q, s, _ = add_rms_norm_quant(x, w, block=128)
    assert s[1].isnan().all() and s[2, 0].isnan() and torch.isfinite(s[2, 1:]).all()
    big = torch.full((2, 64), 3e38, device=DEV)                 # squares beyond float32: 64 bits in the 8-bit form
    q, s, _ = add_rms_norm_quant(big, torch.ones(64, device=DEV))
    assert (q.float() == 448).all() and torch.isfinite(s).all()


def test_rows_apart_shapes_repeats_graphs_and_empty():
    from palimpsa_b200.layers import add_rms_norm, add_rms_norm_quant
    wide = torch.randn(2, 5, 800, device=DEV, dtype=BF)
    x, w = wide[..., 16:784], torch.randn(768, device=DEV)
    ref = add_rms_norm(x.contiguous(), w)[0]
    assert torch.equal(add_rms_norm(x, w)[0], ref)
    assert torch.equal(add_rms_norm(wide[..., 1:769], w)[0], add_rms_norm(wide[..., 1:769].contiguous(), w)[0])
    assert torch.equal(add_rms_norm(x.transpose(0, 1), w)[0], ref.transpose(0, 1))
    assert torch.equal(add_rms_norm_quant(x, w, block=64)[1], add_rms_norm_quant(x.contiguous(), w, block=64)[1])
    assert add_rms_norm(x[0, 0], w)[0].shape == (768,)
    xl = x.contiguous().requires_grad_(True)
    wl = w.bfloat16().requires_grad_(True)
    many = torch.randn(5000, 768, device=DEV, dtype=BF).requires_grad_(True)

    def grads():
        y, _ = add_rms_norm(many, wl)
        return torch.autograd.grad(y, [many, wl], torch.ones_like(y))

    a = grads()
    assert a[1].dtype == BF and all(torch.equal(p, q) for p, q in zip(a, grads()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b = grads()
    for t in b:
        t.zero_()
    graph.replay()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    e = torch.zeros(0, 64, device=DEV, requires_grad=True)
    we = torch.ones(64, device=DEV, requires_grad=True)
    y, z = add_rms_norm(e, we, residual=e)
    assert y.shape == z.shape == (0, 64) and not torch.autograd.grad(y.sum(), we)[0].any()
    assert add_rms_norm_quant(e.detach(), we.detach(), block=32)[1].shape == (0, 2)


def test_argument_errors():
    from palimpsa_b200.layers import add_rms_norm, add_rms_norm_quant
    x, w = torch.randn(4, 64, device=DEV, dtype=BF), torch.ones(64, device=DEV)
    with pytest.raises(ValueError):
        add_rms_norm(x, w[:63])
    with pytest.raises(ValueError):
        add_rms_norm(x, w, residual=x[:3])
    with pytest.raises(TypeError):
        add_rms_norm(x, w, residual=x.half())
    with pytest.raises(ValueError):
        add_rms_norm(x, w, eps=-1.0)
    with pytest.raises(ValueError):
        add_rms_norm(torch.zeros(1, 16385, device=DEV), torch.ones(16385, device=DEV))
    with pytest.raises(RuntimeError, match="no gradient"):
        add_rms_norm_quant(x, w.clone().requires_grad_(True))
    with pytest.raises(RuntimeError, match="second derivatives"):
        wl = w.clone().requires_grad_(True)
        torch.autograd.grad(add_rms_norm(x, wl)[0].float().sum(), wl, create_graph=True)
