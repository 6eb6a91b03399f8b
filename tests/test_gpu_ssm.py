"""chunk_ssm / ssm_step against the 64-bit recurrence.

Bounds are elementwise and relative to the sums of the terms' magnitudes (the oracle over absolute values):
float32: every result is a sum of at most K + V + T + ... products whose factors carry a few roundings of 2^-24 each, and the
decays' exponents are good to 2^-24 relative to |L| e^{-|L|} <= 0.4: n * 2^-24 with n = K + V + 4 rep + 2 chunk + 64 covers any
order of summation.  16-bit results add their own rounding, eps/2 of the value.  On the tensor cores the products' operands that
are made inside (P, dS, the scaled v and do, the state and its gradient as operands) are rounded to bfloat16 once, 2^-8 relative
at most, at most three of them in a chain: 3 * 2^-8 of the magnitudes; results in float32 (states, dgt's sums, dg, dD, dgt_bias)
use operands in two parts, 2^-16 relative each: 4 * 2^-16.
"""
import pytest
import torch

from oracle import block_oracle as bo

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make(seed, B, T, H, Hq, K, V, dtype, softplus=True, D=True, bias=True, h0=True, n=None, fast=False, gt_dtype=None):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    n = B if n is None else n
    d = dict(q=r(B, T, Hq, K).to(dtype), k=r(B, T, Hq, K).to(dtype), v=r(B, T, H, V).to(dtype))
    gt = r(B, T, H) - (1.0 if softplus else 0.0)
    d["gt"] = (gt if softplus else gt.abs() * 0.2).to(gt_dtype or dtype)
    d["g"] = torch.rand(H, generator=gen) * (40 if fast else 2) + 0.01
    d["D"] = r(H) if D else None
    d["gt_bias"] = 0.3 * r(H).abs() if bias else None
    d["h0"] = r(n, H, V, K) if h0 else None
    d["do"], d["dh"] = r(B, T, H, V).to(dtype), r(n, H, V, K)
    return d


def on_gpu(d, grads=True):
    leaf = lambda x: None if x is None else x.to(DEV).requires_grad_(grads)
    return {n: leaf(x) if n not in ("do", "dh") else x.to(DEV) for n, x in d.items()}


def run(d, softplus, cu=None, final=True, grads=True):
    from palimpsa_b200.ops import chunk_ssm
    x = on_gpu(d, grads)
    cut = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=DEV)
    out = chunk_ssm(x["q"], x["k"], x["v"], x["gt"], x["g"], D=x["D"], gt_bias=x["gt_bias"], gt_softplus=softplus,
                    initial_state=x["h0"], output_final_state=final, cu_seqlens=cut)
    o, h = out if final else (out, None)
    got = {"o": o, "h": h}
    if grads:
        names = [n for n in ("q", "k", "v", "gt", "g", "D", "gt_bias", "h0") if x[n] is not None]
        outs, cot = ([o, h], [x["do"], x["dh"]]) if final else ([o], [x["do"]])
        for n, gr in zip(names, torch.autograd.grad(outs, [x[n] for n in names], cot)):
            assert gr.dtype == x[n].dtype and gr.shape == x[n].shape, n
            got["d" + n] = gr
    torch.cuda.synchronize()
    return {n: t.detach().cpu() for n, t in got.items() if t is not None}


def tensor_cores(d):
    K, V = d["q"].shape[-1], d["v"].shape[-1]
    return d["q"].dtype == torch.bfloat16 and K % 8 == 0 and V % 8 == 0 and K <= 128


def check(d, got, softplus, cu=None, final=True, what=""):
    kw = dict(D=d["D"], gt_bias=d["gt_bias"], softplus=softplus, h0=d["h0"], do=d["do"], dh=d["dh"] if final else None, cu=cu)
    ref = bo.ssm(d["q"], d["k"], d["v"], d["gt"], d["g"], **kw)
    mag = bo.ssm(d["q"], d["k"], d["v"], d["gt"], d["g"], magnitude=True, **kw)
    (B, T, Hq, K), (H, V) = d["q"].shape, d["v"].shape[2:]
    tc = tensor_cores(d)
    n = K + V + 4 * (H // Hq) + 2 * (128 if tc else 32) + 64
    worst = {}
    for name, x in got.items():
        inner = n * 2.0 ** -24
        if tc:
            inner += 3 * 2.0 ** -8 if name in ("o", "dq", "dk", "dv") else 4 * 2.0 ** -16
        if name in ("dg", "dgt_bias", "dD"):
            inner += 64 * 2.0 ** -24                  # shares of chunks, summed in 64 bits
        bound = inner * mag[name] + HALF[x.dtype] * ref[name].abs() + (2.0 ** -25 if x.dtype == torch.float16 else 1e-30)
        err = (x.double() - ref[name]).abs()
        worst[name] = float((err / bound).nan_to_num(nan=1e9).max()) if err.numel() else 0.0
    bad = {k: w for k, w in worst.items() if not w <= 1}
    assert not bad, f"{what}: error / bound {bad} of {worst}"


SHAPES = [(2, 70, 4, 2, 31, 65), (1, 1, 2, 1, 16, 8), (2, 33, 2, 2, 48, 96), (1, 130, 3, 1, 128, 64), (1, 40, 2, 2, 200, 24),
          (1, 300, 2, 1, 64, 64), (1, 257, 2, 2, 96, 192), (3, 32, 1, 1, 5, 3), (1, 64, 2, 1, 256, 130)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_forward_and_backward(shape, dtype):
    d = make(1, *shape, dtype)
    check(d, run(d, True), True, what=f"{shape} {dtype}")


@pytest.mark.parametrize("softplus,D,bias,h0,final", [(False, False, False, False, False), (True, False, True, False, True),
                                                      (False, True, False, True, False), (True, True, False, False, False)])
@pytest.mark.parametrize("dtype,K,V", [(torch.float32, 24, 40), (torch.bfloat16, 64, 48)])
def test_optional_parts(softplus, D, bias, h0, final, dtype, K, V):
    d = make(2, 2, 150, 4, 2, K, V, dtype, softplus=softplus, D=D, bias=bias, h0=h0)
    check(d, run(d, softplus, final=final), softplus, final=final)


CUTS = [[0, 1, 1, 130, 131, 260, 290], [0, 0, 0], [5, 9, 200, 290], [0, 290], [0] + list(range(1, 291, 17)) + [290], [0, 290, 290, 290]]


@pytest.mark.parametrize("cu", CUTS)
@pytest.mark.parametrize("dtype,K,V", [(torch.float32, 16, 24), (torch.bfloat16, 128, 64), (torch.bfloat16, 30, 17)])
def test_packed(cu, dtype, K, V):
    """Empty and one-token sequences, chunks that end inside, rows in front of the first and behind the last."""
    d = make(3, 1, 290, 4, 1, K, V, dtype, n=len(cu) - 1)
    got = run(d, True, cu=cu)
    for name in ("o", "dq", "dk", "dv", "dgt"):      # rows of no sequence
        assert not got[name][0, :cu[0]].any() and not got[name][0, cu[-1]:].any(), name
    check(d, got, True, cu=cu)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_fast_and_vanishing_decays(dtype):
    """Products that underflow inside a chunk, tokens that reset the state, steps of zero, a step that underflows."""
    d = make(4, 2, 200, 2, 1, 64, 64, dtype, fast=True, softplus=False, bias=False, gt_dtype=torch.float32)
    d["gt"][:, 20:40] = 0
    d["gt"][0, 50] = 1e6
    d["gt"][1, 60] = 3e38
    d["v"][1, 60] = 0                                  # its step times v would be infinite
    d["q"][1, 60] = 0
    d["do"][1, 60] = 0
    got = run(d, False)
    ref = bo.ssm(d["q"], d["k"], d["v"], d["gt"], d["g"], D=d["D"], h0=d["h0"], do=d["do"], dh=d["dh"])
    for n, x in got.items():                           # dv of that token is 3e38 (G k): beyond float32 by its formula
        assert torch.isfinite(x[ref[n].abs() < 1e37]).all(), n
    d["gt"][1, 60] = 1e4
    check(d, run(d, False), False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_sequence_of_slow_decays(dtype):
    """2000 tokens, states carried over many chunks."""
    d = make(5, 1, 2000, 2, 1, 32, 16, dtype, softplus=False, bias=False, gt_dtype=torch.float32)
    d["gt"] *= 0.01
    got = run(d, False)
    check(d, got, False)


@pytest.mark.parametrize("dtype,K,V", [(torch.float32, 16, 24), (torch.bfloat16, 64, 64), (torch.bfloat16, 128, 96)])
def test_what_one_sequence_holds_stays_in_it(dtype, K, V):
    """NaN and infinities in one sequence of a batch, packed or not: the others come out, forward and backward, as without them."""
    cu = [0, 70, 200, 330]
    d = make(16, 1, 330, 2, 1, K, V, dtype, n=3)
    clean = run(d, True, cu=cu)
    for n, bad in (("q", float("nan")), ("k", float("inf")), ("v", float("nan")), ("do", float("inf")), ("gt", float("nan"))):
        e = {m: None if t is None else t.clone() for m, t in d.items()}
        e[n][0, 70:200] = bad
        got = run(e, True, cu=cu)
        for m in ("o", "dq", "dk", "dv", "dgt"):
            for a, b in ((0, 70), (200, 330)):
                assert torch.equal(got[m][0, a:b], clean[m][0, a:b]), (n, m)
        for m in ("h", "dh0"):
            assert torch.equal(got[m][[0, 2]], clean[m][[0, 2]]), (n, m)
    batch = make(17, 3, 130, 2, 1, K, V, dtype)
    clean = run(batch, True)
    for n in ("q", "k", "v", "do"):
        e = {m: None if t is None else t.clone() for m, t in batch.items()}
        e[n][1] = float("nan")
        got = run(e, True)
        for m in ("o", "dq", "dk", "dv", "dgt", "h", "dh0"):
            assert torch.equal(got[m][[0, 2]], clean[m][[0, 2]]), (n, m)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient_through_the_final_state_alone(dtype):
    from palimpsa_b200.ops import chunk_ssm
    d = make(18, 2, 128, 2, 1, 64, 64, dtype)
    x = on_gpu(d)
    _, h = chunk_ssm(x["q"], x["k"], x["v"], x["gt"], x["g"], gt_softplus=True, initial_state=x["h0"], output_final_state=True)
    got = torch.autograd.grad(h, [x["v"], x["h0"], x["q"]], x["dh"])
    assert not got[2].any()
    kw = dict(softplus=True, h0=d["h0"], do=torch.zeros_like(d["do"]), dh=d["dh"])
    ref, mag = (bo.ssm(d["q"], d["k"], d["v"], d["gt"], d["g"], magnitude=m, **kw) for m in (False, True))
    for name, y in (("dv", got[0]), ("dh0", got[1])):
        inner = 600 * 2.0 ** -24 + (4 * 2.0 ** -16 if dtype == torch.bfloat16 else 0)
        assert ((y.cpu().double() - ref[name]).abs() <= inner * mag[name] + HALF[y.dtype] * ref[name].abs() + 1e-30).all()


def test_rows_apart_are_read_in_place_and_copied_where_they_must_be():
    from palimpsa_b200.ops import chunk_ssm
    for dtype, T in ((torch.float32, 37), (torch.bfloat16, 140)):
        d = make(6, 2, T, 4, 2, 48, 32, dtype, h0=False)
        x = {n: t.to(DEV) for n, t in d.items() if t is not None}
        base = chunk_ssm(x["q"], x["k"], x["v"], x["gt"], x["g"], gt_softplus=True)
        H, V, Hq, K = 4, 32, 2, 48
        wide = torch.cat([x["v"].flatten(2), x["k"].flatten(2), x["q"].flatten(2)], -1)
        for pad in (0, 8, 1):                          # an odd row length leaves the rows unaligned
            row = torch.cat([wide, wide.new_zeros(2, T, pad)], -1) if pad else wide
            v, k, q, _ = row.split([H * V, Hq * K, Hq * K, pad], -1)
            o = chunk_ssm(q.unflatten(-1, (Hq, K)), k.unflatten(-1, (Hq, K)), v.unflatten(-1, (H, V)), x["gt"], x["g"], gt_softplus=True)
            if pad != 1 or dtype == torch.float32:
                assert torch.equal(o, base)
            else:    # CUDA cores here, tensor cores there: each within its bound of the recurrence, see the top
                mag = bo.ssm(d["q"], d["k"], d["v"], d["gt"], d["g"], softplus=True, magnitude=True)["o"]
                bound = 3.1 * 2.0 ** -8 * mag + 2 * 2.0 ** -8 * base.cpu().double().abs() * (1 + 2.0 ** -6)
                assert ((o.double() - base.double()).abs().cpu() <= bound).all()
        heads_first = x["v"].transpose(1, 2).contiguous().transpose(1, 2)
        assert torch.equal(chunk_ssm(x["q"], x["k"], heads_first, x["gt"], x["g"], gt_softplus=True), base)
        assert torch.equal(chunk_ssm(x["q"][:, ::2], x["k"][:, ::2], x["v"][:, ::2], x["gt"][:, ::2], x["g"]),
                           chunk_ssm(*[x[n][:, ::2].contiguous() for n in ("q", "k", "v", "gt")], x["g"]))
        one = x["q"][:, :1].expand(-1, T, -1, -1)      # stride 0; steps below zero let the state grow past float32: compare the bits
        bits = lambda y: y.view(torch.int16 if dtype == torch.bfloat16 else torch.int32)
        assert torch.equal(bits(chunk_ssm(one, one, x["v"], x["gt"], x["g"])),
                           bits(chunk_ssm(one.contiguous(), one.contiguous(), x["v"], x["gt"], x["g"])))


def test_mixed_types_take_the_widest():
    from palimpsa_b200.ops import chunk_ssm
    d = make(7, 1, 20, 2, 1, 16, 16, torch.float32, h0=False)
    x = {n: t.to(DEV) for n, t in d.items() if t is not None}
    v16 = x["v"].bfloat16()
    o = chunk_ssm(x["q"], x["k"], v16, x["gt"], x["g"])
    assert o.dtype == torch.bfloat16
    assert torch.equal(o, chunk_ssm(x["q"], x["k"], v16.float(), x["gt"], x["g"]).bfloat16())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_repeat_runs_are_bitwise_equal(dtype):
    d = make(8, 2, 333, 4, 1, 64, 64, dtype)
    a, b = run(d, True), run(d, True)
    for n in a:
        assert torch.equal(a[n], b[n]), n


def test_empty_calls():
    from palimpsa_b200.ops import chunk_ssm, ssm_step
    z = lambda *s: torch.zeros(*s, device=DEV, requires_grad=True)
    h0 = torch.randn(2, 2, 4, 4, device=DEV, requires_grad=True)
    o, h = chunk_ssm(z(2, 0, 1, 4), z(2, 0, 1, 4), z(2, 0, 2, 4), z(2, 0, 2), z(2), initial_state=h0, output_final_state=True)
    assert o.shape == (2, 0, 2, 4) and torch.equal(h, h0)
    (gr,) = torch.autograd.grad(h, h0, torch.ones_like(h))
    assert torch.equal(gr, torch.ones_like(gr))
    o, h = chunk_ssm(z(0, 3, 1, 4), z(0, 3, 1, 4), z(0, 3, 2, 4), z(0, 3, 2), z(2), output_final_state=True)
    assert o.shape == (0, 3, 2, 4) and h.shape == (0, 2, 4, 4)
    cu = torch.zeros(1, dtype=torch.int32, device=DEV)
    o = chunk_ssm(z(1, 5, 1, 4), z(1, 5, 1, 4), torch.ones(1, 5, 2, 4, device=DEV), z(1, 5, 2), z(2), cu_seqlens=cu)
    assert not o.any()
    assert ssm_step(z(0, 1, 1, 4), z(0, 1, 1, 4), z(0, 1, 2, 4), z(0, 1, 2), z(2), torch.zeros(0, 2, 4, 4, device=DEV)).shape == (0, 1, 2, 4)


def test_wrong_offsets_stay_inside():
    """Offsets that run backwards or beyond the row: whatever comes out, every access is inside."""
    from palimpsa_b200.ops import chunk_ssm
    for dtype in (torch.float32, torch.bfloat16):
        d = make(9, 1, 200, 2, 1, 64, 64, dtype, n=3)
        for cu in ([0, 500, 20, 9000], [-7, 100, 50, 200], [200, 100, 0, 0]):
            run(d, True, cu=cu)
    x = on_gpu(make(9, 1, 100, 2, 1, 16, 16, torch.float32, n=3), False)
    a = chunk_ssm(x["q"], x["k"], x["v"], x["gt"], x["g"], cu_seqlens=torch.tensor([0, 30, 100], device=DEV))     # int64 offsets
    b = chunk_ssm(x["q"], x["k"], x["v"], x["gt"], x["g"], cu_seqlens=torch.tensor([0, 30, 100], dtype=torch.int32, device=DEV))
    assert torch.equal(a, b)


@pytest.mark.parametrize("shape", [(3, 4, 2, 31, 65), (1, 2, 1, 128, 64), (5, 2, 2, 48, 96), (2, 2, 1, 200, 24), (1, 1, 1, 1, 1), (4, 3, 1, 64, 130),
                                   (2, 2, 2, 256, 16), (3, 2, 1, 12, 9)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_single_tokens_continue_a_prompt(shape, dtype):
    """ssm_step from the final state of chunk_ssm: 3 tokens, each against the recurrence; the state changes in place."""
    from palimpsa_b200.ops import ssm_step
    N, H, Hq, K, V = shape
    d = make(10, N, 3, H, Hq, K, V, dtype)
    ref = bo.ssm(d["q"], d["k"], d["v"], d["gt"], d["g"], D=d["D"], gt_bias=d["gt_bias"], softplus=True, h0=d["h0"])
    mag = bo.ssm(d["q"], d["k"], d["v"], d["gt"], d["g"], D=d["D"], gt_bias=d["gt_bias"], softplus=True, h0=d["h0"], magnitude=True)
    x = on_gpu(d, False)
    state, version = x["h0"], x["h0"]._version
    where = state.data_ptr()
    for t in range(3):
        o = ssm_step(x["q"][:, t:t + 1], x["k"][:, t:t + 1], x["v"][:, t:t + 1], x["gt"][:, t:t + 1], x["g"], state, D=x["D"],
                     gt_bias=x["gt_bias"], gt_softplus=True)
        assert o.shape == (N, 1, H, V) and o.dtype == dtype
        bound = (K + 48) * 2.0 ** -24 * mag["o"][:, t] + HALF[dtype] * ref["o"][:, t].abs() + 2.0 ** -25
        assert ((o[:, 0].cpu().double() - ref["o"][:, t]).abs() <= bound).all()
    assert state.data_ptr() == where and state._version > version
    assert ((state.cpu().double() - ref["h"]).abs() <= 48 * 2.0 ** -24 * mag["h"]).all()
    flat = ssm_step(x["q"][:, 0], x["k"][:, 0], x["v"][:, 0], x["gt"][:, 0], x["g"], state.clone(), gt_softplus=True)
    assert flat.shape == (N, 1, H, V)


def test_step_replays_from_a_graph_and_training_from_another():
    from palimpsa_b200.ops import chunk_ssm, ssm_step
    d = make(11, 4, 130, 4, 1, 64, 64, torch.bfloat16)
    x = on_gpu(d, False)
    tok = {n: x[n][:, :1].clone() for n in ("q", "k", "v", "gt")}
    ref_state = x["h0"].clone()
    refs = []
    for t in range(3):
        refs.append(ssm_step(*[x[n][:, t:t + 1] for n in ("q", "k", "v", "gt")], x["g"], ref_state))
    state = x["h0"].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ssm_step(tok["q"], tok["k"], tok["v"], tok["gt"], x["g"], state.clone())
        chunk_ssm(x["q"], x["k"], x["v"], x["gt"], x["g"])
    torch.cuda.current_stream().wait_stream(side)
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(one):
        o = ssm_step(tok["q"], tok["k"], tok["v"], tok["gt"], x["g"], state)
    with torch.cuda.graph(two):
        whole = chunk_ssm(x["q"], x["k"], x["v"], x["gt"], x["g"])
    for t in range(3):
        for n in tok:
            tok[n].copy_(x[n][:, t:t + 1])
        one.replay()
        two.replay()
        assert torch.equal(o, refs[t])
    assert torch.equal(state, ref_state)
    # steps below zero let the state grow past float32 here: the same bits all the same
    assert torch.equal(whole.view(torch.int16), chunk_ssm(x["q"], x["k"], x["v"], x["gt"], x["g"]).view(torch.int16))


def test_captured_training_step_repeats_the_eager_one():
    from palimpsa_b200.ops import chunk_ssm
    for dtype in (torch.float32, torch.bfloat16):
        d = make(12, 2, 150, 2, 1, 64, 64, dtype)
        x = on_gpu(d)
        leaves = [x[n] for n in ("q", "k", "v", "gt", "g", "D", "gt_bias", "h0")]

        def step():
            o, h = chunk_ssm(x["q"], x["k"], x["v"], x["gt"], x["g"], D=x["D"], gt_bias=x["gt_bias"], gt_softplus=True,
                             initial_state=x["h0"], output_final_state=True)
            return [o.detach(), h.detach(), *torch.autograd.grad([o, h], leaves, [x["do"], x["dh"]])]

        ref = step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for t in out:
            t.zero_()
        graph.replay()
        for a, b in zip(out, ref):
            assert torch.equal(a, b)


def test_backward_in_a_thread_that_has_not_used_the_device():
    """Autograd's thread with every allocation cached: the first thing it does with the device is this backward."""
    import os
    import subprocess
    import sys
    code = """
import torch
from palimpsa_b200.ops import chunk_ssm
r = lambda *s: torch.randn(*s, device='cuda', dtype=torch.bfloat16)
keep = [torch.empty(n, device='cuda', dtype=torch.uint8) for n in (1 << 20, 64 << 20, 256 << 20) for _ in range(8)]
q, v, gt, g, do = r(2, 256, 1, 64), r(2, 256, 4, 64), r(2, 256, 4), torch.ones(4, device='cuda'), r(2, 256, 4, 64)
chunk_ssm(q, q, v, gt, g, gt_softplus=True)
del keep
v.requires_grad_(True)
torch.autograd.grad(chunk_ssm(q, q, v, gt, g, gt_softplus=True), v, do)
torch.cuda.synchronize()
print('done')
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "done" in r.stdout, r.stderr[-2000:]


def test_two_calls_on_two_streams():
    from palimpsa_b200.ops import chunk_ssm
    d = [make(s, 2, 260, 4, 2, 64, 64, torch.bfloat16) for s in (13, 14)]
    x = [on_gpu(y, False) for y in d]
    call = lambda y: chunk_ssm(y["q"], y["k"], y["v"], y["gt"], y["g"], initial_state=y["h0"], gt_softplus=True)
    ref = [call(y) for y in x]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in x]
    outs = []
    for y, st in zip(x, streams):
        with torch.cuda.stream(st):
            outs.append([call(y) for _ in range(4)])
    torch.cuda.synchronize()
    for o, r in zip(outs, ref):
        assert all(torch.equal(y, r) for y in o)


def test_argument_errors():
    from palimpsa_b200.ops import chunk_ssm, ssm_step
    x = on_gpu(make(15, 2, 6, 4, 2, 8, 8, torch.float32), False)
    a = lambda **kw: chunk_ssm(*[kw.get(n, x[n]) for n in ("q", "k", "v", "gt", "g")],
                               **{n: y for n, y in kw.items() if n not in ("q", "k", "v", "gt", "g")})
    with pytest.raises(ValueError):
        a(q=x["q"][:, :, :1])
    with pytest.raises(ValueError):
        a(v=x["v"][:, :, :3], gt=x["gt"][:, :, :3], g=x["g"][:3])
    with pytest.raises(ValueError):
        a(gt=x["gt"][:, :5])
    with pytest.raises(ValueError):
        a(initial_state=x["h0"][:1])
    with pytest.raises(ValueError):
        a(D=x["D"][:2])
    with pytest.raises(ValueError, match="packed row"):
        a(cu_seqlens=torch.tensor([0, 6], device=DEV))
    with pytest.raises(TypeError):
        a(q=x["q"].double(), k=x["k"].double())
    with pytest.raises(TypeError):
        a(gt=x["gt"].long())
    big = torch.zeros(1, 1, 1, 257, device=DEV)
    with pytest.raises(ValueError, match="256"):
        chunk_ssm(big, big, torch.zeros(1, 1, 1, 4, device=DEV), torch.zeros(1, 1, 1, device=DEV), torch.ones(1, device=DEV))
    with pytest.raises(ValueError, match="one token"):
        ssm_step(x["q"], x["k"], x["v"], x["gt"], x["g"], x["h0"])
    t = [x[n][:, :1] for n in ("q", "k", "v", "gt")]
    for state in (x["h0"].bfloat16(), x["h0"].transpose(2, 3), x["h0"][:1], x["h0"].clone().requires_grad_(True)):
        with pytest.raises((ValueError, RuntimeError)):
            ssm_step(*t, x["g"], state)
    q = x["q"].clone().requires_grad_(True)
    (gr,) = torch.autograd.grad(a(q=q).sum(), q, create_graph=False)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(a(q=q).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="traced"):
        torch.func.vmap(lambda y: chunk_ssm(y, x["k"], x["v"], x["gt"], x["g"]))(torch.stack([x["q"], x["q"]]))
