"""``add_rms_norm`` against its definition in 64 bits, forward and backward, and its MXFP8 rows against the row quantiser.

Bounds, u = 2^-24 (half a step of fp32), h = half a step of the output's type (bf16 2^-9 of the value's power of two, so 2^-8 of the
value at most; fp32 u).  The stored sum is the correctly rounded fp32 sum rounded again: compared bit for bit with the same two
roundings.  Mean of squares: D terms, each rounded, added in at most D / 32 + 10 steps (a thread's own, then a tree), so relative
error (D / 32 + 12) u; a reciprocal square root halves it and adds 2 u; two more products.  y is within (D / 64 + 12) u + h of the
exact value, relatively.  Gradients likewise, relative to the sum of the absolute terms."""

import pytest
import torch

import dist_moe_b200 as dm

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _inputs(T, D, residual, gain, center, seed=0, device=DEV):
    g = torch.Generator().manual_seed(1000 * T + D + seed)
    x = torch.randn(T, D, generator=g).bfloat16()
    r = None if residual is None else (2 * torch.randn(T, D, generator=g)).to(residual)
    w = (1.0 - center + 0.2 * torch.randn(D, generator=g)).to(gain)
    return x.to(device), None if r is None else r.to(device), w.to(device)


def _exact(x, r, w, eps, center):
    s = x if r is None else (x.float() + r.float()).to(r.dtype)
    a = s.double()
    rstd = 1.0 / (a.pow(2).mean(1, keepdim=True) + eps).sqrt()
    return s, a, rstd, a * rstd * (w.double() + center)


def _within(got, want, relative, what, scale=None):
    err = (got.double() - want).abs()
    bound = relative * (want.abs() if scale is None else scale) + 1e-38
    assert bool((err <= bound).all()), f"{what}: {(err / bound).max().item():.3g} times the bound"


# a warp's rows, 128 / 256 / 512 threads, ragged last pieces, lengths that are no multiple of 8, rows that no registers hold
SIZES = [(1, 8), (3, 64), (5, 1024), (2, 1088), (7, 2048), (4, 2816), (3, 4096), (2, 7168), (2, 8200), (1, 16384), (2, 16400), (6, 1),
         (3, 33), (2, 1001), (1000, 256)]


@pytest.mark.parametrize("residual", [None, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,D", SIZES)
def test_forward(T, D, residual):
    gain, center = (torch.float32, 1.0) if T % 2 else (torch.bfloat16, 0.0)
    x, r, w = _inputs(T, D, residual, gain, center)
    y, total = dm.add_rms_norm(x, w, residual_TD=r, eps=1e-5, gain_center=center)
    s, _, _, want = _exact(x, r, w, 1e-5, center)
    assert y.dtype == torch.bfloat16 and total.dtype == (residual or torch.bfloat16)
    assert torch.equal(total, s) and (r is not None or total is x)
    _within(y, want, (D / 64 + 12) * U + HALF[torch.bfloat16], "y")


@pytest.mark.parametrize("residual", [None, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,D", SIZES + [(700, 1088), (1300, 2048)])
def test_backward(T, D, residual):
    gain, center = (torch.float32, 1.0) if D % 3 else (torch.bfloat16, 0.0)
    x, r, w = _inputs(T, D, residual, gain, center)
    leaves = [t.requires_grad_() for t in (x, r, w) if t is not None]
    y, total = dm.add_rms_norm(x, w, residual_TD=r, gain_center=center)
    g = torch.Generator().manual_seed(5)
    gy, gs = torch.randn(T, D, generator=g).bfloat16().to(DEV), torch.randn(T, D, generator=g).to(total.dtype).to(DEV)
    got = torch.autograd.grad((y,) if r is None else (y, total), leaves, (gy,) if r is None else (gy, gs))
    _, a, rstd, _ = _exact(x.detach(), None if r is None else r.detach(), w.detach(), 1e-6, center)
    u = gy.double() * (w.detach().double() + center)
    mean = (u * a).mean(1, keepdim=True)
    want = (0 if r is None else gs.double()) + rstd * (u - a * rstd.pow(2) * mean)
    scale = (0 if r is None else gs.double().abs()) + rstd * (u.abs() + a.abs() * rstd.pow(2) * (u * a).abs().mean(1, keepdim=True))
    steps = (D / 16 + 40) * U  # the sums over a row appear to the third power
    _within(got[0], want, steps + HALF[torch.bfloat16], "grad_x", scale)
    if r is not None:
        _within(got[1], want, steps + HALF[r.dtype], "grad_residual", scale)
    terms = gy.double() * a * rstd
    # T terms, one row after another in a block and the blocks' shares after that
    _within(got[-1], terms.sum(0), (D / 64 + 12 + T) * U + HALF[gain], "grad_weight", terms.abs().sum(0))


def test_gradients_agree_with_differences():
    """The definition itself is differentiated by central differences in 64 bits; its analytic form is what test_backward uses."""
    x, r, w = _inputs(2, 40, torch.float32, torch.float32, 0.0)
    gy, gs = torch.randn(2, 40, device=DEV).bfloat16(), torch.randn(2, 40, device=DEV)
    for t in (r, w):
        t.requires_grad_()
    y, total = dm.add_rms_norm(x, w, residual_TD=r)
    got = torch.autograd.grad((y, total), (r, w), (gy, gs))

    def value(rr, ww):
        a = x.double() + rr
        out = a / (a.pow(2).mean(1, keepdim=True) + 1e-6).sqrt() * ww
        return (out * gy.double()).sum() + (a * gs.double()).sum()

    h = 1e-5
    for which, grad in enumerate(got):
        base = [r.detach().double(), w.detach().double()]
        for i in range(0, base[which].numel(), 7):
            up, down = [b.clone() for b in base], [b.clone() for b in base]
            up[which].view(-1)[i] += h
            down[which].view(-1)[i] -= h
            slope = (value(*up) - value(*down)) / (2 * h)
            assert abs(slope.item() - grad.reshape(-1)[i].item()) < 1e-4  # fp32 sums of 80 terms of order 1, h^2 third derivatives


def test_one_output_alone_and_one_input_alone():
    x, r, w = _inputs(9, 256, torch.float32, torch.float32, 0.0)
    r.requires_grad_()
    y, total = dm.add_rms_norm(x, w, residual_TD=r)
    gy, gs = torch.randn(9, 256, device=DEV).bfloat16(), torch.randn(9, 256, device=DEV)
    only_y, = torch.autograd.grad(y, r, gy, retain_graph=True)
    only_sum, = torch.autograd.grad(total, r, gs, retain_graph=True)
    both, = torch.autograd.grad((y, total), r, (gy, gs))
    assert torch.equal(only_sum, gs)
    torch.testing.assert_close(only_y + only_sum, both, rtol=4 * U, atol=16 * U)  # one addition of values below 8
    w = w.requires_grad_()
    y, total = dm.add_rms_norm(x, w)
    assert total is x and torch.autograd.grad(y, w, gy)[0].abs().sum() > 0
    y, total = dm.add_rms_norm(x, w, residual_TD=r)
    gx, gw = torch.autograd.grad(total.sum(), (r, w), allow_unused=True)
    assert torch.equal(gx, torch.ones_like(gx)) and (gw is None or not gw.any())


def test_expanded_gradients_and_a_backward_taken_twice():
    x, r, w = _inputs(40, 1088, torch.bfloat16, torch.bfloat16, 0.0)
    x.requires_grad_(), w.requires_grad_(), r.requires_grad_()
    y, total = dm.add_rms_norm(x, w, residual_TD=r)
    loss = y.float().sum() + total.float().sum()
    a = torch.autograd.grad(loss, (x, r, w), retain_graph=True)
    b = torch.autograd.grad(loss, (x, r, w))
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and torch.equal(a[0], a[1])


def test_rows_that_lie_apart_and_unaligned_ones():
    wide = torch.randn(6, 4200, device=DEV).bfloat16()
    w = torch.rand(2048, device=DEV) + 0.5
    for first in (0, 8, 3):
        x, r = wide[:, first:first + 2048], wide[:, 2100 + first:4148 + first]
        got = dm.add_rms_norm(x, w, residual_TD=r)
        want = dm.add_rms_norm(x.contiguous(), w, residual_TD=r.contiguous())
        assert torch.equal(got[1], want[1])
        torch.testing.assert_close(got[0], want[0], rtol=2 * HALF[torch.bfloat16], atol=0)  # another order of the sum may round apart
    t = torch.randn(256, 6, device=DEV).bfloat16()
    assert torch.equal(dm.add_rms_norm(t.t(), w[:256])[0], dm.add_rms_norm(t.t().contiguous(), w[:256])[0])
    assert torch.equal(dm.add_rms_norm(wide[:1].expand(5, -1), torch.ones(4200, device=DEV))[0][4],
                       dm.add_rms_norm(wide[:1], torch.ones(4200, device=DEV))[0][0])


def test_zeros_infinities_and_no_tokens():
    w = torch.ones(512, device=DEV)
    x = torch.zeros(3, 512, device=DEV, dtype=torch.bfloat16)
    x[1, 7], x[2, 9] = float("inf"), float("nan")
    y, _ = dm.add_rms_norm(x, w)
    assert not y[0].any() and y[1, 7].isnan() and not y[1, :7].any() and y[2].isnan().all()
    x = torch.empty(0, 512, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    w.requires_grad_()
    y, total = dm.add_rms_norm(x, w, residual_TD=torch.empty(0, 512, device=DEV))
    assert y.shape == total.shape == (0, 512)
    gx, gw = torch.autograd.grad(y.sum(), (x, w))
    assert gx.shape == (0, 512) and not gw.any()
    with torch.no_grad():
        assert dm.add_rms_norm(x, w, quantize=True)[2].dequantize().shape == (0, 512)


@pytest.mark.parametrize("residual", [None, torch.float32])
@pytest.mark.parametrize("T,D", [(1, 32), (5, 96), (9, 1024), (33, 2816), (4, 7168), (2, 16384), (3, 1056)])
def test_rows_are_those_of_the_row_quantiser(T, D, residual):
    from dist_moe_b200 import _native as nat

    x, r, w = _inputs(T, D, residual, torch.bfloat16, 0.0)
    x[0, :32] = 0  # a block of zeros where nothing is added
    y, total, rows = dm.add_rms_norm(x, w, residual_TD=r, quantize=True)
    plain = dm.add_rms_norm(x, w, residual_TD=r)
    assert torch.equal(y, plain[0]) and torch.equal(total, plain[1])
    want = torch.zeros_like(rows.packed)
    stride = want.shape[1]
    nat.check(nat.lib.dm_quant_mxfp8_row(y.data_ptr(), None, T, D, want.data_ptr(), stride, want.data_ptr() + D, stride, 0,
                                         nat.stream_ptr()), "dm_quant_mxfp8_row")
    assert torch.equal(rows.packed, want)
    value = rows.data.float().double() * torch.exp2(rows.scales.double() - 127).repeat_interleave(32, 1)
    assert torch.equal(rows.dequantize().double(), value.bfloat16().double())
    # half a step of E4M3 relative to a value above the smallest normal of its block, else of the smallest step
    err = (value - y.double()).abs()
    smallest = torch.exp2(rows.scales.double() - 127 - 10).repeat_interleave(32, 1)
    assert bool((err <= torch.maximum(2.0 ** -4 * y.double().abs(), smallest)).all())


def test_rows_of_unaligned_and_strided_tokens():
    wide = torch.randn(5, 1000, device=DEV).bfloat16()
    w = torch.rand(300, device=DEV).bfloat16()
    x = wide[:, 3:259]
    got, want = dm.add_rms_norm(x, w[1:257], quantize=True), dm.add_rms_norm(x.clone(), w[1:257].clone(), quantize=True)
    assert torch.equal(got[2].packed, want[2].packed) and got[1] is not None


def test_nonfinite_blocks_of_rows():
    w = torch.ones(64, device=DEV)
    x = torch.ones(1, 64, device=DEV).bfloat16()
    x[0, 40] = float("inf")
    _, _, rows = dm.add_rms_norm(x, w, quantize=True)
    assert rows.scales[0].tolist()[1] == 0xFF and rows.dequantize()[0, 32:].isnan().all()


def test_a_captured_step_replays_on_new_values():
    x, r, w = _inputs(24, 2048, torch.float32, torch.float32, 0.0)
    x.requires_grad_(), r.requires_grad_(), w.requires_grad_()
    gy, gs = torch.randn(24, 2048, device=DEV).bfloat16(), torch.randn(24, 2048, device=DEV)

    def step():
        y, total = dm.add_rms_norm(x, w, residual_TD=r)
        return (y, total) + torch.autograd.grad((y, total), (x, r, w), (gy, gs))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.copy_(torch.randn_like(x)), r.copy_(torch.randn_like(r)), gs.copy_(torch.randn_like(gs))
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_same_bits_every_time_and_on_another_stream():
    x, r, w = _inputs(3000, 1088, torch.bfloat16, torch.float32, 0.0)
    w.requires_grad_()
    gy = torch.randn(3000, 1088, device=DEV).bfloat16()
    first = torch.autograd.grad(dm.add_rms_norm(x, w, residual_TD=r)[0], w, gy)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = torch.autograd.grad(dm.add_rms_norm(x, w, residual_TD=r)[0], w, gy)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, again)


def test_rows_behind_32_bit_offsets():
    D, last = 8192, 5
    T = 2 ** 31 // D + 100
    w = torch.rand(D, device=DEV)
    x, gy = (torch.zeros(T, D, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    for t in (x, gy):
        t[-last:] = torch.randn(last, D, device=DEV)
    few = [t[-last:].clone().requires_grad_() for t in (x, x)] + [w.clone().requires_grad_()]
    many = [x.requires_grad_(), x.detach().clone().requires_grad_(), w.requires_grad_()]
    got = []
    for a, r, g in (many, few):
        y, total = dm.add_rms_norm(a, g, residual_TD=r)
        ga, gr, gg = torch.autograd.grad((y, total), (a, r, g), (gy[-len(a):], gy[-len(a):]))
        got.append([t[-last:].clone() for t in (y, total, ga, gr)] + [gg])
        del y, total, ga, gr
    for a, b in zip(got[0][:4], got[1][:4]):
        assert torch.equal(a, b)
    # The other rows add zeros.  The five meet in another order: two roundings of a product and four of sums on either side, 2^-24 each
    # of the sum of |gy s rstd|, and |s rstd| is at most sqrt(D).
    bound = 12 * 2.0 ** -24 * D ** 0.5 * gy[-last:].double().abs().sum(0)
    assert bool(((got[0][4].double() - got[1][4].double()).abs() <= bound).all())
    with torch.no_grad():
        rows = dm.add_rms_norm(x, w, residual_TD=x, quantize=True)[2]
        want = dm.add_rms_norm(x[-last:].clone(), w, residual_TD=x[-last:].clone(), quantize=True)[2]
        assert torch.equal(rows.packed[-last:], want.packed)


def test_gradients_are_not_differentiated_again():
    x, r, w = (t.requires_grad_() for t in _inputs(5, 256, torch.float32, torch.float32, 0.0))
    y, total = dm.add_rms_norm(x, w, residual_TD=r)
    loss = y.float().pow(2).sum() + total.sum()
    first = torch.autograd.grad(loss, (x, r, w), retain_graph=True)
    again = torch.autograd.grad(loss, (x, r, w), create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, again)) and again[0].requires_grad
    with pytest.raises(RuntimeError, match="differentiate twice"):
        again[1].sum().backward()
