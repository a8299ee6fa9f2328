"""The norm's backward where every block walks over several rows, in each of its forms.

A block takes one row at a time, or four of up to 1024 values, and up to four blocks an SM walk over them: with four and a half rounds of
that, stages are filled again and used again, the gain's gradient is a sum over rows in a block before it is one over blocks, and the last
round is not full.  Bounds as in test_add_rms_norm_gpu.py; the gain's gradient is a sum of T terms in at most T steps of any order."""

import pytest
import torch

import dist_moe_b200 as dm
from tests.test_add_rms_norm_gpu import DEV, HALF, U, _exact, _inputs, _within

pytestmark = pytest.mark.gpu

# row length, rows of a block at a time, blocks of an SM: rows to a warp; two pieces a thread; four pieces, two stages and one (fp32);
# lengths and addresses that no vectors hold, rows that no registers hold
FORMS = [(256, 4, 4), (1024, 4, 4), (1088, 1, 4), (8200, 1, 2), (10248, 1, 2), (16384, 1, 2), (33, 1, 4), (1001, 1, 4), (16392, 1, 4)]


@pytest.mark.parametrize("wanted", ["all", "gain", "rows"])
@pytest.mark.parametrize("residual", [None, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,rows,blocks", FORMS)
def test_backward_over_several_rounds(D, rows, blocks, residual, wanted):
    sms = torch.cuda.get_device_properties(DEV).multi_processor_count
    T = 9 * sms * blocks * rows // 2 + 1
    x, r, w = _inputs(T, D, residual, torch.float32, 0.0)
    g = torch.Generator(device=DEV).manual_seed(5)
    gy, gs = torch.randn(T, D, generator=g, device=DEV).bfloat16(), torch.randn(T, D, generator=g, device=DEV).to(residual or torch.bfloat16)
    stream = [t for t in (x, r) if t is not None]
    leaves = [t.requires_grad_() for t in {"all": stream + [w], "gain": [w], "rows": stream}[wanted]]
    y, total = dm.add_rms_norm(x, w, residual_TD=r)
    got = torch.autograd.grad((y,) if r is None else (y, total), leaves, (gy,) if r is None else (gy, gs), retain_graph=True)
    again = torch.autograd.grad((y,) if r is None else (y, total), leaves, (gy,) if r is None else (gy, gs))
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    _, a, rstd, _ = _exact(x.detach(), None if r is None else r.detach(), w.detach(), 1e-6, 0.0)
    if wanted != "gain":
        u = gy.double() * w.detach().double()
        mean = (u * a).mean(1, keepdim=True)
        want = (0 if r is None else gs.double()) + rstd * (u - a * rstd.pow(2) * mean)
        scale = (0 if r is None else gs.double().abs()) + rstd * (u.abs() + a.abs() * rstd.pow(2) * (u * a).abs().mean(1, keepdim=True))
        steps = (D / 16 + 40) * U
        _within(got[0], want, steps + HALF[torch.bfloat16], "grad_x", scale)
        if r is not None:
            _within(got[1], want, steps + HALF[residual], "grad_residual", scale)
        del u, want, scale
    if wanted != "rows":
        terms = gy.double() * a * rstd
        _within(got[-1], terms.sum(0), (D / 64 + 12 + T) * U + HALF[torch.float32], "grad_weight", terms.abs().sum(0))


@pytest.mark.parametrize("residual", [torch.bfloat16, torch.float32])
def test_unaligned_rows_over_several_rounds(residual):
    """Rows of 512 values that do not start on 16 bytes take the form of odd lengths; the same values aligned take another."""
    sms = torch.cuda.get_device_properties(DEV).multi_processor_count
    T, D = 18 * sms + 1, 512
    x, r, w = _inputs(T, D, residual, torch.float32, 0.0)
    gy = torch.randn(T, D, device=DEV).bfloat16()

    def grads(gain):
        leaves = [x.clone().requires_grad_(), r.clone().requires_grad_(), gain.requires_grad_()]
        y, _ = dm.add_rms_norm(leaves[0], leaves[2], residual_TD=leaves[1])
        return torch.autograd.grad(y, leaves, gy)

    moved = torch.zeros(D + 1, device=DEV)
    moved[1:] = w
    odd, even = grads(moved[1:].detach()), grads(w.clone())
    _, a, rstd, _ = _exact(x, r, w, 1e-6, 0.0)
    u = gy.double() * w.double()
    scale = rstd * (u.abs() + a.abs() * rstd.pow(2) * (u * a).abs().mean(1, keepdim=True))
    for p, q, h in ((odd[0], even[0], HALF[torch.bfloat16]), (odd[1], even[1], HALF[residual])):
        assert bool(((p.double() - q.double()).abs() <= 2 * ((D / 16 + 40) * U + h) * scale + 1e-38).all())
    terms = (gy.double() * a * rstd).abs().sum(0)
    assert bool(((odd[2].double() - even[2].double()).abs() <= 2 * ((D / 64 + 12 + T) * U + U) * terms).all())
