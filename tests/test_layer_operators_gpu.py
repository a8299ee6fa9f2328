"""The operators of a layer as a program runs them: norm, router, experts, in training (BF16) and in decode steps (few tokens, MXFP8
rows), against a plain implementation in 64 bits or against the same steps taken apart."""

import pytest
import torch

import dist_moe_b200 as dm
from tests.helpers import BF16_FWD, BF16_GRAD, BF16_WGRAD, assert_close

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
D, F, E, K = 256, 384, 8, 2


def _weights(seed=0, layers=1):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape, fan):
        return (torch.randn(*shape, generator=g) * fan ** -0.5).bfloat16().to(DEV)

    return [dict(gain=(1 + 0.1 * torch.randn(D, generator=g)).to(DEV), gate=normal(E, D, fan=D), w13=normal(E, 2 * F, D, fan=D),
                 w2=normal(E, D, F, fan=F)) for _ in range(layers)]


def _context(T, **more):
    return dm.create_context(group=None, device=DEV, config=dm.Config(
        max_num_local_input_tokens=T, hidden_dim=D, intermediate_dim=F, top_k=K, num_experts=E, max_moe_layers_per_activation_slot=1, **more))


def test_a_training_step():
    T = 96
    w, = _weights()
    g = torch.Generator().manual_seed(3)
    x, stream = torch.randn(T, D, generator=g).bfloat16().to(DEV), (2 * torch.randn(T, D, generator=g)).to(DEV)
    mask = torch.arange(T, device=DEV) < T - 5
    leaves = [t.clone().requires_grad_() for t in (x, stream, w["gain"], w["gate"], w["w13"], w["w2"])]
    ctx = _context(T)
    y, total = dm.add_rms_norm(leaves[0], leaves[2], residual_TD=leaves[1])
    ids, scores = dm.select_experts(y.float() @ leaves[3].float().t(), K, renormalize=True, token_mask_T=mask)
    out = dm.routed_experts(y, ids, scores, leaves[4], leaves[5], ctx)
    grad = torch.randn(T, D, generator=g).to(DEV)
    got = torch.autograd.grad(out.float() + total, leaves, grad)
    ctx.check_status()
    ctx.close()

    ref = [t.detach().double().requires_grad_() for t in leaves]
    s = (x.float() + stream).double() + (ref[0] - ref[0].detach()) + (ref[1] - ref[1].detach())
    yy = s / (s.pow(2).mean(1, keepdim=True) + 1e-6).sqrt() * ref[2]
    yy = y.detach().double() + (yy - yy.detach())  # what the experts read is rounded
    p = torch.softmax(yy @ ref[3].t(), 1)
    v = p.gather(1, ids.clamp(min=0).long())
    v = torch.where(mask[:, None], v / v.sum(1, keepdim=True), 0.0)
    experts = torch.zeros_like(s)
    for e in range(E):
        h = yy @ ref[4][e].t()
        h = h[:, :F] * torch.sigmoid(h[:, :F]) * h[:, F:]
        experts = experts + torch.where(ids == e, v, 0.0).sum(1, keepdim=True) * (h @ ref[5][e].t())
    want = torch.autograd.grad(experts + s, ref, grad.double())
    assert (ids[T - 5:] == -1).all() and (ids[:T - 5] >= 0).all()
    assert_close(out, experts, what="out", **BF16_FWD)
    for name, a, b in zip(("x", "stream", "gain", "gate", "w13", "w2"), got, want):
        assert_close(a, b, what=name, **(BF16_GRAD if name in ("x", "stream") else BF16_WGRAD))


def test_a_captured_decode_step_of_two_layers():
    T, layers = 5, _weights(layers=2)
    ctx = _context(16, inference=True)

    @torch.no_grad()
    def step(x, stream):
        for w in layers:
            y, stream = dm.add_rms_norm(x, w["gain"], residual_TD=stream)
            ids, scores = dm.select_experts(y.float() @ w["gate"].float().t(), K, score="sigmoid", renormalize=True, scale=1.5)
            x = dm.routed_experts_few_tokens(y, ids, scores, w["w13"], w["w2"], ctx)
        return dm.add_rms_norm(x, layers[0]["gain"], residual_TD=stream)

    @torch.no_grad()
    def plain(x, stream):
        x, stream = x.double(), stream.double()
        for w in layers:
            stream = x + stream
            y = (stream / (stream.pow(2).mean(1, keepdim=True) + 1e-6).sqrt() * w["gain"].double()).bfloat16().double()
            p = torch.sigmoid(y @ w["gate"].double().t())
            v, ids = p.topk(K, 1)
            v = 1.5 * v / v.sum(1, keepdim=True)
            x = torch.zeros_like(stream)
            for e in range(E):
                h = y @ w["w13"][e].double().t()
                h = h[:, :F] * torch.sigmoid(h[:, :F]) * h[:, F:]
                x += torch.where(ids == e, v, 0.0).sum(1, keepdim=True) * (h @ w["w2"][e].double().t())
        stream = x + stream
        return stream / (stream.pow(2).mean(1, keepdim=True) + 1e-6).sqrt() * layers[0]["gain"].double()

    x, stream = torch.randn(T, D, device=DEV).bfloat16(), torch.randn(T, D, device=DEV)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(x, stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, stream)
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        x.copy_(torch.randn(T, D, generator=g).bfloat16()), stream.copy_(torch.randn(T, D, generator=g))
        graph.replay()
        assert_close(out[0], plain(x, stream), what="decode step", **BF16_FWD)
        eager = step(x, stream)
        assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])
    ctx.check_status()
    ctx.close()


@pytest.mark.parametrize("T", [1, 40, 300])
def test_quantised_rows_in_front_of_mxfp8_experts(T):
    w, = _weights()
    config = dict(inference=True, block_scaled=dm.BlockScaledConfig())
    ctx = _context(T, **config)
    p13 = dm.prepare_block_scaled_weight(w["w13"], ctx.config, fuse_swiglu=True, inference=True)
    p2 = dm.prepare_block_scaled_weight(w["w2"], ctx.config, inference=True)
    x, stream = torch.randn(T, D, device=DEV).bfloat16(), torch.randn(T, D, device=DEV).bfloat16()
    y, _, rows = dm.add_rms_norm(x, w["gain"], residual_TD=stream, quantize=True)
    ids, scores = dm.select_experts(rows.dequantize().float() @ w["gate"].float().t(), K)
    post = dm.ExecutionOptions(experts_output_postprocess=dm.RMSNormPostprocess(
        eps=1e-6, norm_output_dtype=torch.bfloat16, output_dtype=torch.bfloat16))
    for options in (None, post, dm.ExecutionOptions(validate_expert_ids=True)):
        a, b = (dm.routed_experts(t, ids, scores, p13, p2, ctx, options=options) for t in (rows, y))
        assert torch.equal(a, b)
    assert torch.equal(dm.routed_experts(rows, ids, scores, w["w13"], w["w2"], ctx), dm.routed_experts(y, ids, scores, w["w13"], w["w2"], ctx))
    ctx.check_status()
    with pytest.raises(ValueError, match="hidden dimension"):
        dm.routed_experts(dm.QuantizedRows(torch.zeros(T, 48, dtype=torch.uint8, device=DEV), 32), ids, scores, p13, p2, ctx)
    with pytest.raises(ValueError, match="tokens"):
        dm.routed_experts(dm.QuantizedRows(torch.zeros(T + 1, 272, dtype=torch.uint8, device=DEV), D), ids, scores, p13, p2, ctx)
    ctx.close()
    plain = _context(T, inference=True)
    with pytest.raises(ValueError, match="MXFP8 context"):
        dm.routed_experts(rows, ids, scores, w["w13"], w["w2"], plain)
    with pytest.raises(TypeError, match="x_TD"):
        dm.routed_experts_few_tokens(rows, ids, scores, w["w13"], w["w2"], plain)
    plain.close()
    training = _context(T, block_scaled=dm.BlockScaledConfig())
    with pytest.raises(RuntimeError, match="forward-only"):
        dm.routed_experts(rows, ids, scores.clone().requires_grad_(), w["w13"], w["w2"], training)
    training.close()


def test_quantised_rows_refuse_gradients_and_odd_sizes():
    x, gain = torch.randn(3, 64, device=DEV).bfloat16(), torch.ones(64, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        dm.add_rms_norm(x, gain, quantize=True)
    with torch.no_grad():
        assert dm.add_rms_norm(x, gain, quantize=True)[2].packed.shape == (3, 80)
    for dim in (40, 16416):
        with pytest.raises(ValueError, match="multiple of 32"):
            dm.add_rms_norm(torch.zeros(1, dim, device=DEV, dtype=torch.bfloat16), torch.ones(dim, device=DEV), quantize=True)
    for eps, center in ((0.0, 0.0), (float("nan"), 0.0), (1e-6, float("inf"))):
        with pytest.raises(ValueError, match="finite"):
            dm.add_rms_norm(x, gain, eps=eps, gain_center=center)
    for shape, dim in (((3, 64), 64), ((3, 81), 64)):
        with pytest.raises(ValueError, match="packed"):
            dm.QuantizedRows(torch.zeros(shape, dtype=torch.uint8, device=DEV), dim)
