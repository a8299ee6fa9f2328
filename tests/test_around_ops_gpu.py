"""Calls around the experts under tracers, dispatch modes, recorders and activation checkpointing: they are operators then, and a trace
computes on other inputs what the calls compute, bit for bit."""

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.profiler import ProfilerActivity, profile
from torch.utils.checkpoint import checkpoint

import dist_moe_b200 as dm
from tests.test_direct_execution_gpu import _Watch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
T, D, F, E, K = 9, 256, 128, 8, 2


def _inputs(seed, residual, D=D):
    g = torch.Generator().manual_seed(seed)
    x, w = torch.randn(T, D, generator=g).bfloat16(), 1 + 0.1 * torch.randn(D, generator=g)
    r = torch.randn(T, D, generator=g).to(residual or torch.bfloat16)
    return [t.to(DEV) for t in (x, r, w, 0.1 * torch.randn(E, D, generator=g))]


def _training(residual):
    def step(x, r, w, gate):
        leaves = [t.detach().requires_grad_() for t in (x, r, w, gate)]
        y, total = dm.add_rms_norm(leaves[0], leaves[2], residual_TD=leaves[1] if residual else None, gain_center=0.5)
        ids, scores = dm.select_experts(y.float() @ leaves[3].t(), K, renormalize=True)
        loss = (y.float() * scores.sum(1, keepdim=True)).sum() + (scores * ids).sum() + total.float().pow(2).sum()
        return (y, total, ids, scores) + torch.autograd.grad(loss, leaves if residual else [leaves[0], *leaves[2:]])

    return step


def _serving(context, w13, w2):
    def step(x, r, w, gate):
        with torch.no_grad():
            y, total, rows = dm.add_rms_norm(x, w, residual_TD=r, quantize=True)
            mask = torch.arange(len(x), device=DEV) != 2
            ids, scores = dm.select_experts((y.float() @ gate.t()).bfloat16(), K, score="sigmoid", bias_E=gate[:, 0].contiguous(),
                                            num_groups=4, num_kept_groups=2, token_mask_T=mask, scores_dtype=torch.bfloat16)
            return y, total, rows.dequantize(), ids, scores, dm.routed_experts_few_tokens(y, ids, scores, w13, w2, context)

    return step


@pytest.fixture
def serving():
    ctx = dm.create_context(group=None, device=DEV, config=dm.Config(
        max_num_local_input_tokens=T, hidden_dim=D, intermediate_dim=F, top_k=K, num_experts=E, max_moe_layers_per_activation_slot=1,
        inference=True))
    g = torch.Generator().manual_seed(1)
    w13, w2 = ((torch.randn(*s, generator=g) * s[-1] ** -0.5).bfloat16().to(DEV) for s in ((E, 2 * F, D), (E, D, F)))
    yield _serving(ctx, w13, w2)
    ctx.check_status()
    ctx.close()


def _equal(a, b):
    assert len(a) == len(b)
    for i, (p, q) in enumerate(zip(a, b)):
        assert p.dtype == q.dtype and torch.equal(p, q), i


TRAINING = ["add_rms_norm", "select_experts", "select_experts_backward", "add_rms_norm_backward"]
SERVING = ["add_rms_norm", "select_experts", "dequantize_mxfp8_rows", "routed_experts_few_tokens"]


def _operators(graph):
    return [n.target._schema.name.split("::")[1] for n in graph.graph.nodes if str(n.target).startswith("dist_moe.")]


@pytest.mark.parametrize("residual", [None, torch.bfloat16, torch.float32])
def test_a_traced_training_step(residual):
    step = _training(residual)
    graph = make_fx(step)(*_inputs(0, residual))
    assert sorted(_operators(graph)) == sorted(TRAINING)
    for seed in (0, 5):
        _equal(graph(*_inputs(seed, residual)), step(*_inputs(seed, residual)))


@pytest.mark.parametrize("tracer", ["make_fx", "jit"])
def test_a_traced_serving_step(serving, tracer):
    first, other = _inputs(0, torch.float32), _inputs(7, torch.float32)
    if tracer == "make_fx":
        traced = make_fx(serving)(*first)
        assert sorted(_operators(traced)) == sorted(SERVING)
    else:
        traced = torch.jit.trace(serving, first, check_trace=False)
        assert all(f"dist_moe::{name}" in str(traced.graph) for name in SERVING)
    for inputs in (first, other):
        _equal(traced(*inputs), serving(*inputs))


@pytest.mark.parametrize("residual", [None, torch.bfloat16, torch.float32])
def test_operators_equal_direct_calls(residual, serving):
    for step, names in ((_training(residual), TRAINING), (serving, SERVING)):
        for d in (D, 33) if names is TRAINING else (D,):
            inputs, watch = _inputs(3, residual, d), _Watch()
            with watch:
                through = step(*inputs)
            assert sorted(watch.seen) == sorted(names)
            _equal(through, step(*inputs))


def test_a_profiler_sees_them(serving):
    inputs = _inputs(3, torch.float32)
    with profile(activities=[ProfilerActivity.CPU]) as prof:
        seen = serving(*inputs)
    assert {f"dist_moe::{n}" for n in SERVING} <= {e.key for e in prof.key_averages()}
    _equal(seen, serving(*inputs))


@pytest.mark.parametrize("watched", [False, True])
def test_under_activation_checkpointing(watched):
    x, r, w, gate = (t.requires_grad_() for t in _inputs(4, torch.float32))

    def layer(x, r, w, gate):
        y, total = dm.add_rms_norm(x, w, residual_TD=r)
        return y.float() * dm.select_experts(y.float() @ gate.t(), K)[1].sum(1, keepdim=True) + total

    leaves = (x, r, w, gate)
    plain = torch.autograd.grad(layer(*leaves).sum(), leaves)
    out = checkpoint(layer, *leaves, use_reentrant=False)
    if watched:  # the repetition runs under a mode, the first forward did not
        with _Watch():
            again = torch.autograd.grad(out.sum(), leaves)
    else:
        again = torch.autograd.grad(out.sum(), leaves)
    _equal(again, plain)


def test_operators_refuse_what_the_calls_refuse():
    x, r, w, _ = _inputs(0, torch.float32)
    op = torch.ops.dist_moe
    with pytest.raises(ValueError, match="weight_D"):
        op.add_rms_norm(x, None, w[:-1], 1e-6, 0.0, False, False)
    with pytest.raises(ValueError, match="eps"):
        op.add_rms_norm(x, None, w, 0.0, 0.0, False, False)
    with pytest.raises(RuntimeError, match="kept"):
        op.add_rms_norm_backward(x, None, x, w[:-1], w[:T], 0.0, True, False, False)
    with pytest.raises(RuntimeError, match="match the sum"):
        op.add_rms_norm_backward(x[:1], None, x, w, w[:T], 0.0, True, False, False)
    with pytest.raises(ValueError, match="packed"):
        op.dequantize_mxfp8_rows(torch.zeros(3, 48, dtype=torch.uint8, device=DEV), 64)
    logits, ids = torch.randn(T, E, device=DEV), torch.zeros(T, K, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="top_k"):
        op.select_experts(logits, None, None, E + 1, "softmax", 1, 1, 2, False, 1.0, torch.int32, torch.float32)
    with pytest.raises(RuntimeError, match="match the logits"):
        op.select_experts_backward(logits, ids, logits, "softmax", False, 1.0)
    with pytest.raises(RuntimeError, match="not live"):
        op.routed_experts_few_tokens(x, ids, logits[:, :K].contiguous(), x, x, "no-such-context")


@pytest.mark.parametrize("mode", [torch.inference_mode, lambda: torch.device("cuda"), lambda: torch.autocast("cuda", dtype=torch.bfloat16)])
def test_under_modes_that_change_nothing(serving, mode):
    inputs = _inputs(3, torch.float32)
    want = serving(*inputs)
    for watched in (False, True):
        watch = _Watch()
        with mode():
            if watched:
                with watch:
                    got = serving(*inputs)
                assert sorted(watch.seen) == sorted(SERVING)
            else:
                got = serving(*inputs)
        if mode is torch.inference_mode:
            assert got[0].is_inference()
        _equal(got[:3], want[:3])  # autocast takes the router's product in bf16


def test_quantised_tokens_are_not_traced():
    ctx = dm.create_context(group=None, device=DEV, config=dm.Config(
        max_num_local_input_tokens=T, hidden_dim=D, intermediate_dim=F, top_k=K, num_experts=E, max_moe_layers_per_activation_slot=1,
        inference=True, block_scaled=dm.BlockScaledConfig()))
    w13, w2 = (torch.randn(*s, device=DEV).bfloat16() * 0.06 for s in ((E, 2 * F, D), (E, D, F)))
    ids, scores = torch.arange(K, device=DEV, dtype=torch.int32).expand(T, K).contiguous(), torch.rand(T, K, device=DEV)
    x, _, w, _ = _inputs(0, None)

    def call(x):
        with torch.no_grad():
            return dm.routed_experts(dm.add_rms_norm(x, w, quantize=True)[2], ids, scores, w13, w2, ctx)

    want = call(x)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(call)(x)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(call, (x,), check_trace=False)
    with _Watch(), profile(activities=[ProfilerActivity.CPU]):  # others do no harm
        assert torch.equal(call(x), want)
    ctx.check_status()
    ctx.close()


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_under_a_tracer_of_python_code(serving, backend):
    import torch._dynamo

    torch._dynamo.reset()
    inputs, compiled = _inputs(3, torch.float32), torch.compile(serving, backend=backend)
    _equal(compiled(*inputs), serving(*inputs))
    inputs = [t.requires_grad_() for t in inputs]

    def layer(x, r, w, gate):
        y, total = dm.add_rms_norm(x, w, residual_TD=r)
        return y.float() * dm.select_experts(y.float() @ gate.t(), K)[1].sum(1, keepdim=True) + total

    _equal(*(torch.autograd.grad(f(*inputs).sum(), inputs) for f in (torch.compile(layer, backend=backend), layer)))
    torch._dynamo.reset()
