"""Registered operators of what stands around the experts: names, shapes under fake tensors, and the nodes that a tracer of the public
calls sees (no GPU: a context is the shape facts that the checks read)."""

import types

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import dist_moe_b200 as dm
from dist_moe_b200 import _ops, api

OPS = ("add_rms_norm", "add_rms_norm_backward", "dequantize_mxfp8_rows", "select_experts", "select_experts_backward",
       "routed_experts_few_tokens")
BF, F32 = torch.bfloat16, torch.float32


def test_they_are_registered_beside_the_ten():
    assert sorted(_ops.AROUND) == sorted(OPS) and not set(OPS) & set(_ops.register())
    for name in OPS:
        schema = getattr(torch.ops.dist_moe, name).default._schema
        assert all(a.alias_info is None for a in schema.arguments) and all(r.alias_info is None for r in schema.returns)


@pytest.fixture
def context():
    ctx = object.__new__(dm.Context)
    ctx.config = dm.Config(max_num_local_input_tokens=100, hidden_dim=64, intermediate_dim=32, top_k=2, num_experts=4,
                           max_moe_layers_per_activation_slot=1, inference=True)
    ctx._closed, ctx._context_id = False, "test-around"
    ctx._state = types.SimpleNamespace(ep=1, e_local=4, device=torch.device("cuda", 0), few_workspace=object(), config=ctx.config)
    api._CONTEXTS[ctx._context_id] = ctx
    yield ctx
    api._CONTEXTS.pop(ctx._context_id)
    ctx._closed = True


def _nodes(graph):
    return [n.target._schema.name for n in graph.graph.nodes if n.op == "call_function" and hasattr(n.target, "_schema")]


@pytest.mark.parametrize("residual", [None, BF, F32])
@pytest.mark.parametrize("gain", [BF, F32])
def test_norm(residual, gain):
    with FakeTensorMode():
        x, w = torch.empty(5, 96, dtype=BF, device="cuda:0"), torch.empty(96, dtype=gain, device="cuda:0")
        r = None if residual is None else torch.empty(5, 96, dtype=residual, device="cuda:0")
        y, total = dm.add_rms_norm(x, w, residual_TD=r)
        assert y.shape == (5, 96) and y.dtype == BF and total.dtype == (residual or BF) and (r is not None or total is x)
        y, total, rows = dm.add_rms_norm(x, w, residual_TD=r, quantize=True)
        assert rows.packed.shape == (5, 112) and rows.dequantize().shape == (5, 96) and rows.dequantize().dtype == BF
        base = x if r is None else r  # what the norm kept
        for wanted in ((True, residual is F32, True), (False, False, False)):
            grads = torch.ops.dist_moe.add_rms_norm_backward(y, None if r is None else torch.empty_like(r), base, w,
                                                             torch.empty(5, device="cuda:0"), 0.0, *wanted)
            assert [(g.shape if want else g.numel(), g.dtype) for g, want in zip(grads, wanted)] == \
                [(t.shape if want else 0, t.dtype) for t, want in zip((y, base, w), wanted)]
    leaves = [t for t in (x, r, w) if t is not None]

    def step(*tensors):
        y, total = dm.add_rms_norm(tensors[0], tensors[-1], residual_TD=tensors[1] if r is not None else None)
        return y, total, dm.add_rms_norm(tensors[0].detach(), tensors[-1].detach(), quantize=True)[2].dequantize()

    for grad in (False, True):
        graph = make_fx(step, tracing_mode="fake")(*(t.detach().requires_grad_(grad) for t in leaves))
        assert [n for n in _nodes(graph) if n.startswith("dist_moe::")] == [
            "dist_moe::add_rms_norm", "dist_moe::add_rms_norm", "dist_moe::dequantize_mxfp8_rows"]
        assert not any("empty" in n for n in _nodes(graph))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_selection(dtype):
    with FakeTensorMode():
        logits, bias = torch.empty(5, 16, dtype=dtype, device="cuda:0"), torch.empty(16, device="cuda:0")
        mask = torch.empty(5, dtype=torch.bool, device="cuda:0")
        ids, scores = dm.select_experts(logits, 3, bias_E=bias, token_mask_T=mask, num_groups=4, num_kept_groups=2, ids_dtype=torch.int64,
                                        scores_dtype=BF)
        assert ids.shape == scores.shape == (5, 3) and ids.dtype == torch.int64 and scores.dtype == BF

        grad = torch.ops.dist_moe.select_experts_backward(logits, ids, scores, "softmax", False, 1.0)
        assert grad.shape == logits.shape and grad.dtype == dtype

    def step(l, b, m):
        return dm.select_experts(l, 3, score="sigmoid", bias_E=b, token_mask_T=m, renormalize=True)

    for grad in (False, True):
        graph = make_fx(step, tracing_mode="fake")(logits.detach().requires_grad_(grad), bias, mask)
        assert _nodes(graph) == ["dist_moe::select_experts"]


def test_few_tokens(context):
    with FakeTensorMode():
        args = [torch.empty(3, 64, dtype=BF, device="cuda:0"), torch.empty(3, 2, dtype=torch.int32, device="cuda:0"),
                torch.empty(3, 2, device="cuda:0"), torch.empty(4, 2, 32, 64, dtype=BF, device="cuda:0"),
                torch.empty(4, 64, 32, dtype=BF, device="cuda:0")]
        out = dm.routed_experts_few_tokens(*args, context)
        assert out.shape == (3, 64) and out.dtype == BF
        with pytest.raises(ValueError, match="hidden"):
            dm.routed_experts_few_tokens(*args[:4], args[4][:, :32], context)
    graph = make_fx(lambda *a: dm.routed_experts_few_tokens(*a, context), tracing_mode="fake")(*args)
    assert "dist_moe::routed_experts_few_tokens" in _nodes(graph)


class _OnDevice(torch.Tensor):
    """A CPU tensor that says it lies on a GPU."""

    device = torch.device("cuda", 0)


def test_rows_of_a_tensor_class_of_its_own_have_to_be_aligned_too():
    raw = torch.zeros(2 * 48 + 16, dtype=torch.uint8)
    first = -raw.data_ptr() % 16
    dm.QuantizedRows(raw[first:first + 96].view(2, 48).as_subclass(_OnDevice), 32)
    with pytest.raises(ValueError, match="aligned"):
        dm.QuantizedRows(raw[first + 8:first + 104].view(2, 48).as_subclass(_OnDevice), 32)
