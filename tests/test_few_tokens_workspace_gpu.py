"""The workspace of calls of few tokens: nobody who does not make them holds it, and the first one may be a captured one."""

import pytest
import torch

import dist_moe_b200 as dm
from dist_moe_b200 import _few_tokens
from tests.test_few_tokens_gpu import _case, _check, _context

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
T, D, F, E, K = 6, 512, 256, 8, 2  # sizes that routed_experts takes too


@pytest.mark.parametrize("inference", [True, False])
def test_a_context_holds_none_before_its_first_call(inference):
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    ctx = _context(64, D, F, E, K, inference=inference)
    held = torch.cuda.memory_allocated() - before
    need = _few_tokens.workspace_bytes(ctx._state)
    case = _case(T, D, F, E, K)
    with torch.no_grad():
        dm.routed_experts(*case, ctx)
    assert ctx._state.few_workspace is None
    del case
    case = _case(T, D, F, E, K)
    at = torch.cuda.memory_allocated()
    with torch.no_grad():
        got = dm.routed_experts_few_tokens(*case, ctx)
    assert need <= torch.cuda.memory_allocated() - at <= need + (2 << 20)  # a block that was not split, and the output
    _check(got, case)
    ctx.check_status()
    ctx.close()
    assert held > 0 and ctx._state.few_workspace is None


def test_graphs_captured_before_the_first_call():
    x, ids, scores, w13, w2 = _case(T, D, F, E, K)
    ctx = _context(T, D, F, E, K)
    graphs, outs = [], []
    torch.cuda.synchronize()
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):  # two calls on the graph's workspace, with other allocations between them
            first = dm.routed_experts_few_tokens(x, ids, scores, w13, w2, ctx)
            filler = torch.full((1 << 21,), 3.0, device=DEV) * 2
            outs.append((first, dm.routed_experts_few_tokens(x, ids, scores, w13, w2, ctx), filler))
        graphs.append(graph)
    assert ctx._state.few_workspace is None
    for step in range(4):
        x.copy_(_case(T, D, F, E, K, seed=step)[0])
        graphs[step % 2].replay()
        want = dm.routed_experts_few_tokens(x, ids, scores, w13, w2, ctx)
        graphs[1 - step % 2].replay()
        torch.cuda.synchronize()
        for first, second, filler in outs:
            assert torch.equal(first, want) and torch.equal(second, want) and bool((filler == 6.0).all())
        _check(want, (x, ids, scores, w13, w2))
        if step == 1:
            ctx.reset()
    ctx.check_status()
    ctx.close()


def test_a_first_call_in_inference_mode():
    case = _case(T, D, F, E, K)
    ctx = _context(T, D, F, E, K)
    with torch.inference_mode():
        first = dm.routed_experts_few_tokens(*case, ctx)
    ctx.reset()
    case[1][0, 0] = E
    dm.routed_experts_few_tokens(*case, ctx)
    with pytest.raises(RuntimeError, match="expert id"):
        ctx.check_status()  # clears the counters as well
    case[1][0, 0] = _case(T, D, F, E, K)[1][0, 0]
    assert torch.equal(dm.routed_experts_few_tokens(*case, ctx), first)
    ctx.check_status()
    ctx.close()
