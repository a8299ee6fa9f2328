"""``routed_experts_few_tokens`` against its definition in 64 bits.

Bound of an output value, u = 2^-24, b = 2^-8 (a bf16 rounding, relative): products and sums in 32 bits over D values, then over all
chosen experts' F values, at most (D + A F) u of the sum of absolute terms, A <= 8 here; the activation is rounded to bf16 once, b of every
term of the second sum; the output once more.  The terms' absolute sum S is taken of the 64-bit activations.  An activation's own
error enters through its derivative, below 1.1 for SwiGLU in either factor (2.5 clamped), times D u of the first sum's absolute terms:
below 2^-8 of S for D <= 7168 and random signs; it is counted as one more b."""

import pytest
import torch

import dist_moe_b200 as dm

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U, B = 2.0 ** -24, 2.0 ** -8


def _case(T, D, F, E, K, *, clamped=False, seed=0, scores_dtype=torch.float32, ids_dtype=torch.int32):
    g = torch.Generator().manual_seed(seed + 7 * T + D)
    x = torch.randn(T, D, generator=g).bfloat16().to(DEV)
    w13 = (torch.randn(E, 2 * F, D, generator=g) * D ** -0.5).bfloat16().to(DEV)
    w2 = (torch.randn(E, D, F, generator=g) * F ** -0.5).bfloat16().to(DEV)
    ids = torch.rand(T, E, generator=g).argsort(1)[:, :K].to(ids_dtype).to(DEV)
    scores = torch.rand(T, K, generator=g).to(scores_dtype).to(DEV)
    return x, ids, scores, w13, w2


def _context(T, D, F, E, K, clamped=False, **more):
    return dm.create_context(group=None, device=DEV, config=dm.Config(
        max_num_local_input_tokens=T, hidden_dim=D, intermediate_dim=F, top_k=K, num_experts=E, max_moe_layers_per_activation_slot=1,
        activation="swiglu_clamped" if clamped else "swiglu", **{"inference": True, **more}))


def _exact(x, ids, scores, w13, w2, clamped):
    out = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
    size = torch.zeros_like(out)
    F = w2.shape[2]
    for e in range(w13.shape[0]):
        share = torch.where(ids == e, scores.double(), 0.0).sum(1)
        hit = (ids == e).any(1)
        if not hit.any():
            continue
        h = x[hit].double() @ w13[e].double().t()
        gate, up = h[:, :F], h[:, F:]
        if clamped:
            gate = gate.clamp(max=7.0)
            h = gate * torch.sigmoid(1.702 * gate) * (up.clamp(-7.0, 7.0) + 1)
        else:
            h = gate * torch.sigmoid(gate) * up
        h = h * share[hit, None]
        out[hit] += h @ w2[e].double().t()
        size[hit] += h.abs() @ w2[e].double().abs().t()
    return out, size


def _check(got, case, clamped=False):
    x, ids, scores, w13, w2 = case
    want, size = _exact(x, ids, scores, w13, w2, clamped)
    D, F = x.shape[1], w2.shape[2]
    err = (got.double() - want).abs()
    bound = (2 * B + (D + 8 * F) * U) * size + B * want.abs() + 1e-30
    assert bool((err <= bound).all()), (err / bound).max().item()
    assert (err.norm() / want.norm().clamp_min(1e-30)) < 2 * B


# one token; a full tile of eight; one more; every tile count; features that end inside a strip and inner sizes that end inside a step;
# experts all hit, nearly none hit; a single expert
SIZES = [(1, 64, 8, 1, 1), (1, 256, 256, 8, 2), (1, 2048, 1408, 16, 6), (8, 128, 72, 4, 2), (9, 192, 104, 5, 3), (16, 1088, 704, 24, 3),
         (17, 320, 264, 16, 4), (32, 512, 328, 64, 6), (33, 256, 40, 3, 1), (61, 1088, 712, 24, 3), (64, 640, 512, 8, 8), (64, 64, 16, 300, 8),
         (4, 7168, 512, 8, 8), (2, 64, 2048, 4, 2)]


@pytest.mark.parametrize("T,D,F,E,K", SIZES)
@pytest.mark.parametrize("clamped", [False, True])
def test_against_the_definition(T, D, F, E, K, clamped):
    kinds = dict(scores_dtype=torch.bfloat16 if F % 3 else torch.float32, ids_dtype=torch.int64 if T % 2 else torch.int32)
    case = _case(T, D, F, E, K, **kinds)
    ctx = _context(T, D, F, E, K, clamped)
    got = dm.routed_experts_few_tokens(*case, ctx)
    _check(got, case, clamped)
    for _ in range(3):  # the same bits every time: parts of a strip are summed in order
        assert torch.equal(got, dm.routed_experts_few_tokens(*case, ctx))
    ctx.check_status()
    ctx.close()


def test_agrees_with_routed_experts():
    T, D, F, E, K = 24, 1024, 512, 16, 4
    case = _case(T, D, F, E, K)
    ctx = _context(T, D, F, E, K)
    few, whole = dm.routed_experts_few_tokens(*case, ctx), dm.routed_experts(*case, ctx)
    # the other rounds h1, h2 and every expert's output to bf16 as well: five roundings of size B / 2 on average-sized terms
    assert ((few.double() - whole.double()).norm() / whole.double().norm()).item() < 2 * B
    ctx.close()


def test_dropped_routes_repeated_experts_and_tokens_routed_nowhere():
    T, D, F, E, K = 13, 256, 136, 12, 4
    x, ids, scores, w13, w2 = _case(T, D, F, E, K)
    ctx = _context(T, D, F, E, K)
    ids[0] = -1
    ids[3, 1:] = -1
    ids[5] = 7                # the same expert four times
    ids[6, 2] = ids[6, 0]     # and twice
    scores[7] = 0.0
    case = (x, ids, scores, w13, w2)
    got = dm.routed_experts_few_tokens(*case, ctx)
    _check(got, case)
    assert not got[0].any() and not got[7].any()
    ids[:] = -1               # a padded batch
    got = dm.routed_experts_few_tokens(x, ids, scores, w13, w2, ctx)
    assert got.shape == x.shape and not got.any()
    ctx.check_status()
    # weights of experts that nobody is routed to are not looked at
    ids[:] = torch.arange(K, device=DEV).to(ids.dtype)
    case = (x, ids, scores, w13.clone(), w2.clone())
    case[3][K:], case[4][K:] = float("nan"), float("nan")
    assert torch.equal(dm.routed_experts_few_tokens(*case, ctx), dm.routed_experts_few_tokens(x, ids, scores, w13, w2, ctx))
    ctx.close()


def test_ids_outside_the_experts_are_reported_and_go_nowhere():
    T, D, F, E, K = 3, 128, 64, 4, 2
    x, ids, scores, w13, w2 = _case(T, D, F, E, K)
    ctx = _context(T, D, F, E, K)
    good = ids.clone()
    ids[1, 0], good[1, 0] = E, -1
    ids[2, 1], good[2, 1] = -5, -1
    got = dm.routed_experts_few_tokens(x, ids, scores, w13, w2, ctx)
    with pytest.raises(RuntimeError, match="expert id"):
        ctx.check_status()
    assert torch.equal(got, dm.routed_experts_few_tokens(x, good, scores, w13, w2, ctx))
    ctx.check_status()
    ctx.close()


def test_nonfinite_tokens_stay_with_themselves():
    T, D, F, E, K = 10, 128, 64, 4, 2
    case = _case(T, D, F, E, K)
    ctx = _context(T, D, F, E, K)
    clean = dm.routed_experts_few_tokens(*case, ctx)
    case[0][4, 9] = float("nan")
    got = dm.routed_experts_few_tokens(*case, ctx)
    keep = torch.arange(T) != 4
    assert got[4].isnan().all() and torch.equal(got[keep], clean[keep])
    ctx.close()


@pytest.mark.parametrize("T", [2, 8, 20])
@pytest.mark.parametrize("which", ["w13", "w2"])
def test_nonfinite_weights_reach_their_own_tokens_alone(T, which):
    D, F, E, K = 128, 72, 6, 2
    x, ids, scores, w13, w2 = _case(T, D, F, E, K)
    ids[:] = torch.tensor([0, 1], device=DEV, dtype=ids.dtype)
    ids[1] = torch.tensor([4, 2], device=DEV, dtype=ids.dtype)
    ctx = _context(T, D, F, E, K)
    clean = dm.routed_experts_few_tokens(x, ids, scores, w13, w2, ctx)
    w = (w13 if which == "w13" else w2).clone()
    w[4] = float("inf")
    got = dm.routed_experts_few_tokens(x, ids, scores, w if which == "w13" else w13, w2 if which == "w13" else w, ctx)
    keep = torch.arange(T) != 1
    assert not got[1].isfinite().any() and torch.equal(got[keep], clean[keep])
    ctx.close()


def test_fewer_tokens_than_the_context_holds_and_calls_in_turn():
    D, F, E, K = 256, 264, 16, 4
    ctx = _context(500, D, F, E, K)
    for T in (64, 1, 33, 8, 64):
        case = _case(T, D, F, E, K, seed=T)
        _check(dm.routed_experts_few_tokens(*case, ctx), case)
    training = _context(500, D, F, E, K, inference=False)
    case = _case(5, D, F, E, K)
    with torch.no_grad():
        assert torch.equal(dm.routed_experts_few_tokens(*case, training), dm.routed_experts_few_tokens(*case, ctx))
    small = _context(500, D, F, E, K, num_sms=3)
    _check(dm.routed_experts_few_tokens(*case, small), case)
    wide = [torch.cat([t, t], 1)[:, :t.shape[1]] for t in case[:3]]  # slices are copied
    assert torch.equal(dm.routed_experts_few_tokens(*wide, *case[3:], ctx), dm.routed_experts_few_tokens(*case, ctx))
    with pytest.raises(ValueError, match="contiguous"):
        dm.routed_experts_few_tokens(*case[:4], case[4].transpose(1, 2).contiguous().transpose(1, 2), ctx)
    w4 = case[3].view(E, 2, F, D)
    assert torch.equal(dm.routed_experts_few_tokens(*case[:3], w4, case[4], ctx), dm.routed_experts_few_tokens(*case, ctx))
    for c in (ctx, training, small):
        c.close()


def test_captured_calls_replay_on_new_tokens_between_eager_ones():
    T, D, F, E, K = 6, 512, 256, 8, 2
    x, ids, scores, w13, w2 = _case(T, D, F, E, K)
    ctx = _context(T, D, F, E, K)
    graphs, outs = [], []
    torch.cuda.synchronize()
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(dm.routed_experts_few_tokens(x, ids, scores, w13, w2, ctx))
        graphs.append(graph)
    for step in range(4):
        other = _case(T, D, F, E, K, seed=step)
        x.copy_(other[0]), ids.copy_(other[1]), scores.copy_(other[2])
        graphs[step % 2].replay()
        want = dm.routed_experts_few_tokens(x, ids, scores, w13, w2, ctx)
        graphs[step % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[step % 2], want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = dm.routed_experts_few_tokens(x, ids, scores, w13, w2, ctx)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, want)
    ctx.check_status()
    ctx.close()


def test_experts_that_lie_behind_32_bit_offsets():
    T, D, F, E, K, last = 6, 2048, 1408, 500, 3, 5
    case = _case(T, D, F, last, K)
    w13, w2 = (torch.empty(E, *t.shape[1:], device=DEV, dtype=t.dtype) for t in case[3:])
    w13[-last:], w2[-last:] = case[3], case[4]
    assert w13.numel() > 2 ** 31 and w2.numel() * 2 > 2 ** 31
    ctx, small = _context(T, D, F, E, K), _context(T, D, F, last, K)
    want = dm.routed_experts_few_tokens(*case, small)
    _check(want, case)
    assert torch.equal(dm.routed_experts_few_tokens(case[0], case[1] + (E - last), case[2], w13, w2, ctx), want)
    for c in (ctx, small):
        c.check_status()
        c.close()


@pytest.mark.parametrize("priority", [0, -1])
def test_contexts_at_the_same_time(priority):
    """Two contexts on two streams, beside products that hold SMs: every launch gets all of its blocks."""
    T, D, F, E, K = 12, 512, 1408, 16, 4
    cases = [_case(T, D, F, E, K, seed=i) for i in range(2)]
    contexts = [_context(T, D, F, E, K) for _ in cases]
    want = [dm.routed_experts_few_tokens(*case, ctx) for case, ctx in zip(cases, contexts)]
    a = torch.randn(2048, 2048, device=DEV).bfloat16()
    streams = [torch.cuda.Stream(), torch.cuda.Stream(priority=priority), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(50):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(dm.routed_experts_few_tokens(*cases[i], contexts[i]))
        with torch.cuda.stream(streams[2]):
            b = a @ a
    torch.cuda.synchronize()
    for i, ctx in enumerate(contexts):
        ctx.check_status()
        assert all(torch.equal(g, want[i]) for g in got[i])
        ctx.close()
    del b


def test_refusals_that_need_a_device():
    T, D, F, E, K = 4, 128, 64, 4, 2
    x, ids, scores, w13, w2 = _case(T, D, F, E, K)
    ctx = _context(100, D, F, E, K)
    with pytest.raises(ValueError, match="at most 64 tokens"):
        dm.routed_experts_few_tokens(x[:1].expand(65, -1).contiguous(), ids[:1].expand(65, -1).contiguous(),
                                     scores[:1].expand(65, -1).contiguous(), w13, w2, ctx)
    with pytest.raises(RuntimeError, match="forward-only"):
        dm.routed_experts_few_tokens(x.clone().requires_grad_(), ids, scores, w13, w2, ctx)
    with pytest.raises(ValueError, match="same CUDA device"):
        dm.routed_experts_few_tokens(x, ids.cpu(), scores, w13, w2, ctx)
    flat = torch.zeros(E * 2 * F * D + 1, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="16-byte"):
        dm.routed_experts_few_tokens(x, ids, scores, flat[1:].view(E, 2 * F, D), w2, ctx)
    moved = torch.zeros(T * D + 1, device=DEV, dtype=torch.bfloat16)[1:].view(T, D).copy_(x)  # tokens are copied instead
    assert torch.equal(dm.routed_experts_few_tokens(moved, ids, scores, w13, w2, ctx), dm.routed_experts_few_tokens(x, ids, scores, w13, w2, ctx))
    ctx.close()
    with pytest.raises(RuntimeError, match="closed"):
        dm.routed_experts_few_tokens(x, ids, scores, w13, w2, ctx)
    odd = _context(T, D, 60, E, K)  # rows of W2 that do not start on 16 bytes
    with pytest.raises(ValueError, match="multiples of 8"):
        dm.routed_experts_few_tokens(x, ids, scores, torch.zeros(E, 120, D, device=DEV, dtype=torch.bfloat16),
                                     torch.zeros(E, D, 60, device=DEV, dtype=torch.bfloat16), odd)
    odd.close()
