"""``select_experts`` against its definition in 64 bits.

Ids are exact.  Scores, u = 2^-24: exponential 2 u, a sum of E terms in at most E / 32 + 5 steps, quotient, scale and output: within
(E / 32 + 14) u of the exact value, relatively (a sigmoid's and a normalised softmax' sums are shorter); bf16 outputs add 2^-8.
Gradients: products of two such values and a sum of K of them, within 4 times that of the sum of the absolute terms."""

import numpy as np
import pytest
import torch

import dist_moe_b200 as dm

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:invalid value encountered")]  # inf - inf, not taken
DEV = torch.device("cuda", 0)
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: U}


def _definition(logits, K, *, score="softmax", bias_E=None, num_groups=1, num_kept_groups=1, group_top=2, renormalize=False, scale=1.0,
                token_mask_T=None, grad=None, **_):
    """ids, scores and the logits' gradient, row by row in numpy."""
    l = logits.detach().double().cpu().numpy()
    T, E = l.shape
    b = np.zeros(E) if bias_E is None else bias_E.double().cpu().numpy()
    ids, scores, dl, terms = np.full((T, K), -1), np.zeros((T, K)), np.zeros((T, E)), np.zeros((T, E))
    for t in range(T):
        if token_mask_T is not None and not token_mask_T[t]:
            continue
        row = np.where(np.isnan(l[t]), -np.inf, l[t])
        if score == "softmax":
            top = row.max()
            if top == -np.inf:
                continue
            z = np.where(row == top, 1.0, np.exp(np.where(row == top, 0.0, row - top)))
            p = z / z.sum()
        else:
            with np.errstate(over="ignore"):
                p = np.where(row < 0, np.exp(np.minimum(row, 0)) / (1 + np.exp(np.minimum(row, 0))), 1 / (1 + np.exp(-np.maximum(row, 0))))
        # without a bias the order of p is that of the logits, also where p cannot tell them apart
        c = np.where(row > -np.inf, p + b, -np.inf)
        c = np.where(np.isnan(c), -np.inf, c)
        order = c if bias_E is not None else row
        if num_groups > 1:
            size = E // num_groups
            values = []
            for i in range(num_groups):
                best = sorted([v for v in c[i * size:(i + 1) * size] if v > -np.inf], reverse=True)[:group_top]
                values.append(sum(best) if best else -np.inf)
            kept = sorted(range(num_groups), key=lambda i: (-values[i], i))[:num_kept_groups]
            order = np.where(np.isin(np.arange(E) // size, kept), order, -np.inf)
        chosen = [e for e in sorted(range(E), key=lambda e: (-order[e], e)) if order[e] > -np.inf][:K]
        if not chosen:
            continue
        n = len(chosen)
        ids[t, :n] = chosen
        v = p[chosen]
        if renormalize:
            rel = row[chosen]
            m = rel.max()
            e = np.where(rel == m, 1.0, np.exp(np.where(rel == m, 0.0, rel - m)))
            w = e if score == "softmax" else np.where(np.isinf(rel), 1.0, e / (1 + np.exp(np.minimum(rel, 700)))) if m < 0 else v
            w = w / w.sum()
        scores[t, :n] = scale * (w if renormalize else v)
        if grad is not None:
            g = scale * grad[t, :n].double().cpu().numpy()
            if renormalize:
                own = w * (g - (w * g).sum())
                size_of = w * (np.abs(g) + (w * np.abs(g)).sum())
                q = 1.0 if score == "softmax" else 1 - v
                dl[t, chosen], terms[t, chosen] = own * q, size_of * q
            elif score == "sigmoid":
                dl[t, chosen] = g * v * (1 - v)
                terms[t, chosen] = np.abs(g) * v * (1 - v)
            else:
                dl[t] = -p * (v * g).sum()
                terms[t] = p * (v * np.abs(g)).sum()
                dl[t, chosen] += v * g
                terms[t, chosen] += v * np.abs(g)
    return ids, scores, dl, terms


def _check(logits, K, *, ids_dtype=torch.int32, scores_dtype=torch.float32, **options):
    T, E = logits.shape
    leaf = logits.detach().requires_grad_()
    ids, scores = dm.select_experts(leaf, K, ids_dtype=ids_dtype, scores_dtype=scores_dtype, **options)
    assert ids.dtype == ids_dtype and scores.dtype == scores_dtype and ids.shape == scores.shape == (T, K)
    grad = torch.randn(T, K, device=DEV).to(scores_dtype)
    got, = torch.autograd.grad(scores, leaf, grad)
    w_ids, w_scores, w_dl, terms = _definition(logits, K, grad=grad, **options)
    assert np.array_equal(ids.cpu().numpy(), w_ids)
    steps = (E / 32 + 14) * U
    err = np.abs(scores.detach().double().cpu().numpy() - w_scores)
    assert (err <= (steps + HALF[scores_dtype]) * np.abs(w_scores) + 1e-37).all(), (err / np.maximum(np.abs(w_scores), 1e-30)).max()
    err = np.abs(got.double().cpu().numpy() - w_dl)
    bound = 4 * steps * terms + HALF[logits.dtype] * np.abs(w_dl) + 1e-37
    assert (err <= bound).all(), (err / bound).max()
    with torch.no_grad():
        again = dm.select_experts(logits, K, ids_dtype=ids_dtype, scores_dtype=scores_dtype, **options)
    assert torch.equal(again[0], ids) and torch.equal(again[1], scores)


def _logits(T, E, dtype=torch.float32, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(T * 31 + E + seed)
    return (torch.randn(T, E, generator=g) * spread).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("T,E,K", [(1, 1, 1), (1, 64, 6), (5, 2, 2), (33, 24, 3), (7, 33, 32), (130, 128, 8), (9, 256, 8), (6, 511, 5), (3, 1024, 32)])
def test_plain(T, E, K, score, renormalize, dtype):
    _check(_logits(T, E, dtype), K, score=score, renormalize=renormalize, scale=1.5 if T % 2 else 1.0,
           ids_dtype=torch.int64 if E % 2 else torch.int32, scores_dtype=torch.bfloat16 if E == 24 else torch.float32)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("T,E,K,groups,kept,top", [(40, 256, 8, 8, 4, 2), (40, 256, 8, 8, 4, 1), (11, 24, 3, 3, 2, 2), (9, 96, 5, 32, 7, 2),
                                                  (5, 10, 2, 5, 1, 2), (6, 12, 1, 12, 3, 2), (4, 1024, 8, 2, 1, 1), (8, 60, 4, 4, 4, 2)])
def test_groups_and_bias(T, E, K, groups, kept, top, score, biased):
    bias = torch.randn(E, generator=torch.Generator().manual_seed(E)).to(DEV) * 0.1 if biased else None
    _check(_logits(T, E), K, score=score, bias_E=bias, num_groups=groups, num_kept_groups=kept, group_top=top, renormalize=biased)


def test_equal_values_go_to_the_lowest_index():
    logits = torch.zeros(3, 100, device=DEV)
    logits[1, 40:] = 1.0
    logits[2, ::3] = -0.0
    ids, scores = dm.select_experts(logits, 4)
    assert ids.tolist() == [[0, 1, 2, 3], [40, 41, 42, 43], [0, 1, 2, 3]]
    ids, _ = dm.select_experts(logits, 4, bias_E=torch.zeros(100, device=DEV), num_groups=4, num_kept_groups=2)
    assert ids.tolist() == [[0, 1, 2, 3], [40, 41, 42, 43], [0, 1, 2, 3]]
    _check(logits, 4, bias_E=torch.zeros(100, device=DEV), num_groups=4, num_kept_groups=2)
    _check(_logits(50, 64, torch.bfloat16, spread=0.02), 8, bias_E=torch.zeros(64, device=DEV))  # many equal logits


# few experts near one another; more than a warp has lanes; as many chosen as a warp has lanes
@pytest.mark.parametrize("E,K", [(24, 6), (48, 6), (66, 32)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_values_that_32_bits_cannot_tell_apart(score, E, K):
    """Choices that hang on differences far below an fp32 unit of c: they are made in 64 bits."""
    g = torch.Generator().manual_seed(1)
    T = 64
    logits = torch.randn(T, 1, generator=g).expand(T, E).clone()
    logits += torch.randint(-3, 4, (T, E), generator=g) * 2.0 ** -22  # neighbours in fp32
    bias = torch.randint(0, 2, (E,), generator=g) * 2.0 ** -26
    logits, bias = logits.to(DEV), bias.to(DEV)
    _check(logits, K, score=score, bias_E=bias)
    _check(logits, K, score=score, bias_E=bias, num_groups=6, num_kept_groups=3)
    _check(logits, K, score=score, num_groups=6, num_kept_groups=3)
    logits[:, ::5] += 1.0  # some stand clear
    _check(logits, K, score=score, bias_E=bias)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_masks_infinities_and_nan(score, renormalize):
    inf, nan = float("inf"), float("nan")
    logits = _logits(9, 40)
    logits[0] = -inf                      # nothing left
    logits[1, 1:] = -inf                  # one left
    logits[2, ::2] = nan
    logits[3, 5] = inf
    logits[4, [7, 30]] = inf
    logits[5] = nan
    logits[6] = torch.finfo(torch.float32).min
    logits[7, 3] = torch.finfo(torch.float32).max
    mask = torch.ones(9, dtype=torch.bool, device=DEV)
    mask[8] = False
    options = dict(score=score, renormalize=renormalize, token_mask_T=mask)
    ids, scores = dm.select_experts(logits, 3, **options)
    w_ids, w_scores, _, _ = _definition(logits, 3, **options)
    assert np.array_equal(ids.cpu().numpy(), w_ids)
    np.testing.assert_allclose(scores.cpu().numpy(), w_scores, rtol=20 * U, atol=1e-37)
    assert ids[0].tolist() == ids[8].tolist() == [-1] * 3 and ids[1].tolist() == [0, -1, -1] and not scores[[0, 8]].any()
    bias = torch.zeros(40, device=DEV)
    bias[:20], bias[20], bias[21] = -inf, nan, inf
    ids, scores = dm.select_experts(logits, 3, bias_E=bias, num_groups=4, num_kept_groups=3, **options)
    w_ids, w_scores, _, _ = _definition(logits, 3, bias_E=bias, num_groups=4, num_kept_groups=3, **options)
    assert np.array_equal(ids.cpu().numpy(), w_ids) and scores.isfinite().all()
    leaf = logits.clone().requires_grad_()
    g, = torch.autograd.grad(dm.select_experts(leaf, 3, **options)[1].sum(), leaf)
    assert g.isfinite().all() and not g[8].any() and not g[0].any() and not g[2, ::2].any()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_normalised_scores_of_far_logits(score):
    """All chosen probabilities underflow in 32 bits; their shares do not.  (Beside a bias of 5 they are equal in 64 bits too.)"""
    logits = torch.full((2, 8), -200.0, device=DEV)
    logits[:, 3], logits[:, 5], logits[1, 0] = -199.0, -198.0, 90.0
    bias = torch.zeros(8, device=DEV)
    bias[3] = bias[5] = 5.0
    _check(logits, 2, score=score, renormalize=True, bias_E=bias)


def test_gradients_agree_with_differences():
    logits = _logits(2, 12)
    g = torch.randn(2, 3, device=DEV)
    for score in ("softmax", "sigmoid"):
        for renormalize in (False, True):
            options = dict(score=score, renormalize=renormalize)
            leaf = logits.clone().requires_grad_()
            ids, scores = dm.select_experts(leaf, 3, **options)
            got, = torch.autograd.grad(scores, leaf, g)

            def value(l):
                p = torch.softmax(l, 1) if score == "softmax" else torch.sigmoid(l)
                v = p.gather(1, ids.long())
                return ((v / v.sum(1, keepdim=True) if renormalize else v) * g.double()).sum()

            for i in range(24):
                up, down = logits.double().clone(), logits.double().clone()
                up.view(-1)[i] += 1e-5
                down.view(-1)[i] -= 1e-5
                assert abs((value(up) - value(down)).item() / 2e-5 - got.reshape(-1)[i].item()) < 1e-6


def test_layouts_streams_capture_and_no_tokens():
    wide = _logits(20, 200)
    view, mask = wide[:, 3:131], torch.rand(40, device=DEV) > 0.3
    plain = dm.select_experts(view.contiguous(), 8, token_mask_T=mask[::2].contiguous())
    for got in (dm.select_experts(view, 8, token_mask_T=mask[::2]), dm.select_experts(view.t().contiguous().t(), 8, token_mask_T=mask[::2])):
        assert torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1])
    leaf = wide.clone().requires_grad_()
    g = torch.randn(20, 8, device=DEV)
    strided, = torch.autograd.grad(dm.select_experts(leaf[:, 3:131], 8)[1], leaf, g)
    dense_leaf = view.contiguous().requires_grad_()
    dense, = torch.autograd.grad(dm.select_experts(dense_leaf, 8)[1], dense_leaf, g)
    assert torch.equal(strided[:, 3:131], dense) and not strided[:, :3].any()
    ids, scores = dm.select_experts(torch.empty(0, 16, device=DEV), 2)
    assert ids.shape == scores.shape == (0, 2)
    logits = _logits(20, 128)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = dm.select_experts(logits, 8)
    logits.copy_(_logits(20, 128, seed=9))
    graph.replay()
    want = dm.select_experts(logits, 8)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_rows_behind_32_bit_offsets():
    E, K, last = 1024, 8, 7
    T = 2 ** 31 // E + 100
    logits = torch.zeros(T, E, device=DEV, dtype=torch.bfloat16)
    logits[-last:] = torch.randn(last, E, device=DEV)
    few = logits[-last:].clone()
    got = []
    for l in (logits, few):
        l.requires_grad_()
        ids, scores = dm.select_experts(l, K)
        grad, = torch.autograd.grad(scores, l, torch.ones_like(scores))
        got.append([t[-last:].clone() for t in (ids, scores, grad)])
        del ids, scores, grad
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_gradients_are_not_differentiated_again():
    logits = torch.randn(5, 16, device=DEV, requires_grad=True)
    loss = dm.select_experts(logits, 4)[1].pow(2).sum()
    first, = torch.autograd.grad(loss, logits, retain_graph=True)
    again, = torch.autograd.grad(loss, logits, create_graph=True)
    assert torch.equal(first, again) and again.requires_grad
    with pytest.raises(RuntimeError, match="differentiate twice"):
        again.sum().backward()
