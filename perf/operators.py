"""Performance cases of the operators around the routed experts of one layer: what stands in front of them and their form for a
few tokens.

* ``add_rms_norm``: the residual's addition and the RMS norm whose output the router and the experts read, as bf16 tokens and, for
  MXFP8 experts, as quantised rows; training returns the gradients of tokens, residual and gain;
* ``select_experts``: expert ids and scores of every token from the router's logits; training returns the logits' gradient;
* ``routed_experts_few_tokens``: the whole routed-expert layer for a decode step of up to 64 tokens.

Sizes come from the configurations that this repository's benchmark and tests name, plus ragged ones of the same ranges.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
EPS = 1e-6
ALPHA, LIMIT = 1.702, 7.0  # clamped SwiGLU
_MAX_PLAIN_BYTES = 12 << 30  # 32-bit weights that a plain pass may hold
_MAX_WEIGHT_BYTES = 4 << 30


def _norm(name=None, *, T, D, residual="bfloat16", gain="bfloat16", center=0.0, rows=False, train=False):
    case = dict(op="norm", T=T, D=D, residual=residual, gain=gain, center=center, rows=rows, train=train)
    return {"name": name, **case} if name else case


def _select(name=None, *, T, E, K, score="softmax", bias=False, groups=1, kept=1, renormalize=False, scale=1.0, masked=False,
            logits="float32", scores="float32", ids="int32", train=False):
    case = dict(op="select", T=T, E=E, K=K, score=score, bias=bias, groups=groups, kept=kept, renormalize=renormalize, scale=scale,
                masked=masked, logits=logits, scores=scores, ids=ids, train=train)
    return {"name": name, **case} if name else case


def _few(name=None, *, T, D, F, E, K, clamped=False, scores="float32", ids="int32", dropped=False, skewed=False):
    case = dict(op="few", T=T, D=D, F=F, E=E, K=K, clamped=clamped, scores=scores, ids=ids, dropped=dropped, skewed=skewed)
    return {"name": name, **case} if name else case


def listed():
    return [
        # a decode step of 16 sequences: one short launch, latency counts
        _norm("norm-decode", T=16, D=2048),
        # prefill in front of MXFP8 experts: tokens for the router, quantised rows for the experts, 32-bit residual stream
        _norm("norm-prefill-rows", T=4096, D=2816, residual="float32", rows=True),
        # fine-tuning on a ragged batch: 32-bit residual and gain, gain stored around zero
        _norm("norm-train-ragged", T=1531, D=1088, residual="float32", gain="float32", center=1.0, train=True),
        # a training step's micro-batch, two sequences of 8192 tokens
        _norm("norm-train", T=16384, D=4096, train=True),
        # a decode step of 32 sequences
        _select("select-decode", T=32, E=64, K=6),
        # prefill of 4096 tokens with 256 experts in groups, balanced by a bias; padding tokens routed nowhere
        _select("select-groups", T=4096, E=256, K=8, score="sigmoid", bias=True, groups=8, kept=4, renormalize=True, scale=1.5,
                masked=True),
        # fine-tuning on a ragged batch, logits and scores as the model's product leaves them
        _select("select-train-ragged", T=1531, E=24, K=3, score="sigmoid", renormalize=True, logits="bfloat16", scores="bfloat16",
                ids="int64", train=True),
        # a training step's micro-batch
        _select("select-train", T=16384, E=128, K=8, train=True),
        # decoding one sequence
        _few("few-one-token", T=1, D=2048, F=1408, E=64, K=6),
        # decoding a batch of 32 sequences: nearly every expert is hit
        _few("few-batch", T=32, D=2048, F=1408, E=64, K=6),
        # four sequences on one rank's experts of a large layer
        _few("few-large-layer", T=4, D=7168, F=2048, E=32, K=8),
        # a padded batch on ragged sizes, clamped activation, skewed experts
        _few("few-ragged", T=61, D=1088, F=712, E=24, K=3, clamped=True, scores="bfloat16", ids="int64", dropped=True, skewed=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ranges."""
    bound = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("norm", "select", "few")}
    while True:
        op = rng.choice(["norm", "select", "few"])
        if op == "norm":
            rows, train = rng.choice([(False, False), (True, False), (False, True)])
            D = rng.choice([128 * rng.randint(1, 56), 64 * rng.randint(1, 112), rng.randint(33, 5000)])
            case = _norm(T=_log_int(rng, 1, 16384), D=-(-D // 128) * 128 if rows else D, residual=rng.choice(["bfloat16", "float32"]),
                         gain=rng.choice(["bfloat16", "float32"]), center=rng.choice([0.0, 1.0]), rows=rows, train=train)
        elif op == "select":
            groups = rng.choice([1, 1, 2, 4, 8])
            E = groups * rng.randint(2, 256 // groups)
            kept = rng.randint(1, groups)
            K = rng.randint(1, min(8, kept * (E // groups)))
            case = _select(T=_log_int(rng, 1, 16384), E=E, K=K, score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.4,
                           groups=groups, kept=kept, renormalize=rng.random() < 0.5, scale=rng.choice([1.0, 1.5]),
                           masked=rng.random() < 0.3, logits=rng.choice(["float32", "bfloat16"]),
                           scores=rng.choice(["float32", "float32", "bfloat16"]), ids=rng.choice(["int32", "int64"]),
                           train=rng.random() < 0.5)
        else:
            E = rng.randint(4, 64)
            case = _few(T=_log_int(rng, 1, 64), D=64 * _log_int(rng, 4, 112), F=8 * _log_int(rng, 16, 256), E=E,
                        K=rng.randint(1, min(8, E // 2)), clamped=rng.random() < 0.3, scores=rng.choice(["float32", "bfloat16"]),
                        ids=rng.choice(["int32", "int64"]), dropped=rng.random() < 0.3, skewed=rng.random() < 0.3)
            if case["E"] * 6 * case["D"] * case["F"] > _MAX_WEIGHT_BYTES or _plain_bytes(case) > _MAX_PLAIN_BYTES:
                continue
        if _cost(case) <= bound[op]:
            return case


def _plain_bytes(case):
    return min(case["T"] * case["K"], case["E"]) * 12 * case["D"] * case["F"]


def _cost(case):
    w = work(case)
    return w["bytes"] + w["flops"] / 200.0


def _size(dtype):
    return getattr(torch, dtype).itemsize


def work(case):
    """Each input read once, each output written once; for the few tokens the weights of the experts that are hit on average."""
    if case["op"] == "norm":
        n, D, r = case["T"] * case["D"], case["D"], _size(case["residual"])
        nbytes, flops = n * (2 + r + 2 + r) + D * _size(case["gain"]), 6 * n
        if case["rows"]:
            nbytes, flops = nbytes + n * (1 + 1 / 32), flops + 3 * n
        if case["train"]:  # gradients of both outputs and the sum in, gradients of both inputs out
            nbytes, flops = nbytes + n * (2 + r + r + 2 + r) + 2 * D * _size(case["gain"]), flops + 12 * n
        return {"bytes": nbytes, "flops": flops}
    T, E, K = case["T"], case["E"], case["K"]
    routes = T * K * (_size(case["ids"]) + _size(case["scores"]))
    if case["op"] == "select":
        row = T * E * _size(case["logits"])
        nbytes = row + routes + (4 * E if case["bias"] else 0) + (T if case["masked"] else 0)
        flops = 6 * T * E
        if case["train"]:
            nbytes, flops = nbytes + (2 * row if case["score"] == "softmax" and not case["renormalize"] else row) \
                + routes, flops + 6 * T * E
        return {"bytes": nbytes, "flops": flops}
    D, F = case["D"], case["F"]
    hit = E * (1.0 - (1.0 - K / E) ** T)
    if case["skewed"]:
        hit *= 0.8
    return {"bytes": hit * 6 * D * F + 4 * T * D + routes, "flops": 6 * T * K * D * F}


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32) * scale).to(dtype)

    T = case["T"]
    s = dict(case)
    if case["op"] == "norm":
        D, train = case["D"], case["train"]
        residual, gain = getattr(torch, case["residual"]), getattr(torch, case["gain"])
        # the stream is wider than what one layer adds to it, and every token has a scale of its own
        spread = torch.exp(torch.randn(T, 1, generator=g, device=DEVICE) * 0.5)
        s["x"] = (torch.randn(T, D, generator=g, device=DEVICE) * 0.7 * spread).bfloat16().requires_grad_(train)
        s["residual_TD"] = (torch.randn(T, D, generator=g, device=DEVICE) * 2.0 * spread).to(residual).requires_grad_(train)
        s["weight"] = (1.0 - case["center"] + normal(D, scale=0.1)).to(gain).requires_grad_(train)
        if train:
            s["grad_y"], s["grad_sum"] = normal(T, D, dtype=torch.bfloat16), normal(T, D, dtype=residual)
        return s
    E, K = case["E"], case["K"]
    ids_dtype, scores_dtype = getattr(torch, case["ids"]), getattr(torch, case["scores"])
    if case["op"] == "select":
        popularity = normal(E, scale=0.5)
        s["l"] = (normal(T, E, scale=1.5) + popularity).to(getattr(torch, case["logits"])).requires_grad_(case["train"])
        s["bias_E"] = -0.1 * popularity if case["bias"] else None
        s["mask"] = torch.rand(T, generator=g, device=DEVICE) > 0.1 if case["masked"] else None
        if case["train"]:
            s["grad_scores"] = normal(T, K, dtype=scores_dtype)
        return s
    D, F = case["D"], case["F"]
    s["x"] = normal(T, D, dtype=torch.bfloat16)
    s["w13"] = torch.empty(E, 2 * F, D, device=DEVICE, dtype=torch.bfloat16)
    s["w2"] = torch.empty(E, D, F, device=DEVICE, dtype=torch.bfloat16)
    for w, fan in ((s["w13"], D), (s["w2"], F)):
        w.normal_(0.0, fan ** -0.5, generator=g)
    key = torch.rand(T, E, generator=g, device=DEVICE)
    if case["skewed"]:  # the first eighth of the experts takes part in every other choice
        key[:, :max(1, E // 8)] += 0.5
    ids = key.argsort(dim=1, descending=True)[:, :K]
    scores = torch.softmax(normal(T, K), dim=1)
    if case["dropped"]:  # padding tokens, and routes that the router left out
        ids = torch.where((torch.rand(T, 1, generator=g, device=DEVICE) < 0.1) | (torch.rand(T, K, generator=g, device=DEVICE) < 0.1),
                          torch.full_like(ids, -1), ids)
    s["ids_TK"], s["scores_TK"] = ids.to(ids_dtype), scores.to(scores_dtype)
    if own:  # a program makes its context once
        import dist_moe_b200 as dm

        s["context"] = dm.create_context(group=None, device=DEVICE, config=dm.Config(
            max_num_local_input_tokens=T, hidden_dim=D, intermediate_dim=F, top_k=K, num_experts=E,
            max_moe_layers_per_activation_slot=1, inference=True, activation="swiglu_clamped" if case["clamped"] else "swiglu",
            swiglu_alpha=ALPHA, swiglu_limit=LIMIT))
    return s


def run(s):
    return _RUN[s["op"]](s)


# ---- add_rms_norm ------------------------------------------------------------------------------------------
def _run_norm(s):
    x, r, w = s["x"], s["residual_TD"], s["weight"]
    if own:
        import dist_moe_b200 as dm

        if s["rows"]:
            y, total, rows = dm.add_rms_norm(x, w, residual_TD=r, eps=EPS, gain_center=s["center"], quantize=True)
            return {"y": y, "sum": total, "rows": rows.dequantize()}
        y, total = dm.add_rms_norm(x, w, residual_TD=r, eps=EPS, gain_center=s["center"])
        if not s["train"]:
            return {"y": y, "sum": total}
        gx, gr, gw = torch.autograd.grad((y, total), (x, r, w), (s["grad_y"], s["grad_sum"]))
        return {"y": y, "sum": total, "grad_x": gx, "grad_residual": gr, "grad_weight": gw}
    with torch.no_grad():
        total = (x.float() + r.float()).to(r.dtype)
        t, gain = total.float(), w.float() + s["center"]
        rstd = torch.rsqrt((t * t).mean(dim=1, keepdim=True) + EPS)
        y = (t * rstd * gain).bfloat16()
        out = {"y": y, "sum": total}
        if s["rows"]:
            blocks = y.float().view(s["T"], -1, 32)
            # the smallest power of two that brings a block's largest value down to 448
            mantissa, exponent = torch.frexp(blocks.abs().amax(dim=2, keepdim=True) * (1.0 / 448.0))
            scale = torch.where(mantissa == 0.5, exponent - 1, exponent).clamp(min=-127)
            q = torch.ldexp(blocks, -scale).to(torch.float8_e4m3fn)
            out["rows"] = torch.ldexp(q.float(), scale).view(s["T"], -1).bfloat16()
        if s["train"]:
            gy = s["grad_y"].float()
            u = gy * gain
            g = s["grad_sum"].float() + rstd * (u - t * (rstd * rstd) * (u * t).mean(dim=1, keepdim=True))
            out["grad_x"], out["grad_residual"] = g.bfloat16(), g.to(r.dtype)
            out["grad_weight"] = (gy * t * rstd).sum(dim=0).to(w.dtype)
        return out


# ---- select_experts ----------------------------------------------------------------------------------------
def _run_select(s):
    l, K = s["l"], s["K"]
    ids_dtype, scores_dtype = getattr(torch, s["ids"]), getattr(torch, s["scores"])
    if own:
        import dist_moe_b200 as dm

        ids, scores = dm.select_experts(l, K, score=s["score"], bias_E=s["bias_E"], num_groups=s["groups"], num_kept_groups=s["kept"],
                                        renormalize=s["renormalize"], scale=s["scale"], token_mask_T=s["mask"], ids_dtype=ids_dtype,
                                        scores_dtype=scores_dtype)
        if not s["train"]:
            return {"ids": ids, "scores": scores}
        return {"ids": ids, "scores": scores, "grad_logits": torch.autograd.grad(scores, l, s["grad_scores"])[0]}
    with torch.no_grad():
        x = l.double()  # 64 bits: what is compared may lie next to a border
        p = torch.softmax(x, dim=1) if s["score"] == "softmax" else torch.sigmoid(x)
        choice = p + s["bias_E"].double() if s["bias_E"] is not None else p
        if s["groups"] > 1:
            grouped = choice.view(s["T"], s["groups"], -1)
            best = grouped.sort(dim=2, descending=True).values[:, :, :2].sum(dim=2)
            kept = best.sort(dim=1, descending=True, stable=True).indices[:, :s["kept"]]
            keep = torch.zeros_like(best, dtype=torch.bool).scatter_(1, kept, True)
            choice = torch.where(keep[:, :, None], grouped, -math.inf).view(s["T"], -1)
        ids = choice.sort(dim=1, descending=True, stable=True).indices[:, :K]
        p = p.float()
        v = p.gather(1, ids)
        total = v.sum(dim=1, keepdim=True)
        scores = s["scale"] * (v / total if s["renormalize"] else v)
        live = s["mask"][:, None] if s["mask"] is not None else torch.ones_like(ids[:, :1], dtype=torch.bool)
        out = {"ids": torch.where(live, ids, -1).to(ids_dtype), "scores": torch.where(live, scores, 0.0).to(scores_dtype)}
        if s["train"]:
            dv = torch.where(live, s["scale"] * s["grad_scores"].float(), 0.0)
            if s["renormalize"]:
                dv = (dv - (dv * v).sum(dim=1, keepdim=True) / total) / total
            dp = torch.zeros_like(p).scatter_(1, ids, dv)
            dl = p * (dp - (p * dp).sum(dim=1, keepdim=True)) if s["score"] == "softmax" else dp * p * (1.0 - p)
            out["grad_logits"] = dl.to(l.dtype)
        return out


# ---- routed_experts_few_tokens -----------------------------------------------------------------------------
def _run_few(s):
    x, ids, scores, w13, w2 = s["x"], s["ids_TK"], s["scores_TK"], s["w13"], s["w2"]
    T, D, F, E, K = (s[k] for k in "TDFEK")
    if own:
        import dist_moe_b200 as dm

        return dm.routed_experts_few_tokens(x, ids, scores, w13, w2, s["context"])
    xf, c = x.float(), torch.where(ids >= 0, scores.float(), 0.0)
    if T * K <= E:  # the routes' own weights
        e = ids.clamp(min=0).long().view(-1)
        rows = xf.repeat_interleave(K, dim=0)
        h1 = torch.matmul(w13[e].float(), rows[:, :, None])[:, :, 0]
        h2 = _activate(h1[:, :F], h1[:, F:], s["clamped"]) * c.view(-1, 1)
        return torch.matmul(w2[e].float(), h2[:, :, None])[:, :, 0].view(T, K, D).sum(dim=1).bfloat16()
    coefficient = torch.zeros(T, E, device=x.device).scatter_add_(1, ids.clamp(min=0).long(), c)
    h1 = torch.matmul(xf, w13.float().transpose(1, 2))  # [E, T, 2F]
    h2 = _activate(h1[:, :, :F], h1[:, :, F:], s["clamped"]) * coefficient.t()[:, :, None]
    return torch.matmul(h2, w2.float().transpose(1, 2)).sum(dim=0).bfloat16()


def _activate(gate, up, clamped):
    if clamped:
        gate = gate.clamp(max=LIMIT)
        return gate / (1.0 + torch.exp(-ALPHA * gate)) * (up.clamp(-LIMIT, LIMIT) + 1.0)
    return gate / (1.0 + torch.exp(-gate)) * up


_RUN = {"norm": _run_norm, "select": _run_select, "few": _run_few}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------
def exact(case, seed):
    return _EXACT[case["op"]](prepare(case, seed))


def _exact_norm(s):
    with torch.no_grad():
        r = s["residual_TD"]
        total = (s["x"].double() + r.double()).to(r.dtype)  # the stream is what is normalised, as it is stored
        a = total.double()
        length = ((a ** 2).sum(1) / s["D"] + EPS).sqrt()
        unit = a / length[:, None]
        gain = s["weight"].double() + s["center"]
        y = unit * gain
        out = {"y": y, "sum": total.double()}
        if s["rows"]:
            b = y.bfloat16().double().reshape(-1, 32).cpu().numpy()
            top = np.abs(b).max(axis=1)
            scale = np.exp2(np.ceil(np.log2(np.where(top > 0, top, 448.0 * 2.0 ** -127) / 448.0)))[:, None]
            step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(np.abs(b / scale), 2.0 ** -20))), -6.0) - 3.0)
            q = np.rint(b / scale / step) * step * scale
            out["rows"] = torch.from_numpy(q).reshape(s["T"], s["D"])
        if s["train"]:
            gy = s["grad_y"].double()
            u = gy * gain
            g = s["grad_sum"].double() + (u - unit * ((u * unit).sum(1) / s["D"])[:, None]) / length[:, None]
            out["grad_x"] = out["grad_residual"] = g
            out["grad_weight"] = (gy * unit).sum(0)
        return out


def _exact_select(s):
    l = s["l"].detach().double().cpu().numpy()
    T, E, K, G = s["T"], s["E"], s["K"], s["groups"]
    rows = np.arange(T)[:, None]
    if s["score"] == "softmax":
        p = np.exp(l - l.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
    else:
        p = 1.0 / (1.0 + np.exp(-l))
    c = p if s["bias_E"] is None else p + s["bias_E"].double().cpu().numpy()
    if G > 1:
        by_group = np.sort(c.reshape(T, G, E // G), axis=2)[:, :, ::-1]
        order = np.argsort(-by_group[:, :, :2].sum(2), axis=1, kind="stable")
        rank = np.empty_like(order)
        rank[rows, order] = np.arange(G)[None]
        c = np.where(np.repeat(rank < s["kept"], E // G, axis=1), c, -np.inf)
    ids = np.argsort(-c, axis=1, kind="stable")[:, :K]
    v = p[rows, ids]
    weight = v / v.sum(1, keepdims=True) if s["renormalize"] else v
    live = np.ones(T, bool) if s["mask"] is None else s["mask"].cpu().numpy()
    scores = np.where(live[:, None], s["scale"] * weight, 0.0)
    out = {"ids": np.where(live[:, None], ids, -1), "scores": scores}
    if s["train"]:
        ds = np.where(live[:, None], s["scale"] * s["grad_scores"].double().cpu().numpy(), 0.0)
        if s["renormalize"]:
            ds = (ds - (ds * weight).sum(1, keepdims=True)) / v.sum(1, keepdims=True)
        dl = np.zeros((T, E))
        if s["score"] == "softmax":
            dl -= p * (ds * v).sum(1, keepdims=True)
            dl[rows, ids] += ds * v
        else:
            dl[rows, ids] = ds * v * (1.0 - v)
        out["grad_logits"] = dl
    return out


def _exact_few(s):
    x = s["x"].double()
    out = torch.zeros_like(x)
    for e in range(s["E"]):
        share = torch.where(s["ids_TK"] == e, s["scores_TK"].double(), 0.0).sum(1)
        hit = (s["ids_TK"] == e).any(1).nonzero()[:, 0]
        if not len(hit):
            continue
        h = x[hit] @ s["w13"][e].double().t()
        gate, up = h[:, :s["F"]], h[:, s["F"]:]
        if s["clamped"]:
            gate, up = torch.minimum(gate, torch.full_like(gate, LIMIT)), up.clamp(-LIMIT, LIMIT) + 1.0
            h = gate * torch.sigmoid(ALPHA * gate) * up
        else:
            h = gate * torch.sigmoid(gate) * up
        out[hit] += share[hit, None] * (h @ s["w2"][e].double().t())
    return out


_EXACT = {"norm": _exact_norm, "select": _exact_select, "few": _exact_few}
