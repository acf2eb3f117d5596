"""The row operators of a mixture-of-experts language model's step, as measured work.

Four operators over the rows of a matrix: the root-mean-square norm (with the residual's addition,
with 8-bit output, and its gradient), the routing of tokens to experts (and its gradient), the order
of routed tokens by expert, and the sampling of tokens from logits.  ``run`` computes them from
elementary torch operations, or, with ``own`` set, through ``hephaestus_b200.torch_ops``.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_FP8_MAX = 448.0          # largest finite e4m3 value
_FP8_FLOOR = 2.0 ** -100  # smallest row maximum that a scale is made for
_EPS = 1e-6


def listed():
    return [
        # One decoding step of a small batch: residual added, row scales for an 8-bit product.
        dict(name="norm_decode", op="norm", rows=8, cols=4096, dtype="bf16", residual=True, out="fp8", group=0),
        # A prompt batch entering an 8-bit product with a scale for each 128 columns.
        dict(name="norm_prompt_fp8", op="norm", rows=16384, cols=4096, dtype="bf16", residual=True, out="fp8",
             group=128),
        # An odd width in half precision, no residual (rows start off every vector boundary).
        dict(name="norm_odd", op="norm", rows=5003, cols=2049, dtype="f16", residual=False, out="same", group=0),
        # The norm's backward pass of a training step, the residual stream's gradient joining in.
        dict(name="norm_grad", op="norm_grad", rows=8192, cols=4096, dtype="bf16", residual=True),
        # A decoding step's routing: sigmoid scores, balance bias, the best 4 of 8 groups, 8 of 256 experts.
        dict(name="route_decode", op="route", rows=64, experts=256, k=8, dtype="f32", score="sigmoid", bias=True,
             groups=8, kept=4, renorm=True),
        # A training batch's routing with the same rule.
        dict(name="route_train", op="route", rows=32768, experts=256, k=8, dtype="f32", score="sigmoid", bias=True,
             groups=8, kept=4, renorm=True),
        # Gradient of a plain softmax router, weights not renormalised (every logit gets a gradient).
        dict(name="route_grad", op="route_grad", rows=32768, experts=100, k=6, dtype="bf16", score="softmax",
             bias=False, groups=1, kept=1, renorm=False),
        # Expert order of a decoding step, a tenth of its rows being padding.
        dict(name="order_decode", op="order", rows=64, k=8, experts=256, padded=0.1),
        # Expert order of a training batch.
        dict(name="order_train", op="order", rows=32768, k=8, experts=256, padded=0.0),
        # Latency of one sequence: the usual top-k and top-p.
        dict(name="sample_one", op="sample", rows=1, vocab=131072, dtype="bf16", top_k=50, top_p=0.95, min_p=0.0,
             temperature=0.8, per_row=False),
        # A serving batch, each request with settings of its own.
        dict(name="sample_mixed", op="sample", rows=256, vocab=131072, dtype="f32", top_k=0, top_p=1.0, min_p=0.0,
             temperature=1.0, per_row=True),
        # Rollouts at temperature 1 from the whole distribution, an odd vocabulary.
        dict(name="sample_plain", op="sample", rows=128, vocab=50257, dtype="bf16", top_k=0, top_p=1.0, min_p=0.0,
             temperature=1.0, per_row=False),
    ]


def draw(rng):
    def spread(low, high):
        return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))

    op = rng.choice(["norm", "norm", "norm_grad", "route", "route_grad", "order", "sample", "sample"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op in ("norm", "norm_grad"):
        cols = spread(200, 12000)
        if rng.random() < 0.5:
            cols = (cols + 63) // 64 * 64
        rows = spread(1, max(1, min(16384, (1 << 25) // cols)))
        case = dict(op=op, rows=rows, cols=cols, dtype=dtype, residual=rng.random() < 0.5)
        if op == "norm":
            case["out"] = rng.choice(["same", "fp8"])
            case["group"] = rng.choice([0, 64, 128]) if case["out"] == "fp8" else 0
        return case
    if op in ("route", "route_grad"):
        groups = rng.choice([1, 1, 4, 8])
        experts = groups * spread(max(2, 8 // groups), 512 // groups)
        kept = rng.randint(max(1, groups // 2), groups)
        k = rng.randint(1, min(16, kept * (experts // groups)))
        return dict(op=op, rows=spread(1, 32768), experts=experts, k=k, dtype=dtype,
                    score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, groups=groups, kept=kept,
                    renorm=rng.random() < 0.7)
    if op == "order":
        return dict(op=op, rows=spread(1, 32768), k=rng.randint(1, 8), experts=spread(4, 512),
                    padded=rng.choice([0.0, 0.1, 0.5]))
    vocab = spread(1000, 131072)
    return dict(op=op, rows=spread(1, 192), vocab=vocab, dtype=dtype,
                top_k=rng.choice([0, spread(1, 1000)]), top_p=rng.choice([1.0, round(rng.uniform(0.5, 0.99), 3)]),
                min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.2), 3)]),
                temperature=round(rng.uniform(0.5, 1.5), 3), per_row=rng.random() < 0.3)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    d = "cuda"

    def normal(*shape):
        return torch.randn(*shape, device=d, generator=g)

    def uniform(*shape):
        return torch.rand(*shape, device=d, generator=g)

    s = dict(case)
    op = case["op"]
    if op in ("norm", "norm_grad"):
        n, c, t = case["rows"], case["cols"], _DTYPES[case["dtype"]]
        # Hidden states: columns of unequal size, a few of them far larger, as a trained model's are.
        column = torch.exp(0.5 * normal(c))
        column[:: max(1, c // 7)] *= 20.0
        s["weight"] = (1.0 + 0.2 * normal(c)).to(t)
        if op == "norm":
            s["x"] = (normal(n, c) * column).to(t)
            s["residual"] = (normal(n, c) * column).to(t) if case["residual"] else None
        else:
            s["x"] = (normal(n, c) * column).to(t)
            s["dy"] = (normal(n, c) * 0.01).to(t)
            s["dsum"] = (normal(n, c) * 0.01).to(t) if case["residual"] else None
    elif op in ("route", "route_grad"):
        n, e = case["rows"], case["experts"]
        logits = normal(n, e) * 1.5 + 0.7 * normal(e)  # some experts are liked by all tokens
        s["logits"] = logits.to(_DTYPES[case["dtype"]])
        s["bias"] = 0.1 * normal(e) if case["bias"] else None
        if op == "route_grad":
            s["picks"] = uniform(n, e).argsort(dim=1)[:, : case["k"]].to(torch.int32)
            s["dweights"] = 0.01 * normal(n, case["k"])
    elif op == "order":
        n, e, k = case["rows"], case["experts"], case["k"]
        liked = uniform(n, e).pow(1.0 / torch.exp(0.7 * normal(e)))  # uneven loads, no expert twice in a row
        picks = liked.topk(min(k, e), dim=1).indices.to(torch.int32)
        picks[uniform(n) < case["padded"]] = -1
        s["picks"] = picks
    else:
        n, v = case["rows"], case["vocab"]
        logits = 2.0 * normal(n, v) - 2.0
        # A few likely continuations above the bulk, their number differing from row to row.
        likely = torch.exp(normal(n, 1) * 1.0 + 2.5) / v
        logits += torch.where(uniform(n, v) < likely, 8.0 + 2.0 * normal(n, v), 0.0)
        logits[:, v - v // 100:] = float("-inf")  # padding of the vocabulary
        s["logits"] = logits.to(_DTYPES[case["dtype"]])
        s["u"] = uniform(n)
        if case["per_row"]:
            r = uniform(n)
            s["temperature"] = 0.5 + uniform(n)
            s["temperature"][r < 0.1] = 0.0  # greedy requests
            s["top_k"] = torch.where(uniform(n) < 0.5, (1 + 200 * uniform(n)).int(), 0).to(torch.int32)
            s["top_p"] = torch.where(uniform(n) < 0.5, 0.5 + 0.5 * uniform(n), 1.0)
            s["min_p"] = torch.where(uniform(n) < 0.3, 0.2 * uniform(n), 0.0)
    return s


def run(state):
    if own:
        return _own(state)
    return {"norm": _norm, "norm_grad": _norm_grad, "route": _route, "route_grad": _route_grad, "order": _order,
            "sample": _sample}[state["op"]](state)


def _own(s):
    from hephaestus_b200 import torch_ops as ops

    op = s["op"]
    if op == "norm":
        if s["out"] == "fp8":
            return ops.rms_norm_fp8(s["x"], s["weight"], _EPS, residual=s["residual"], group=s["group"] or None)
        return ops.rms_norm(s["x"], s["weight"], _EPS, residual=s["residual"])
    if op == "norm_grad":
        return ops.rms_norm_backward(s["dy"], s["x"], s["weight"], _EPS, dsum=s["dsum"])
    if op == "route":
        return ops.route_experts(s["logits"], s["k"], score=s["score"], bias=s["bias"], groups=s["groups"],
                                 groups_kept=s["kept"], renormalize=s["renorm"], scale=2.5)
    if op == "route_grad":
        return ops.route_experts_backward(s["dweights"], s["logits"], s["picks"], score=s["score"],
                                          renormalize=s["renorm"], scale=2.5)
    if op == "order":
        return ops.expert_order(s["picks"], s["experts"])
    return ops.sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                             min_p=s["min_p"])


# ---------------------------------------------------------------- plain forms


def _norm(s):
    x = s["x"].float()
    if s["residual"] is not None:
        x = x + s["residual"].float()
    y = x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + _EPS) * s["weight"].float()
    dtype = s["x"].dtype
    if s["out"] == "fp8":
        n, c = y.shape
        group = s["group"] or c
        parts = -(-c // group)
        wide = torch.zeros(n, parts * group, device=y.device)
        wide[:, :c] = y
        wide = wide.view(n, parts, group)
        scale = wide.abs().amax(dim=2).clamp(min=_FP8_FLOOR) / _FP8_MAX
        q = (wide / scale.unsqueeze(2)).clamp(-_FP8_MAX, _FP8_MAX).view(n, -1)[:, :c]
        out = [q.to(torch.float8_e4m3fn), scale]
    else:
        out = [y.to(dtype)]
    if s["residual"] is not None:
        out.append(x.to(dtype))
    return tuple(out) if len(out) > 1 else out[0]


def _norm_grad(s):
    x, dy, w = s["x"].float(), s["dy"].float(), s["weight"].float()
    rstd = torch.rsqrt((x * x).mean(dim=1, keepdim=True) + _EPS)
    xhat = x * rstd
    wdy = dy * w
    dx = rstd * (wdy - xhat * (wdy * xhat).mean(dim=1, keepdim=True))
    if s["dsum"] is not None:
        dx = dx + s["dsum"].float()
    return dx.to(s["x"].dtype), (dy * xhat).sum(dim=0).to(s["weight"].dtype)


def _scores(logits, score):
    if score == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-logits))
    e = torch.exp(logits - logits.amax(dim=1, keepdim=True))
    return e / e.sum(dim=1, keepdim=True)


def _route(s):
    logits = s["logits"].double()  # which expert wins may hang on the last bits
    n, e = logits.shape
    score = _scores(logits, s["score"])
    rank_by = logits if s["bias"] is None else score + s["bias"].double()
    if s["groups"] > 1:
        chosen_by = score if s["bias"] is None else rank_by
        best = chosen_by.view(n, s["groups"], -1).sort(dim=2, descending=True).values[:, :, :2].sum(dim=2)
        order = best.sort(dim=1, descending=True, stable=True).indices[:, : s["kept"]]
        kept = torch.zeros(n, s["groups"], dtype=torch.bool, device=logits.device).scatter(1, order, True)
        kept = kept.unsqueeze(2).expand(n, s["groups"], e // s["groups"]).reshape(n, e)
        rank_by = torch.where(kept, rank_by, float("-inf"))
    picks = rank_by.sort(dim=1, descending=True, stable=True).indices[:, : s["k"]]
    w = score.gather(1, picks)
    if s["renorm"]:
        w = w / w.sum(dim=1, keepdim=True)
    return (2.5 * w).float(), picks.to(torch.int32)


def _route_grad(s):
    logits, picks, g = s["logits"].float(), s["picks"].long(), s["dweights"]
    score = _scores(logits, s["score"])
    w = score.gather(1, picks)
    if s["renorm"]:
        total = w.sum(dim=1, keepdim=True)
        dw = 2.5 * (g - (g * w).sum(dim=1, keepdim=True) / total) / total
    else:
        dw = 2.5 * g
    ds = torch.zeros_like(score).scatter(1, picks, dw)
    if s["score"] == "sigmoid":
        dl = ds * score * (1.0 - score)
    else:
        dl = score * (ds - (ds * score).sum(dim=1, keepdim=True))
    return dl.to(s["logits"].dtype)


def _order(s):
    picks, e = s["picks"].reshape(-1).long(), s["experts"]
    m = picks.numel()
    key = torch.where(picks < 0, e, picks)
    counts = torch.zeros(e + 1, dtype=torch.int64, device=picks.device).scatter_add(0, key, torch.ones_like(key))
    offsets = torch.zeros(e + 1, dtype=torch.int64, device=picks.device)
    offsets[1:] = counts[:e].cumsum(0)
    order = key.sort(stable=True).indices
    place = torch.arange(m, device=picks.device)
    slot = torch.empty_like(order)
    slot[order] = place
    total = offsets[e]
    order = torch.where(place < total, order, -1)
    slot = torch.where(picks < 0, -1, slot)
    return offsets.to(torch.int32), order.to(torch.int32), slot.view(s["picks"].shape).to(torch.int32)


def _column(v, like):
    v = v.double() if torch.is_tensor(v) else torch.full((like.shape[0],), float(v), dtype=torch.float64,
                                                         device=like.device)
    return v.unsqueeze(1)


def _sample(s):
    logits = s["logits"].float()
    n, v = logits.shape
    t, k = _column(s["temperature"], logits), _column(s["top_k"], logits)
    p, least = _column(s["top_p"], logits), _column(s["min_p"], logits)
    k = torch.where(t <= 0, 1.0, torch.where(k <= 0, float(v), k))
    t = torch.where(t <= 0, 1.0, t)
    # Sums of many terms next to a border: 64 bits.
    ordered, order = logits.sort(dim=1, descending=True, stable=True)
    w = torch.exp((ordered.double() - ordered[:, :1].double()) / t)
    rank = torch.arange(v, device=logits.device).unsqueeze(0)
    w = torch.where(rank < k, w, 0.0)
    before = w.cumsum(dim=1) - w
    keep = (rank == 0) | ((before < p * w.sum(dim=1, keepdim=True)) & (w >= least))
    kept = torch.zeros_like(w).scatter(1, order, torch.where(keep, w, 0.0))
    mass = kept.cumsum(dim=1)
    target = s["u"].double().unsqueeze(1) * mass[:, -1:]
    token = (mass <= target).sum(dim=1, keepdim=True).clamp(max=v - 1)
    return token.squeeze(1), (kept.gather(1, token) / mass[:, -1:]).squeeze(1).float()


# ------------------------------------------------- definitions in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        h = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
        norm = h.pow(2).sum(1).div(case["cols"]).add(_EPS).sqrt().reciprocal()
        y = torch.einsum("nc,n,c->nc", h, norm, s["weight"].double())
        if case["out"] != "fp8":
            return (y, h) if s["residual"] is not None else y
        q, scales = torch.empty_like(y), []
        step = case["group"] or case["cols"]
        for at in range(0, case["cols"], step):
            part = y[:, at:at + step]
            scales.append(torch.maximum(part.amax(1), -part.amin(1)) / _FP8_MAX)
            q[:, at:at + step] = part / scales[-1].unsqueeze(1)
        scales = torch.stack(scales, dim=1)
        return (q, scales, h) if s["residual"] is not None else (q, scales)
    if op == "norm_grad":
        # The gradient of sum(dy * y) by the quotient rule on y_i = w_i x_i / m, m = sqrt(mean(x^2) + eps).
        x, a = s["x"].double(), s["dy"].double() * s["weight"].double()
        m = torch.linalg.vector_norm(x, dim=1).pow(2).div(case["cols"]).add(_EPS).sqrt().unsqueeze(1)
        dx = a / m - x * torch.einsum("nc,nc->n", a, x).unsqueeze(1) / (case["cols"] * m ** 3)
        if s["dsum"] is not None:
            dx = dx + s["dsum"].double()
        return dx, torch.einsum("nc,nc->c", s["dy"].double() / m, x)
    if op == "route":
        l = s["logits"].double()
        log_score = -torch.logaddexp(torch.zeros_like(l), -l) if case["score"] == "sigmoid" else \
            l - torch.logsumexp(l, dim=1, keepdim=True)
        choice = log_score.exp() + s["bias"].double() if s["bias"] is not None else log_score.exp()
        e = case["experts"]
        if case["groups"] > 1:
            top = choice.view(case["rows"], case["groups"], -1).topk(min(2, e // case["groups"]), dim=2).values.sum(2)
            cut = top.topk(case["kept"], dim=1).values[:, -1:]
            choice = choice.masked_fill((top < cut).repeat_interleave(e // case["groups"], dim=1), float("-inf"))
        picked = log_score.gather(1, choice.topk(case["k"], dim=1).indices)
        if case["renorm"]:
            picked = picked - torch.logsumexp(picked, dim=1, keepdim=True)
        return 2.5 * picked.exp(), None
    if op == "route_grad":
        l = s["logits"].double().requires_grad_()
        with torch.enable_grad():
            log_score = -torch.logaddexp(torch.zeros_like(l), -l) if case["score"] == "sigmoid" else \
                l - torch.logsumexp(l, dim=1, keepdim=True)
            picked = log_score.gather(1, s["picks"].long())
            if case["renorm"]:
                picked = picked - torch.logsumexp(picked, dim=1, keepdim=True)
            (2.5 * picked.exp() * s["dweights"].double()).sum().backward()
        return l.grad
    if op == "order":
        return None  # whole numbers
    l = s["logits"].double()
    n, v = l.shape

    def setting(key):
        return torch.as_tensor(s[key], dtype=torch.float64, device=l.device).expand(n).unsqueeze(1)

    greedy = setting("temperature") <= 0
    l = l / torch.where(greedy, 1.0, setting("temperature"))
    value, place = l.sort(dim=1, descending=True, stable=True)
    rank = torch.arange(v, device=l.device)
    count = torch.where(greedy, 1.0, torch.where(setting("top_k") > 0, setting("top_k"), float(v)))
    value = value.masked_fill(rank >= count, float("-inf"))
    p = torch.softmax(value, dim=1)
    drop = ((p.cumsum(1) - p) >= setting("top_p")) | (p < setting("min_p") * p[:, :1])
    drop[:, 0] = False
    p = torch.softmax(value.masked_fill(drop, float("-inf")), dim=1)
    p = torch.empty_like(p).scatter_(1, place, p)
    past = p.cumsum(1) / p.sum(1, keepdim=True) > s["u"].double().unsqueeze(1)
    return None, p.gather(1, past.int().argmax(dim=1, keepdim=True)).squeeze(1)


def work(case):
    op = case["op"]
    if op in ("norm", "norm_grad"):
        n, c, size = case["rows"], case["cols"], _SIZE[case["dtype"]]
        if op == "norm_grad":
            return {"bytes": n * c * size * (4 if case["residual"] else 3) + 2 * c * size, "flops": 11 * n * c}
        out = 1 if case["out"] == "fp8" else size
        scales = 4 * n * (-(-c // case["group"]) if case["group"] else 1) if case["out"] == "fp8" else 0
        return {"bytes": n * c * (size * (3 if case["residual"] else 1) + out) + c * size + scales,
                "flops": 6 * n * c}
    if op == "route":
        n, e, k = case["rows"], case["experts"], case["k"]
        return {"bytes": n * (e * _SIZE[case["dtype"]] + 8 * k) + 4 * e, "flops": 6 * n * e}
    if op == "route_grad":
        n, e, k, size = case["rows"], case["experts"], case["k"], _SIZE[case["dtype"]]
        # Renormalised or sigmoid weights depend on the picked logits alone.
        read = e if case["score"] == "softmax" and not case["renorm"] else k
        return {"bytes": n * (read * size + 8 * k + e * size), "flops": n * (6 * read + 8 * k)}
    if op == "order":
        return {"bytes": 12 * case["rows"] * case["k"] + 4 * (case["experts"] + 1),
                "flops": 2 * case["rows"] * case["k"]}
    n, v = case["rows"], case["vocab"]
    return {"bytes": n * (v * _SIZE[case["dtype"]] + 16 + (16 if case["per_row"] else 0)), "flops": 6 * n * v}
