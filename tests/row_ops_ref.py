"""Plain 64-bit forms of the language-model row operators, for the tests."""
import torch


def rms_norm(x, weight, eps, residual=None):
    s = x.double() + (0 if residual is None else residual.double())
    w = 1.0 if weight is None else weight.double()
    return s / torch.sqrt(s.square().mean(-1, keepdim=True) + eps) * w, s


def scales(y, group):
    cols = y.shape[-1]
    group = group or cols
    parts = -(-cols // group)
    wide = torch.zeros(*y.shape[:-1], parts * group, dtype=y.dtype, device=y.device)
    wide[..., :cols] = y.abs()
    return wide.view(*y.shape[:-1], parts, group).amax(-1).clamp(min=2.0 ** -100) / 448


def rms_norm_grads(dy, s, weight, eps, dsum=None):
    """(ds, dweight) and the sizes of what is added up in them."""
    s, g = s.double(), dy.double()
    w = torch.ones(s.shape[-1], dtype=s.dtype, device=s.device) if weight is None else weight.double()
    r = 1.0 / torch.sqrt(s.square().mean(-1, keepdim=True) + eps)
    ds = r * g * w - s * r ** 3 * (g * w * s).mean(-1, keepdim=True)
    size = (r * g * w).abs() + s.abs() * r ** 3 * (g * w * s).abs().mean(-1, keepdim=True)
    if dsum is not None:
        ds, size = ds + dsum.double(), size + dsum.double().abs()
    dw = (g * s * r).reshape(-1, s.shape[-1])
    return ds, dw.sum(0), size, dw.abs().sum(0)


def route(logits, k, score="softmax", bias=None, groups=1, groups_kept=1, group_top=2, renormalize=True, scale=1.0):
    l = logits.double()
    l = torch.where(l.isnan(), float("-inf"), l)
    n, e = l.shape
    if score == "sigmoid":
        s = torch.sigmoid(l)
        logs = torch.nn.functional.logsigmoid(l)
    else:
        m = l.amax(1, keepdim=True)
        d = torch.where(l == m, 0.0, l - m)
        logs = d - torch.exp(d).sum(1, keepdim=True).log()
        s = logs.exp()
    b = torch.zeros(e, dtype=l.dtype, device=l.device) if bias is None else bias.double()
    usable = (l > float("-inf")) & (b > float("-inf")).unsqueeze(0)
    c = torch.where(usable, s + torch.where(b > float("-inf"), b, 0.0), float("-inf"))
    by = torch.where(usable, l, float("-inf")) if bias is None else c
    if groups > 1:
        parts = c.view(n, groups, -1).sort(dim=2, descending=True).values
        best = parts[:, :, 0].clone()
        if group_top == 2 and parts.shape[2] > 1:
            best += torch.where(parts[:, :, 1] > float("-inf"), parts[:, :, 1], 0.0)
        kept = best.sort(dim=1, descending=True, stable=True).indices[:, :groups_kept]
        keep = torch.zeros(n, groups, dtype=torch.bool, device=l.device).scatter(1, kept, True)
        by = torch.where(keep.repeat_interleave(e // groups, dim=1), by, float("-inf"))
    value, pick = by.sort(dim=1, descending=True, stable=True)
    value, pick = value[:, :k], pick[:, :k]
    chosen = value > float("-inf")
    w = torch.where(chosen, logs.gather(1, pick), float("-inf"))
    if renormalize:
        top = w.amax(1, keepdim=True)
        w = torch.exp(w - torch.where(top > float("-inf"), top, 0.0))
        total = w.sum(1, keepdim=True)
        w = w / torch.where(total > 0, total, 1.0)
    else:
        w = w.exp()
    return scale * w, torch.where(chosen, pick, -1).int()


def route_weights(logits, picks, score, renormalize, scale):
    """The weights of given picks, differentiable by the logits (64 bits)."""
    ok = (picks >= 0) & (picks < logits.shape[1])
    logs = torch.nn.functional.logsigmoid(logits) if score == "sigmoid" else logits - logits.logsumexp(1, keepdim=True)
    a = torch.where(ok, logs.gather(1, picks.long().clamp(0, logits.shape[1] - 1)), float("-inf"))
    if renormalize:
        total = a.logsumexp(1, keepdim=True)
        a = a - torch.where(total > float("-inf"), total, 0.0)
    return scale * torch.where(ok, a.exp(), 0.0)


def order(experts, num):
    flat = experts.reshape(-1).cpu().tolist()
    lists = [[i for i, e in enumerate(flat) if e == x] for x in range(num)]
    offsets = [0]
    for one in lists:
        offsets.append(offsets[-1] + len(one))
    out = [i for one in lists for i in one]
    slot = [-1] * len(flat)
    for at, i in enumerate(out):
        slot[i] = at
    out += [-1] * (len(flat) - len(out))
    return torch.tensor(offsets), torch.tensor(out, dtype=torch.long), torch.tensor(slot).view(experts.shape)


def sample(logits, uniform, temperature, top_k, top_p, min_p):
    """Row by row on the host: (tokens, probs)."""
    tokens, probs = [], []
    n = logits.shape[0]

    def at(v, i):
        return float(v[i]) if torch.is_tensor(v) else float(v)

    for i in range(n):
        l = logits[i].double().cpu()
        l = torch.where(l.isnan(), float("-inf"), l)
        top = l.max()
        if top == float("-inf"):
            tokens.append(-1)
            probs.append(0.0)
            continue
        t, k, p, least = (at(v, i) for v in (temperature, top_k, top_p, min_p))
        if not t > 0:
            t, k = 1.0, 1
        w = torch.where(l == top, 1.0, torch.exp((l - top) / t))
        index = torch.sort(l, descending=True, stable=True).indices
        if k > 0:
            index = index[: int(k)]
        kept = w[index]
        before = torch.cumsum(kept, 0) - kept
        stay = torch.ones_like(kept, dtype=torch.bool)
        if p < 1:
            stay &= before < p * kept.sum()
        if least > 0:
            stay &= kept >= min(least, 1.0)
        stay[0] = True
        w = torch.zeros_like(w).index_copy(0, index[stay], kept[stay])
        run = torch.cumsum(w, 0)
        u = float(uniform[i])
        u = min(max(u, 0.0), 1.0) if u == u else 0.0
        past = (run > u * run[-1]).nonzero()
        token = int(past[0]) if len(past) else int((w > 0).nonzero()[-1])
        tokens.append(token)
        probs.append(float(w[token] / run[-1]))
    return torch.tensor(tokens), torch.tensor(probs, dtype=torch.float64)
