"""The language-model row operators against plain 64-bit forms.

Tolerances: an output of type t is off by at most half a step of t (finfo(t).eps / 2 relative, half
the smallest step near zero) for its one rounding, and by the 32-bit arithmetic before it: a sum of n
terms spread over a block is folded in chains of fewer than 64 additions and a tree of 10 levels, so
FOLD = 96 roundings of 2^-24 cover it with the products, the reciprocal root and the divisions around it.
"""
import ctypes

import pytest
import torch

from tests import row_ops_ref as ref

pytestmark = pytest.mark.gpu

FOLD = 96 * 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def T():
    from hephaestus_b200 import torch_ops
    return torch_ops


def near(got, want, size=None, chain=FOLD):
    """got within one rounding of its type and `chain` of `size` of want."""
    t = torch.finfo(got.dtype)
    size = want.abs() if size is None else size
    tol = t.eps / 2 * want.abs() + t.smallest_normal * t.eps / 2 + chain * size * (1 + t.eps)
    off = (got.double() - want).abs() - tol
    assert bool((off <= 0).all()), f"off by {float((got.double() - want).abs().max())}, {float(off.max())} over the bound"


def rand(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


# ------------------------------------------------------------------- norm

WIDTHS = [1, 2, 7, 8, 31, 64, 127, 128, 256, 1000, 1024, 2049, 4096, 5120, 8192, 8200, 16385, 33000]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", WIDTHS)
def test_rms_norm(T, dtype, cols):
    rows = 1 if cols > 8192 else 11
    x, r = rand(rows, cols, dtype=dtype, seed=1, scale=3), rand(rows, cols, dtype=dtype, seed=2)
    for w in (None, rand(cols, dtype=dtype, seed=3), rand(cols, seed=4)):
        want, _ = ref.rms_norm(x, w, 1e-6)
        near(T.rms_norm(x, w), want)
        y, s = T.rms_norm(x, w, 1e-3, residual=r)
        want, sums = ref.rms_norm(x, w, 1e-3, r)
        near(y, want, want.abs() + (x.abs() + r.abs()).double() * want.abs() / sums.abs().clamp(min=1e-30))
        near(s, sums, (x.abs() + r.abs()).double(), 2.0 ** -24)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols,group", [(1, None), (16, 16), (100, 16), (128, 128), (128, 256), (384, 64), (500, 128),
                                        (1000, 1024), (2048, 32), (2049, 512), (4096, None), (4096, 128), (4100, 2048),
                                        (20001, 128), (36864, 128), (36864, None)])
def test_rms_norm_fp8(T, dtype, cols, group):
    rows = 5 if cols > 8192 else 19
    x, r, w = rand(rows, cols, dtype=dtype, seed=1), rand(rows, cols, dtype=dtype, seed=2), rand(cols, dtype=dtype, seed=3)
    x[1] = 0
    for res in (None, r):
        got = T.rms_norm_fp8(x, w, 1e-6, residual=res, group=group)
        q, scale = got[0], got[1]
        want, s = ref.rms_norm(x, w, 1e-6, res)
        size = want.abs() if res is None else want.abs() + (x.abs() + r.abs()).double() * (want / s).nan_to_num().abs()
        want_scale = ref.scales(want, group)
        near(scale, want_scale, ref.scales(size, group))
        g = group if group and group < cols else cols
        per_col = scale.double().repeat_interleave(g, dim=1)[:, :cols]
        # Half a step of e4m3 (relative 2^-4, 2^-10 below its normal values), after the 32-bit value.
        off = (q.double() - want / per_col).abs()
        assert bool((off <= 2.0 ** -4 * (want / per_col).abs() + 2.0 ** -10 + 2 * FOLD * size / per_col).all())
        # 448 times 1 / (max / 448) may round one step of 32 bits above: saturation keeps it.
        assert float(q.float().abs().max()) <= 448
        if res is not None:
            near(got[2], s, (x.abs() + r.abs()).double(), 2.0 ** -24)


def test_rms_norm_rows_apart_and_shapes(T):
    base = rand(12, 520, dtype=torch.bfloat16, seed=5)
    w = rand(256, dtype=torch.bfloat16, seed=6)
    for x in (base[:, 8:264], base[:, 3:259], base[::3, 8:264], base[2:3].expand(6, 520)[:, :256]):
        near(T.rms_norm(x, w), ref.rms_norm(x, w, 1e-6)[0])
        y, s = T.rms_norm(x.contiguous(), w, residual=x)
        near(y, ref.rms_norm(x, w, 1e-6, x)[0], chain=2 * FOLD)
    x = rand(2, 3, 5, 256, dtype=torch.float16, seed=7)
    w = rand(256, dtype=torch.float16, seed=8)
    y = T.rms_norm(x, w)
    assert y.shape == x.shape
    near(y, ref.rms_norm(x, w, 1e-6)[0])
    q, sc = T.rms_norm_fp8(x, w, group=64)
    assert q.shape == x.shape and sc.shape == (2, 3, 5, 4)
    # Weights and rows off a 16-byte boundary.
    off = rand(257, seed=9)[1:]
    near(T.rms_norm(x, off), ref.rms_norm(x, off, 1e-6)[0])


def test_rms_norm_empty_and_special(T):
    assert T.rms_norm(torch.empty(0, 64, device="cuda")).shape == (0, 64)
    q, s = T.rms_norm_fp8(torch.empty(0, 64, device="cuda"), group=32)
    assert q.shape == (0, 64) and s.shape == (0, 2)
    x = torch.ones(4, 64, device="cuda")
    x[1, 3], x[2, 5] = float("nan"), float("inf")
    y = T.rms_norm(x)
    assert bool(y[1].isnan().all()) and bool(y[2, 5].isnan()) and bool((y[2, :5] == 0).all())
    near(y[::3], ref.rms_norm(x[::3], None, 1e-6)[0])
    q, s = T.rms_norm_fp8(x)
    assert bool(q[1].float().isnan().all()) and bool(s.isfinite().all())
    zero = torch.zeros(3, 128, device="cuda", dtype=torch.bfloat16)
    assert bool((T.rms_norm(zero) == 0).all()) and bool((T.rms_norm_fp8(zero, group=32)[0].float() == 0).all())
    assert bool(T.rms_norm(zero, eps=0.0).isnan().all())  # 0 / 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 64), (1, 4096), (300, 128), (700, 257), (37, 2048),
                                       (64, 5000), (9, 16384), (5, 20001), (3, 33000)])
def test_rms_norm_backward(T, dtype, rows, cols):
    dy, s = rand(rows, cols, dtype=dtype, seed=1), rand(rows, cols, dtype=dtype, seed=2, scale=2)
    d = rand(rows, cols, dtype=dtype, seed=3)
    for w, dsum in ((None, None), (rand(cols, dtype=dtype, seed=4), d), (rand(cols, seed=5), None)):
        ds, dw = T.rms_norm_backward(dy, s, w, 1e-5, dsum=dsum)
        want, want_w, size, size_w = ref.rms_norm_grads(dy, s, w, 1e-5, dsum)
        near(ds, want, size, 2 * FOLD)
        if w is None:
            assert dw is None
        else:
            near(dw, want_w, size_w, 2 * FOLD)


def test_rms_norm_backward_against_differences(T):
    x, w, dy = rand(3, 40, seed=1), rand(40, seed=2), rand(3, 40, seed=3)
    ds, dw = T.rms_norm_backward(dy, x, w, 1e-5)

    def loss(x, w):
        return float((ref.rms_norm(x, w, 1e-5)[0] * dy.double()).sum())

    h = 1e-6  # in 64 bits: differences are good to about h^2 and 1e-16 / h
    for i in range(0, 120, 17):
        step = torch.zeros(120, device="cuda", dtype=torch.float64)
        step[i] = h
        step = step.view(3, 40)
        numeric = (loss(x.double() + step, w) - loss(x.double() - step, w)) / (2 * h)
        assert abs(float(ds.view(-1)[i]) - numeric) < 1e-5
        step = step.view(-1)[:40] if i < 40 else None
        if step is not None:
            numeric = (loss(x, w.double() + step) - loss(x, w.double() - step)) / (2 * h)
            assert abs(float(dw[i]) - numeric) < 1e-5


def test_rms_norm_backward_without_rows(T):
    e = torch.empty(0, 32, device="cuda")
    ds, dw = T.rms_norm_backward(e, e, torch.ones(32, device="cuda"))
    assert ds.shape == (0, 32) and bool((dw == 0).all())


# ---------------------------------------------------------------- routing


def check_route(T, logits, k, **kw):
    w, picks = T.route_experts(logits, k, **kw)
    want, want_picks = ref.route(logits, k, **kw)
    assert torch.equal(picks, want_picks)
    near(w, want)
    return w, picks


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,experts,k", [(1, 1, 1), (2, 2, 1), (5, 8, 2), (33, 31, 31), (7, 32, 32), (65, 60, 4),
                                            (130, 128, 8), (3, 160, 6), (514, 256, 8), (9, 500, 10), (6, 1024, 32)])
def test_route(T, dtype, rows, experts, k):
    logits = rand(rows, experts, dtype=dtype, seed=rows, scale=1.5)
    bias = rand(experts, seed=2, scale=0.2)
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            for b in (None, bias):
                check_route(T, logits, k, score=score, bias=b, renormalize=renormalize, scale=2.5)


@pytest.mark.parametrize("experts,groups,kept,k", [(8, 8, 3, 3), (12, 3, 2, 5), (16, 4, 4, 16), (64, 8, 4, 6),
                                                   (256, 8, 4, 8), (96, 32, 7, 8), (520, 4, 1, 20), (1024, 16, 3, 8),
                                                   (256, 8, 1, 8), (256, 8, 2, 8), (128, 4, 1, 16), (300, 4, 3, 8)])
def test_route_groups(T, experts, groups, kept, k):
    logits = rand(77, experts, seed=experts)
    bias = rand(experts, seed=3, scale=0.3)
    for score in ("softmax", "sigmoid"):
        for b in (None, bias):
            for top in (1, 2):
                check_route(T, logits, k, score=score, bias=b, groups=groups, groups_kept=kept, group_top=top)


def test_route_ties_go_to_the_lowest_index(T):
    logits = torch.zeros(3, 100, device="cuda")
    _, picks = check_route(T, logits, 5)
    assert picks[0].tolist() == [0, 1, 2, 3, 4]
    coarse = (rand(200, 256, seed=1) * 2).round() / 2
    check_route(T, coarse, 8)
    check_route(T, coarse, 8, score="sigmoid", bias=torch.zeros(256, device="cuda"), groups=8, groups_kept=4)
    # Neighbours in 32 bits whose sigmoids are equal there.
    close = torch.full((4, 64), 9.0, device="cuda")
    close[:, 40] = torch.nextafter(torch.tensor(9.0), torch.tensor(10.0))
    _, picks = check_route(T, close, 2, score="sigmoid")
    assert picks[0].tolist() == [40, 0]
    check_route(T, close, 2, score="sigmoid", bias=torch.full((64,), 0.5, device="cuda"))


@pytest.mark.parametrize("experts", [32, 60, 256, 700])
def test_route_near_sums(T, experts):
    """Every score + bias within 1e-7 of the others: what 32 bits cannot tell apart, 64 bits do."""
    logits = rand(1, experts, seed=experts).expand(3, experts)
    for score, s in (("sigmoid", torch.sigmoid(logits[0].double())), ("softmax", torch.softmax(logits[0].double(), 0))):
        bias = (1.0 - s).float()
        for k in (1, 8, 12, 13, 32):
            check_route(T, logits, k, score=score, bias=bias)
        check_route(T, logits, 8, score=score, bias=bias, groups=4, groups_kept=2)
        check_route(T, logits, 3, score=score, bias=bias, groups={32: 8, 60: 15, 256: 32, 700: 20}[experts],
                    groups_kept=3, group_top=1)
    # Logits a unit apart, and equal ones.
    close = torch.full((2, experts), 1.0, device="cuda")
    for at in (3, 17, experts - 1):
        close[:, at] = torch.nextafter(close[0, at], torch.tensor(2.0, device="cuda"))
    for k in (1, 2, 5, 20):
        check_route(T, close, k)
        check_route(T, close, k, score="sigmoid", groups=4, groups_kept=3)


def test_route_infinite_bias(T):
    logits, bias = rand(5, 64, seed=1), torch.zeros(64, device="cuda")
    bias[[4, 9, 33]] = float("inf")
    for k in (1, 2, 3, 6):
        for kw in (dict(), dict(score="sigmoid"), dict(groups=8, groups_kept=2)):
            _, picks = check_route(T, logits, k, bias=bias, **kw)
            if not kw.get("groups"):
                assert picks[0].tolist()[:3] == [4, 9, 33][:k]


def test_route_masked_and_special(T):
    logits = rand(8, 16, seed=1)
    logits[0] = float("-inf")
    logits[1, 2:] = float("-inf")
    logits[2, 5] = float("nan")
    logits[3] = torch.finfo(torch.float32).min
    logits[4, 3] = torch.finfo(torch.float32).min
    logits[5, 7] = 200.0
    logits[6] = -300.0 - torch.arange(16, device="cuda")  # every sigmoid underflows in 32 bits
    logits[7, 1] = float("inf")
    bias = torch.zeros(16, device="cuda")
    bias[9] = float("-inf")
    for kw in (dict(), dict(score="sigmoid"), dict(bias=bias), dict(score="sigmoid", bias=bias),
               dict(groups=4, groups_kept=2), dict(score="sigmoid", groups=4, groups_kept=2, bias=bias)):
        for k in (1, 4):
            w, picks = check_route(T, logits, k, **kw)
            assert bool((picks[0] == -1).all()) and bool((w[0] == 0).all())
    w, picks = T.route_experts(torch.empty(0, 16, device="cuda"), 4)
    assert w.shape == (0, 4) and picks.shape == (0, 4)
    w, picks = T.route_experts(rand(2, 3, 16, seed=2), 4)
    assert w.shape == (2, 3, 4) and picks.dtype == torch.int32


def test_route_rows_apart(T):
    base = rand(40, 300, dtype=torch.bfloat16, seed=4)
    check_route(T, base[::2, 3:103], 6)
    check_route(T, base[5:6].expand(9, 300), 6)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,experts,k", [(1, 1, 1), (3, 5, 2), (66, 64, 6), (40, 100, 6), (130, 256, 8), (5, 1000, 32)])
def test_route_backward(T, dtype, rows, experts, k):
    logits = rand(rows, experts, dtype=dtype, seed=1, scale=1.5)
    g = rand(rows, k, seed=2)
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            w, picks = T.route_experts(logits, k, score=score, renormalize=renormalize, scale=2.5)
            got = T.route_experts_backward(g, logits, picks, score=score, renormalize=renormalize, scale=2.5)
            l = logits.double().requires_grad_()
            (ref.route_weights(l, picks, score, renormalize, 2.5) * g.double()).sum().backward()
            # Differences of g and its weighted mean: the errors are of the larger of these.
            s = torch.softmax(l.detach(), 1) if score == "softmax" else torch.sigmoid(l.detach())
            w64 = ref.route_weights(l.detach(), picks, score, renormalize, 2.5)
            size = torch.zeros_like(l.detach()).scatter_add(1, picks.long(), w64 * (g.double().abs() + (
                (g.double().abs() * w64).sum(1, keepdim=True) / 2.5 if renormalize else 0)))
            if score == "softmax":
                # Renormalised, an expert that is not chosen has a gradient of 0; the 64-bit form gets it as a
                # difference of sums, off by a few 2^-53 of these sums, which 2^-28 of FOLD covers.
                size = size + s * (g.double().abs() * w64).sum(1, keepdim=True) * (2.0 ** -28 if renormalize else 1)
            near(got, l.grad, size)


def test_route_backward_special(T):
    logits = rand(6, 20, seed=1)
    picks = torch.tensor([[0, 1, 2]] * 6, dtype=torch.int32, device="cuda")
    picks[0] = -1
    picks[1, 1:] = -1
    picks[2] = torch.tensor([4, 4, 4])  # one expert named three times
    picks[3, 0] = 20  # past the last
    logits[4, 10:] = float("-inf")
    g = rand(6, 3, seed=2)
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            got = T.route_experts_backward(g, logits, picks, score=score, renormalize=renormalize)
            l = logits.double().requires_grad_()
            want = torch.autograd.grad((ref.route_weights(l, picks, score, renormalize, 1.0) * g.double()).sum(), l)[0]
            want = torch.where(want.isnan(), 0.0, want)
            assert bool(got.isfinite().all())
            near(got, want, torch.full_like(want, float(g.abs().max()) * 4))
    logits[:] = float("-inf")
    assert bool((T.route_experts_backward(g, logits, picks, renormalize=False) == 0).all())
    assert T.route_experts_backward(g[:0], logits[:0], picks[:0]).shape == (0, 20)


def test_route_backward_against_differences(T):
    logits, g = rand(2, 12, seed=1), rand(2, 3, seed=2)
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            _, picks = T.route_experts(logits, 3, score=score, renormalize=renormalize)
            got = T.route_experts_backward(g, logits, picks, score=score, renormalize=renormalize)
            for i in range(12):
                step = torch.zeros_like(logits, dtype=torch.float64)
                step[:, i] = 1e-6
                up, down = (ref.route_weights(logits.double() + d, picks, score, renormalize, 1.0) for d in (step, -step))
                numeric = ((up - down) * g.double()).sum(1) / 2e-6
                assert bool(((got[:, i].double() - numeric).abs() < 1e-5).all())


# ------------------------------------------------------------ expert order


@pytest.mark.parametrize("shape,experts", [((1, 1), 1), ((3, 2), 4), ((64, 8), 256), ((31, 1), 7), ((1000, 3), 1024),
                                           ((4096, 1), 60), ((1025, 4), 33), ((5000, 6), 128), ((40000, 2), 513),
                                           ((65536, 1), 256), ((65537, 1), 1000), ((60000, 5), 31), ((1100000, 2), 64)])
def test_expert_order(T, shape, experts):
    g = torch.Generator(device="cuda").manual_seed(experts)
    picks = torch.randint(-1, experts, shape, device="cuda", dtype=torch.int32, generator=g)
    picks.view(-1)[::97] = experts + 5  # no expert's
    for one in (picks, torch.full_like(picks, experts - 1), torch.full_like(picks, -1)):
        offsets, order, slot = T.expert_order(one, experts)
        key = torch.where((one < 0) | (one >= experts), experts, one).reshape(-1).long()
        counts = torch.bincount(key, minlength=experts + 1)
        want = torch.zeros(experts + 1, dtype=torch.int64, device="cuda")
        want[1:] = counts[:experts].cumsum(0)
        assert torch.equal(offsets.long(), want)
        total = int(want[-1])
        by = key.sort(stable=True).indices
        assert torch.equal(order[:total].long(), by[:total]) and bool((order[total:] == -1).all())
        want_slot = torch.full_like(key, -1)
        want_slot[by[:total]] = torch.arange(total, device="cuda")
        assert torch.equal(slot.reshape(-1).long(), want_slot) and slot.shape == one.shape


def test_expert_order_small_against_lists(T):
    picks = torch.tensor([[2, 0], [2, -1], [1, 2], [9, 0]], dtype=torch.int32, device="cuda")
    for got, want in zip(T.expert_order(picks, 3), ref.order(picks, 3)):
        assert torch.equal(got.cpu().long(), want)
    offsets, order, slot = T.expert_order(picks[:0], 3)
    assert offsets.tolist() == [0, 0, 0, 0] and order.numel() == 0 and slot.shape == (0, 2)


# --------------------------------------------------------------- sampling


def check_sample(T, logits, u, **kw):
    tokens, probs = T.sample_tokens(logits, u, **kw)
    args = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) | kw
    want, want_p = ref.sample(logits, u, **args)
    assert torch.equal(tokens.cpu(), want), (tokens.cpu() != want).nonzero().reshape(-1)[:10]
    near(probs.cpu(), want_p, chain=2.0 ** -40)
    return tokens


SETTINGS = [dict(), dict(temperature=0.7), dict(temperature=0.0), dict(top_k=1), dict(top_k=5), dict(top_k=50, top_p=0.9),
            dict(top_p=0.5), dict(top_p=0.95, temperature=1.4), dict(min_p=0.1), dict(top_k=300, top_p=0.99, min_p=0.02),
            dict(top_p=0.0), dict(min_p=1.0), dict(top_k=10 ** 9), dict(temperature=30.0, top_p=0.7), dict(temperature=1e-4)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 17, 255, 1000, 4099, 32003, 131072])
def test_sample(T, dtype, vocab):
    rows = 3 if vocab > 30000 else 9
    logits = rand(rows, vocab, dtype=dtype, seed=vocab, scale=3)
    g = torch.Generator(device="cuda").manual_seed(vocab)
    for kw in SETTINGS:
        check_sample(T, logits, torch.rand(rows, device="cuda", generator=g), **kw)


@pytest.mark.parametrize("rows", [1, 18, 19, 37, 74, 149, 300])
def test_sample_rows(T, rows):
    """Every number of blocks per row, settings of each row's own."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    logits = rand(rows, 33000, seed=rows, scale=2.5)
    u = torch.rand(rows, device="cuda", generator=g)
    t = torch.rand(rows, device="cuda", generator=g) * 1.5
    t[::5] = 0.0
    k = torch.randint(-2, 400, (rows,), device="cuda", dtype=torch.int32, generator=g)
    p = torch.rand(rows, device="cuda", generator=g) * 1.2
    m = torch.rand(rows, device="cuda", generator=g) * 0.2 - 0.05
    some = slice(0, rows, max(1, rows // 12))
    tokens = T.sample_tokens(logits, u, temperature=t, top_k=k, top_p=p, min_p=m)[0]
    want, _ = ref.sample(logits[some], u[some], t[some], k[some], p[some], m[some])
    assert torch.equal(tokens[some].cpu(), want)


def test_sample_is_the_same_in_any_batch(T):
    logits = rand(200, 50257, dtype=torch.bfloat16, seed=3, scale=2)
    u = torch.rand(200, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    for kw in (dict(), dict(top_p=0.9), dict(top_k=40)):
        whole = T.sample_tokens(logits, u, **kw)
        for n in (1, 20, 70):
            part = T.sample_tokens(logits[:n], u[:n], **kw)
            assert torch.equal(part[0], whole[0][:n]) and torch.equal(part[1], whole[1][:n])


@pytest.mark.parametrize("rows", [296, 297, 320, 511, 512, 513])
def test_sample_rows_in_the_order_of_their_work(T, rows):
    """Batches whose long rows start first: each row's answer is that of a small batch."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    logits = rand(rows, 2500, seed=rows, scale=2.5)
    u = torch.rand(rows, device="cuda", generator=g)
    t = torch.rand(rows, device="cuda", generator=g) * 1.5
    t[torch.rand(rows, device="cuda", generator=g) < 0.3] = 0.0
    k = torch.randint(-60, 60, (rows,), device="cuda", dtype=torch.int32, generator=g)
    p = torch.rand(rows, device="cuda", generator=g) * 1.5
    alike = [torch.full_like(t, 0.0), torch.full_like(t, 0.8)]
    for temperature in (t, *alike):
        for top_k, top_p in ((k, p), (0, p), (k, 1.0), (0, 1.0)):
            got = T.sample_tokens(logits, u, temperature=temperature, top_k=top_k, top_p=top_p)
            for i in range(0, rows, 100):
                part = [v[i:i + 100] if torch.is_tensor(v) else v for v in (temperature, top_k, top_p)]
                want = T.sample_tokens(logits[i:i + 100], u[i:i + 100], temperature=part[0], top_k=part[1], top_p=part[2])
                assert torch.equal(got[0][i:i + 100], want[0]) and torch.equal(got[1][i:i + 100], want[1])


def test_sample_ties_and_masks(T):
    v = 5000
    u = torch.tensor([0.0, 0.2, 0.5, 0.75, 0.999999], device="cuda")
    flat = torch.zeros(5, v, device="cuda")
    tokens = check_sample(T, flat, u, top_k=10)
    assert int(tokens.max()) < 10
    assert check_sample(T, flat, u, temperature=0.0).tolist() == [0] * 5
    check_sample(T, flat, u, top_p=0.5)
    check_sample(T, flat, u, top_k=1000, top_p=0.25)
    coarse = rand(5, v, seed=1, scale=2).round()
    for kw in SETTINGS:
        check_sample(T, coarse, u, **kw)
    low = torch.full((5, v), torch.finfo(torch.float32).min, device="cuda")
    check_sample(T, low, u)  # all equal: all may be drawn
    low[:, 77] = 1.0
    assert check_sample(T, low, u, top_k=20).tolist() == [77] * 5
    masked = torch.full((5, v), float("-inf"), device="cuda")
    masked[1, 4999] = -3.0
    masked[2, 10:20] = 1.0
    masked[3] = float("nan")
    masked[4] = rand(v, seed=2)
    masked[4, ::2] = float("nan")
    for kw in SETTINGS:
        tokens = check_sample(T, masked, u, **kw)
        assert tokens[0] == -1 and tokens[1] == 4999 and tokens[3] == -1
    top = rand(5, v, seed=3)
    top[0, 100], top[1, [5, 4000]] = float("inf"), float("inf")
    for kw in SETTINGS:
        check_sample(T, top, u, **kw)
    signed = torch.zeros(5, v, device="cuda")
    signed[:, ::2] = -0.0
    check_sample(T, signed, u, top_k=7)


def test_sample_scales_of_logits(T):
    """Logits far apart, close together, and around zero: every level of the search."""
    u = torch.rand(6, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9))
    x = rand(6, 20000, seed=4)
    for scale in (1e-30, 1e-6, 1e-2, 50.0, 1e4, 1e30):
        for shift in (0.0, 3.0, -1000.0):
            for kw in (dict(top_k=100), dict(top_k=19999), dict(top_p=0.6), dict(top_p=0.6, temperature=1e3),
                       dict(top_k=3000, top_p=0.3, temperature=scale)):
                check_sample(T, x * scale + shift, u, **kw)


def test_sample_wide_rows(T):
    """Vocabularies past 2^20 (masses in shorter limbs), and the widest."""
    for vocab in (1000000, 1100003, (1 << 22) - (1 << 16)):
        logits = rand(2, vocab, seed=vocab, scale=2)
        u = torch.tensor([0.3, 0.97], device="cuda")
        for kw in (dict(), dict(top_k=700), dict(top_p=0.01), dict(top_p=0.9, temperature=1.3), dict(top_k=5000, top_p=0.5)):
            check_sample(T, logits, u, **kw)
    # All equal: the most that a bin can hold.
    flat = torch.zeros(2, 1100003, device="cuda")
    check_sample(T, flat, u, top_p=0.7)
    check_sample(T, flat, u, top_k=600000, top_p=0.7)


def test_sample_tiny_temperatures(T):
    logits = rand(4, 5000, seed=8)
    logits[:, 100] = logits[:, 4000] = 9.0
    u = torch.tensor([0.1, 0.49, 0.51, 0.9], device="cuda")
    for t in (1e-3, 1e-20, 1e-38, 1e-300):
        for kw in (dict(), dict(top_p=0.4), dict(top_k=3)):
            tokens = check_sample(T, logits, u, temperature=t, **kw)
    assert tokens.tolist() == [100, 100, 4000, 4000]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sample_logits_over_the_whole_range(T, dtype):
    """The largest minus the least passes the largest number of 32 bits."""
    g = torch.Generator(device="cuda").manual_seed(12)
    logits = ((torch.rand(5, 6000, device="cuda", generator=g) * 2 - 1) * 3.38e38).to(dtype)
    logits[0, 7], logits[1, 9] = torch.finfo(dtype).max, torch.finfo(dtype).min
    u = torch.rand(5, device="cuda", generator=g)
    for t in (1.0, 1e36, 1e38, 3e38, 1e300):
        for kw in (dict(), dict(top_p=0.6), dict(top_k=50), dict(top_k=4000, top_p=0.7)):
            check_sample(T, logits, u, temperature=t, **kw)


def test_sample_numbers_outside_the_range(T):
    logits = rand(4, 1000, seed=1)
    u = torch.tensor([-1.0, 1.0, float("nan"), 2.0], device="cuda")
    check_sample(T, logits, u, top_k=20)
    assert T.sample_tokens(logits[:0], u[:0])[0].shape == (0,)
    nan = torch.full((4,), float("nan"), device="cuda")
    check_sample(T, logits, u, temperature=nan)
    a = T.sample_tokens(logits, u, top_p=nan, min_p=nan)[0]
    assert torch.equal(a, T.sample_tokens(logits, u)[0])


def test_sample_rows_apart(T):
    base = rand(9, 9001, dtype=torch.float16, seed=2, scale=2)
    u = torch.rand(9, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    check_sample(T, base[:, 5:8105], u, top_p=0.8)
    check_sample(T, base[::2], u[:5], top_k=30)
    check_sample(T, base[1:2].expand(9, 9001), u)


# ------------------------------------------------- streams, graphs, together


def test_on_another_stream_and_in_a_graph(T):
    x, w = rand(64, 1024, dtype=torch.bfloat16, seed=1), rand(1024, dtype=torch.bfloat16, seed=2)
    gate = rand(1024, 64, dtype=torch.bfloat16, seed=3, scale=0.05)
    head = rand(1024, 5000, dtype=torch.bfloat16, seed=4, scale=0.05)
    u = torch.rand(64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))

    def step(x):
        """A mixture-of-experts layer's bookkeeping and the sampling after it."""
        y, s = T.rms_norm(x, w, residual=x)
        weights, picks = T.route_experts((y @ gate).float(), 4)
        offsets, order, slot = T.expert_order(picks, 64)
        rows = y[order.long() // 4]  # by expert
        back = rows[slot.long()]     # [64, 4, 1024] again
        mixed = (back.float() * weights.unsqueeze(2)).sum(1).to(x.dtype)
        q, scale = T.rms_norm_fp8(mixed, w, group=128)
        tokens, probs = T.sample_tokens((mixed @ head).float(), u, top_k=40, top_p=0.9)
        dl = T.route_experts_backward(weights, (y @ gate).float(), picks)
        ds, dw = T.rms_norm_backward(mixed, s, w, dsum=y)
        return y, s, weights, picks, offsets, order, slot, mixed, q.float(), scale, tokens, probs, dl, ds, dw

    want = step(x)
    y, s, weights, picks, offsets, order, slot, mixed = want[:8]
    # Rows sorted by expert and put back are the rows; renormalised weights sum to 1.
    near(mixed, y.double(), chain=4 * FOLD)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    held = x.clone()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(held)
        graphs.append((graph, out))
    other = rand(64, 1024, dtype=torch.bfloat16, seed=11)
    for value in (other, x):
        want = step(value)
        held.copy_(value)
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)
    # Two replays at once, on streams of their own.
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        for stream, (graph, _out) in zip((a, b), graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _graph, out in graphs:
        for got, one in zip(out, want):
            assert torch.equal(got, one)


def test_trains_through_an_autograd_function(T):
    """The documented way to record gradients: a Function around the two calls."""

    class Norm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, residual, weight):
            y, s = T.rms_norm(x, weight, residual=residual)
            ctx.save_for_backward(s, weight)
            return y, s

        @staticmethod
        def backward(ctx, dy, dsum):
            s, weight = ctx.saved_tensors
            ds, dw = T.rms_norm_backward(dy, s, weight, dsum=dsum)
            return ds, ds, dw

    x, r, w = rand(20, 96, seed=1).requires_grad_(), rand(20, 96, seed=2).requires_grad_(), rand(96, seed=3).requires_grad_()
    a, b = rand(20, 96, seed=4), rand(20, 96, seed=5)
    y, s = Norm.apply(x, r, w)
    (y * a + s * b).sum().backward()
    want, want_w, size, size_w = ref.rms_norm_grads(a, x.detach() + r.detach(), w.detach(), 1e-6, b)
    near(x.grad, want, size, 2 * FOLD)
    assert torch.equal(x.grad, r.grad)
    near(w.grad, want_w, size_w, 2 * FOLD)


def test_calls_of_two_kernels_one_after_the_other(T):
    """The second kernel of a call starts before the first ends: calls that write each other's
    inputs, in a stream and in a graph, between reductions that start early too."""
    picks = torch.randint(0, 60, (80000,), device="cuda", dtype=torch.int32,
                          generator=torch.Generator(device="cuda").manual_seed(1))
    x, w = rand(700, 1000, seed=2), rand(1000, seed=3)

    def chain():
        out, now, grad = [], picks, x
        for _ in range(6):
            offsets, order, slot = T.expert_order(now, 60)
            total = T.sum(offsets)
            now = (order + slot) % 60  # the next call's
            grad, dw = T.rms_norm_backward(grad, x + grad, w)
            out += [offsets, order, slot, total.clone(), grad, dw]
        return out

    want = []
    now, grad = picks, x
    for _ in range(6):
        torch.cuda.synchronize()
        offsets, order, slot = T.expert_order(now, 60)
        torch.cuda.synchronize()
        total = T.sum(offsets)
        torch.cuda.synchronize()
        now = (order + slot) % 60
        torch.cuda.synchronize()
        grad, dw = T.rms_norm_backward(grad, x + grad, w)
        torch.cuda.synchronize()
        want += [offsets, order, slot, total, grad, dw]
    for _ in range(3):
        for a, b in zip(chain(), want):
            assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        offsets, order, slot = T.expert_order(picks, 60)
        again = T.expert_order((order + slot) % 60, 60)
        ds, dw = T.rms_norm_backward(x, x + x, w)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip((offsets, order, slot, *again, ds, dw), (*want[:3], *want[6:9], *want[4:6])):
        assert torch.equal(a, b)


def test_calls_from_several_threads(T):
    """Each thread on a stream of its own, all operators, the answers of one thread alone."""
    import threading
    x, w = rand(500, 1000, dtype=torch.bfloat16, seed=1), rand(1000, seed=2)
    logits = rand(300, 160, seed=3)
    vocab = rand(30, 40000, seed=4, scale=2)
    u = torch.rand(30, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    pairs = torch.randint(0, 160, (100000,), device="cuda", dtype=torch.int32)

    def work():
        ds, dw = T.rms_norm_backward(x, x, w)
        q, scale = T.rms_norm_fp8(x, w, group=64)
        weights, picks = T.route_experts(logits, 6, score="sigmoid", groups=8, groups_kept=4)
        return [T.rms_norm(x, w), ds, dw, q.view(torch.uint8), scale, weights, picks,
                T.route_experts_backward(weights, logits, picks, score="sigmoid"), *T.expert_order(picks, 160),
                *T.expert_order(pairs, 160), *T.sample_tokens(vocab, u, top_k=50, top_p=0.9), *T.sample_tokens(vocab, u)]

    want = work()
    torch.cuda.synchronize()
    wrong = []

    def run():
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got = work()
                    stream.synchronize()
                    wrong.extend(i for i, (a, b) in enumerate(zip(got, want)) if not torch.equal(a, b))
        except Exception as e:  # a thread's own is lost
            wrong.append(repr(e))

    threads = [threading.Thread(target=run) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_rows_more_than_32_bits_apart(T):
    """Inputs and outputs past 2^31 elements: the last rows are the right ones."""
    apart = 2 ** 31 + 64
    base = torch.empty(apart + 9000, device="cuda", dtype=torch.bfloat16)
    near_rows = rand(2, 9000, dtype=torch.bfloat16, seed=1, scale=2)
    x = base.as_strided((2, 9000), (apart, 1))
    x.copy_(near_rows)
    u = torch.tensor([0.2, 0.8], device="cuda")
    for cols in (4096, 4095, 9000):
        a, b = x[:, :cols], near_rows[:, :cols]
        for got, want in zip((T.rms_norm(a), *T.rms_norm_fp8(a, group=128)), (T.rms_norm(b), *T.rms_norm_fp8(b, group=128))):
            assert torch.equal(got.float(), want.float())
        assert torch.equal(T.rms_norm_backward(a, a)[0], T.rms_norm_backward(b, b)[0])
        for kw in (dict(), dict(top_k=9), dict(top_p=0.5)):
            assert torch.equal(T.sample_tokens(a, u, **kw)[0], T.sample_tokens(b, u, **kw)[0])
    a, b = x[:, :200], near_rows[:, :200]
    picked, want = T.route_experts(a, 8), T.route_experts(b, 8)
    assert torch.equal(picked[0], want[0]) and torch.equal(picked[1], want[1])
    assert torch.equal(T.route_experts_backward(want[0], a, want[1]), T.route_experts_backward(want[0], b, want[1]))
    del x, base
    rows = 2 ** 19 + 3  # of 4096: outputs past 2^31 elements
    tall = near_rows[:1, :4096].expand(rows, 4096)
    w = rand(4096, seed=2)
    y = T.rms_norm(tall, w)
    ds, dw = T.rms_norm_backward(tall, tall, w)
    one = T.rms_norm(tall[:1], w), T.rms_norm_backward(tall[:1], tall[:1], w)[0]
    for i in (0, 2 ** 19 - 1, 2 ** 19, rows - 1):
        assert torch.equal(y[i:i + 1], one[0]) and torch.equal(ds[i:i + 1], one[1])


def test_leaves_its_surroundings_alone(T):
    """No byte around the outputs' rows is touched, no current device is changed."""
    from hephaestus_b200 import _native as N
    x = rand(5, 333, dtype=torch.float16, seed=1)
    pad = torch.full((64 + 5 * 333 + 64,), 7.0, dtype=torch.float16, device="cuda")
    out = pad[64:64 + 5 * 333]
    assert N.lib.heph_rms_norm(0, N.ROW_F16, x.data_ptr(), 333, None, 0, None, N.ROW_F16, 1e-6, 5, 333, out.data_ptr(), None,
                               None) == N.OK
    assert bool((pad[:64] == 7).all()) and bool((pad[-64:] == 7).all())
    near(out.view(5, 333), ref.rms_norm(x, None, 1e-6)[0])
    picks = torch.randint(0, 9, (777,), device="cuda", dtype=torch.int32)
    pad = torch.full((3, 1000), 5, dtype=torch.int32, device="cuda")
    assert N.lib.heph_expert_order(0, picks.data_ptr(), 777, 9, pad[0, 10:].data_ptr(), pad[1, 10:].data_ptr(),
                                   pad[2, 10:].data_ptr(), None, 0, None) == N.OK
    assert bool((pad[:, :10] == 5).all()) and bool((pad[0, 20:] == 5).all()) and bool((pad[1:, 787:] == 5).all())
    assert torch.cuda.current_device() == 0


def test_a_device_that_is_not_there(T):
    from hephaestus_b200 import _native as N
    x = rand(2, 8)
    out = torch.empty_like(x)
    assert N.lib.heph_rms_norm(99, N.ROW_F32, x.data_ptr(), 8, None, 0, None, N.ROW_F32, 1e-6, 2, 8, out.data_ptr(), None,
                               None) == N.DEVICE_UNAVAILABLE
    near(T.rms_norm(x), ref.rms_norm(x, None, 1e-6)[0])  # the context is as it was


def test_workspace_too_small_is_refused(T):
    from hephaestus_b200 import _native as N
    x, w = rand(4, 64), rand(64)
    dx, dw, work = torch.empty_like(x), torch.empty_like(w), torch.empty(4 * 64 * 4, dtype=torch.uint8, device="cuda")
    need = ctypes.c_uint64()
    assert N.lib.heph_rms_norm_backward_workspace(0, 4, 64, ctypes.byref(need)) == N.OK and need.value == 4 * 64 * 4
    args = [0, N.ROW_F32, x.data_ptr(), 64, x.data_ptr(), 64, None, 0, w.data_ptr(), N.ROW_F32, 1e-6, 4, 64, dx.data_ptr(),
            dw.data_ptr()]
    assert N.lib.heph_rms_norm_backward(*args, work.data_ptr(), need.value - 1, None) == N.INVALID_CONFIGURATION
    assert "needs a workspace of 1024 bytes" in N.last_error()
    assert N.lib.heph_rms_norm_backward(*args, None, 0, None) == N.INVALID_CONFIGURATION
    assert N.lib.heph_rms_norm_backward(*args, work.data_ptr(), need.value, None) == N.OK
    torch.cuda.synchronize()
