"""The language-model row operators at the ends of their ranges: subnormal, tiny and huge numbers,
neighbouring numbers, NaN in biases, workspaces on the least alignment that is asked for.

Against the 64-bit forms, with the tolerances of test_row_ops_gpu.py.
"""
import ctypes

import pytest
import torch

from tests import row_ops_ref as ref
from tests.test_row_ops_gpu import FOLD, T, check_route, check_sample, near, rand  # noqa: F401  (T: the fixture)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------- norm


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cols", [64, 1000, 4096, 40000])
def test_rms_norm_backward_workspace_on_16_bytes(T, dtype, cols):
    """The workspace is asked for on 16 bytes: one that is on no 32 will do."""
    from hephaestus_b200 import _native as N
    code = {torch.float32: N.ROW_F32, torch.bfloat16: N.ROW_BF16, torch.float16: N.ROW_F16}[dtype]
    rows = 40
    dy, s, w = rand(rows, cols, dtype=dtype, seed=1), rand(rows, cols, dtype=dtype, seed=2), rand(cols, dtype=dtype, seed=3)
    dx, dw = torch.empty_like(s), torch.empty_like(w)
    need = ctypes.c_uint64()
    assert N.lib.heph_rms_norm_backward_workspace(0, rows, cols, ctypes.byref(need)) == N.OK
    memory = torch.full((need.value + 96,), 0xa5, dtype=torch.uint8, device="cuda")
    at = 16 + -memory.data_ptr() % 32  # 16 past a multiple of 32
    torch.cuda.synchronize()
    assert N.lib.heph_rms_norm_backward(0, code, dy.data_ptr(), cols, s.data_ptr(), cols, None, 0, w.data_ptr(), code, 1e-6, rows,
                                        cols, dx.data_ptr(), dw.data_ptr(), memory.data_ptr() + at, need.value, None) == N.OK
    torch.cuda.synchronize()
    want, want_w, size, size_w = ref.rms_norm_grads(dy, s, w, 1e-6)
    near(dx, want, size, 2 * FOLD)
    near(dw, want_w, size_w, 2 * FOLD)
    assert bool((memory[:at] == 0xa5).all()) and bool((memory[at + need.value:] == 0xa5).all())


# The kernels of e4m3 output: scales of groups of lanes, of groups past a warp's lanes, of the row, rows
# of one warp, shifted rows (odd widths) with and without groups, long rows with and without.
FP8_FORMS = [(64, None), (256, 16), (4096, None), (4096, 128), (4096, 1024), (2049, None), (2049, 128), (36864, None),
             (36864, 128), (33001, None), (33001, 64)]


def check_fp8(T, x, w, eps, group):
    q, scale = T.rms_norm_fp8(x, w, eps, group=group)
    want, _ = ref.rms_norm(x, w, eps)
    near(scale, ref.scales(want, group))
    cols = x.shape[1]
    g = group if group and group < cols else cols
    ratio = want / scale.double().repeat_interleave(g, dim=1)[:, :cols]
    # Half a step of e4m3 (relative 2^-4, 2^-10 below its normal values), after the 32-bit value.
    off = (q.double() - ratio).abs()
    assert bool((off <= (2.0 ** -4 + 2 * FOLD) * ratio.abs() + 2.0 ** -10).all())
    return q, scale


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cols,group", FP8_FORMS)
def test_rms_norm_fp8_zeros_at_a_small_eps(T, dtype, cols, group):
    """rstd / scale passes the largest number where the values are zeros: they stay zeros."""
    x, w = rand(4, cols, dtype=dtype, seed=1), rand(cols, dtype=dtype, seed=2)
    x[0] = 0
    x[2, : cols // 2] = 0  # groups of zeros, or of zero weights, in rows that are not
    x[3] = 0
    x[3, cols - 1] = torch.finfo(dtype).smallest_normal if dtype == torch.float16 else 1e-7  # and in a row of tiny rms
    w[cols // 4:cols // 2] = 0
    for eps in (1e-12, 1e-30):
        q, scale = check_fp8(T, x, w, eps, group)
        assert bool((q[0].float() == 0).all()) and bool((q.float()[:, cols // 4:cols // 2] == 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols,group", FP8_FORMS)
def test_rms_norm_fp8_below_the_least_scale(T, dtype, cols, group):
    """Values whose scale is the least one come out in its units."""
    x, w = rand(3, cols, seed=3, scale=5e-38).to(dtype), rand(cols, dtype=dtype, seed=4)
    q, scale = check_fp8(T, x, w, 1e-12, group)
    assert bool((scale == scale.min()).all()) and float(q.float().abs().max()) >= 16


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(300, 64), (5, 4096), (9, 257), (3, 16384), (2, 33000)])
def test_rms_norm_backward_of_tiny_and_huge_rows(T, dtype, rows, cols):
    """Rows whose norm is far from 1: rstd cubed is no number of 32 bits, the gradient is."""
    dy, w, d = rand(rows, cols, dtype=dtype, seed=1), rand(cols, dtype=dtype, seed=2), rand(rows, cols, dtype=dtype, seed=3)
    for scale in (1e-17, 1e-13, 1e-12, 1e-6, 1e4, 1e12, 1e13, 1e14, 1e15, 1e16):
        s = rand(rows, cols, seed=4, scale=scale).to(dtype)
        for eps in (0.0, 1e-30, 1e-6):
            for dsum in (None, (d.double() / scale).to(dtype)):
                ds, dw = T.rms_norm_backward(dy, s, w, eps, dsum=dsum)
                want, want_w, size, size_w = ref.rms_norm_grads(dy, s, w, eps, dsum)
                near(ds, want, size, 2 * FOLD)
                near(dw, want_w, size_w, 2 * FOLD)
    s[:] = 0  # rows of zeros: dx = w dy / sqrt(eps)
    ds, dw = T.rms_norm_backward(dy, s, w, 1e-30)
    near(ds, dy.double() * w.double() * 1e15)
    assert bool((dw == 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [(1 << 24), (1 << 24) - 1, (1 << 22) + 8])
def test_rms_norm_of_the_widest_rows(T, dtype, cols):
    """Sums of up to 2^24 terms, equal ones, whose roundings all go one way.

    A thread adds 2^14 terms at most in chains of 128, 128 and 8, and the block in 10 levels: fewer than 288 roundings, or
    3 FOLD, of a sum.  y has half of the sum of squares' (a root); dx three halves of it and one of the other sum."""
    x = torch.full((1, cols), 0.37, device="cuda").to(dtype)
    dy = torch.full((1, cols), 0.11, device="cuda").to(dtype)
    for apart in (False, True):
        if apart:  # rows off every vector boundary of one another
            memory = torch.empty(cols + 8, device="cuda", dtype=dtype)
            memory[1:cols + 1] = x[0]
            x = memory[1:cols + 1].unsqueeze(0)
        want, s = ref.rms_norm(x, None, 1e-6, dy)
        y, total = T.rms_norm(x, None, residual=dy)
        near(y, want, chain=3 * FOLD)
        q, scale = T.rms_norm_fp8(x, None, residual=dy)[:2]
        near(scale, ref.scales(want, None), chain=3 * FOLD)
        assert bool((q.float() == 448).all())  # all equal to the largest
        del q, total, want, s
        dx = T.rms_norm_backward(dy, x, None, 1e-6)[0]
        want, _, size, _ = ref.rms_norm_grads(dy, x, None, 1e-6)
        near(dx, want, size, 8 * FOLD)


@pytest.mark.parametrize("rows,cols", [((1 << 24) + 5, 8), ((1 << 24) + 5, 7), (1 << 21, 128), (1 << 21, 127), (300000, 4096)])
def test_rms_norm_backward_of_many_rows(T, rows, cols):
    """The weight's gradient is a sum over the rows: of like terms, whose roundings all go one way.

    A block has at most 2^24 / 148 rows, added in chains of 256, these in one of 443, and the blocks' shares in chains
    of 19 and a tree: fewer than 800 roundings, beside those of a term: 9 FOLD."""
    x = torch.full((1, cols), 0.37, device="cuda")
    x[:, ::3] = 0.6
    dy, w = torch.full((1, cols), 0.11, device="cuda"), rand(cols, seed=1)
    memory = torch.empty(cols + 8, device="cuda")
    apart = memory[3:cols + 3].copy_(dy[0]).unsqueeze(0)  # off x's vector boundaries
    ds, want_w, size, size_w = ref.rms_norm_grads(dy, x, w, 1e-6)
    for g in (dy, apart):
        got, dw = T.rms_norm_backward(g.expand(rows, cols), x.expand(rows, cols), w, 1e-6)
        near(dw, want_w * rows, size_w * rows, 9 * FOLD)
        for i in (0, rows // 2, rows - 1):
            near(got[i:i + 1], ds, size, 2 * FOLD)
        del got


# ---------------------------------------------------------------- routing


@pytest.mark.parametrize("experts,groups,kept,k", [(32, 4, 2, 4), (64, 8, 3, 4), (256, 8, 4, 8), (512, 16, 3, 6), (1024, 8, 2, 8),
                                                   (60, 5, 2, 4), (300, 4, 2, 8)])
def test_route_nan_bias_with_groups(T, experts, groups, kept, k):
    """An expert of NaN bias is not chosen, nor is it worth anything to its group."""
    logits, bias = rand(150, experts, seed=experts), rand(experts, seed=1, scale=0.2)
    size = experts // groups
    bias[1::5] = float("nan")
    bias[2 * size:3 * size - 1] = float("nan")  # one expert left in this group
    bias[3 * size:4 * size] = float("nan")      # and none in this
    bias[size] = float("-inf")
    for score in ("softmax", "sigmoid"):
        for top in (1, 2):
            _, picks = check_route(T, logits, k, score=score, bias=bias, groups=groups, groups_kept=kept, group_top=top)
            assert not bool(bias[picks[picks >= 0].long()].isnan().any())


@pytest.mark.parametrize("experts,groups", [(64, 8), (128, 4), (256, 8), (512, 8), (1024, 16), (300, 4), (60, 5)])
def test_route_groups_of_neighbouring_large_logits(T, experts, groups):
    """Which group stays hangs on a few units in the last place of logits beside one another."""
    rows, size = 600, experts // groups
    per_lane = max(1, 1 << (experts - 1).bit_length() >> 5)  # experts that are held together
    g = torch.Generator().manual_seed(experts)

    def pick(*high):
        return [int(torch.randint(0, h, (1,), generator=g)) for h in high]

    logits = torch.zeros(rows, experts)
    for row in range(rows):
        base = float(torch.empty(1).uniform_(100, 1000, generator=g))
        ulp = 2.0 ** (torch.tensor(base).log2().floor().item() - 23)
        base = float(torch.tensor(base))
        one, step = pick(groups, groups - 1)
        other = (one + 1 + step) % groups
        at = one * size + pick(size)[0] // per_lane * per_lane
        for j in range(3):  # beside one another in one group
            logits[row, at + pick(per_lane)[0] if at + per_lane <= (one + 1) * size else at] = base + pick(per_lane + 2)[0] * ulp
        for j in range(2):  # and anywhere in the other
            logits[row, other * size + pick(size)[0]] = base + pick(per_lane + 2)[0] * ulp
    logits[0] = 0.0
    logits[0, 0], logits[0, 1], logits[0, size] = 1000.0, 1000.0 + 7 * 2.0 ** -14, 1000.0 + 3 * 2.0 ** -14
    logits = logits.cuda()
    for score in ("softmax", "sigmoid"):
        for top in (1, 2):
            for kept in (1, 2):
                check_route(T, logits, 2, score=score, groups=groups, groups_kept=kept, group_top=top)


# --------------------------------------------------------------- sampling


def subnormals(least, most):
    """f32 numbers of the bits `least` to `most`."""
    return torch.arange(least, most + 1, dtype=torch.int32, device="cuda").view(torch.float32)


def test_sample_threshold_among_subnormals_beside_zeros(T):
    """A range of the search that ends just below the zeros: the key between them and the largest
    negative number is no number's, and none may be counted under it."""
    g = torch.Generator(device="cuda").manual_seed(2)
    rows = []
    for zeros, below in ((5000, 3000), (1100, 1100), (9000, 8000)):
        row = torch.full((20000,), -9.0, device="cuda")
        row[:zeros] = 0.0
        row[:zeros:3] = -0.0
        row[zeros] = subnormals(0x3ff, 0x3ff)
        row[zeros + 1:zeros + 1 + below] = -subnormals(1, 1000).repeat(9)[:below]
        rows.append(row[torch.randperm(20000, device="cuda", generator=g)])
    logits = torch.stack(rows)
    u = torch.tensor([0.1, 0.6, 0.97], device="cuda")
    for k in (1, 2, 1100, 1101, 1102, 1500, 2200, 5001, 5002, 5500, 9001, 9002, 12000):
        check_sample(T, logits, u, top_k=k)
        check_sample(T, logits, u, top_k=k, top_p=0.7)
    # Weights of 1 but for the -9: masses in the same ranges.
    for p in (0.2, 0.5, 0.63, 0.64, 0.9, 0.99):
        check_sample(T, logits, u, top_p=p)


def check_sample_to_units(T, logits, u, temperature, top_k=0, top_p=1.0, min_p=0.0):
    """check_sample for points that a weight below a unit may decide (u = 0 before all).

    Weights are whole numbers of units of 2^-44 of the largest (vocabularies up to 2^17), each rounded by
    half a unit and made to 1e-14 < 2^-46 of it: a running sum of n weights is within n 2^-44 of the 64-bit
    one, as is the whole.  A token whose running sums, before it and with it, hold the point to within
    that is right; where no border is that near there is only one."""
    tokens, probs = T.sample_tokens(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    for row, (token, prob) in enumerate(zip(tokens.tolist(), probs.tolist())):
        l = logits[row].double().cpu()
        w = torch.exp((l - l.max()) / temperature)
        index = torch.sort(l, descending=True, stable=True).indices[: top_k or len(l)]
        before = torch.cumsum(w[index], 0) - w[index]
        stay = (before < top_p * w[index].sum()) & (w[index] >= min_p)
        stay[0] = True
        kept = torch.zeros_like(w).index_copy(0, index[stay], w[index[stay]])
        run, off = torch.cumsum(kept, 0), 2 * len(l) * 2.0 ** -44
        point = float(u[row]) * float(run[-1])
        assert float(run[token] - kept[token]) <= point + off and float(run[token]) > point - off
        assert bool((index[stay] == token).any())
        want = float(kept[token] / run[-1])
        assert abs(prob - want) <= want * (2.0 ** -24 + 2.0 ** -30) + len(l) * 2.0 ** -44


@pytest.mark.parametrize("vocab", [700, 9001])
def test_sample_neighbours_of_the_largest_at_small_temperatures(T, vocab):
    """The number next below the largest logit may be any number of temperatures away: it has no weight
    where that is far."""
    u = torch.tensor([0.0, 0.3, 0.6, 0.999], device="cuda")
    for top in (1.0, 9.0, -3.0, 1e4, 1e10, 1e12, 3e38):
        logits = (rand(4, vocab, seed=1) - 8) * abs(top)
        top = torch.tensor(top, device="cuda")
        logits[:, 5] = torch.nextafter(top, -top.abs() * 2)
        logits[:, 11:600:7] = logits[:, 5:6]
        logits[:, [300, 650]] = top
        step = float(top.double() - logits[0, 5].double())
        for t in (step / 5e5, step / 59600, step / 3000, step / 1000, step / 100, step / 25, step, 20 * step):
            for kw in (dict(), dict(top_k=40), dict(top_p=0.8), dict(min_p=0.01)):
                check_sample_to_units(T, logits, u, t, **kw)


def test_sample_settings_past_their_ends(T):
    """In arrays, as documented: negative, past one, infinite."""
    n, v = 8, 5003
    logits, u = rand(n, v, seed=5, scale=2).round(), torch.rand(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))

    def each(*values):
        return torch.tensor(values, device="cuda", dtype=torch.float32).repeat(n)[:n]
    tokens = check_sample(T, logits, u, top_p=each(-0.5, 0.0, -float("inf")))
    first = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, 0]
    assert torch.equal(tokens, first)
    tokens = check_sample(T, logits, u, min_p=each(1.0, 2.0, float("inf")))
    assert torch.equal(logits.gather(1, tokens.unsqueeze(1))[:, 0], logits.max(1).values)
    check_sample(T, logits, u, top_p=each(1.5, float("inf")), min_p=each(-1.0, -float("inf")))
    hot = each(float("inf"))
    for kw in (dict(), dict(top_k=100), dict(top_p=0.3), dict(top_k=3000, top_p=0.9)):
        check_sample(T, logits, u, temperature=hot, **kw)
