"""Operators on score rows -- fp8_quantize, fp8_scores, adjust_scores, topk_scores -- against plain
implementations in 64 bits.

Tolerances.  Compression and selection are exact.  A product of two e4m3 codes is exact in fp32 and so
is scaling by a power of two, so a score's error is that of summing dim terms and of the epilogue's
one fused multiply-add: at most dim + 2 roundings, each at most 2^-23 (a truncating adder) of the sum
of magnitudes.  A rule row makes at most 5 + n_bias fp32 roundings (2^-24) of intermediate values that
never exceed the sum of magnitudes.  Rounding to the output's type adds finfo.eps / 2 of the value, or,
below the smallest normal number, where the spacing is smallest_normal * eps whatever the value, half
of that spacing (fp16: 2^-14 * 2^-10 / 2 = 2^-25, which scores of 1e-5 do meet)."""
import numpy as np
import pytest
import torch

from coral_b200 import capi

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
FLT_MAX = 3.4028234663852886e38


@pytest.fixture(scope="module")
def ix():
    with capi.Index(1, 4, 32, "ip") as h:
        yield h
        torch.cuda.synchronize()
        h.scores_check()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# --------------------------------------------------------------------------------------- plain forms
def decode(codes, scales, dim):
    w = torch.exp2(scales.view(torch.uint8).double() - 127.0)
    return codes.double()[:, :dim] * w[:, torch.arange(dim, device=codes.device) // 128]


def plain_quantize(x):
    """(codes as values, scale bytes) in 64 bits; what is not finite leaves the maximum and becomes NaN."""
    x = x.double()
    x = torch.where(torch.isfinite(x), x, float("nan"))
    rows, dim = x.shape
    codes = torch.zeros(rows, -(-dim // 16) * 16, dtype=torch.float64, device=x.device)
    scales = torch.zeros(rows, 4 * -(-dim // 512), dtype=torch.uint8, device=x.device)
    for b in range(-(-dim // 128)):
        v = x[:, 128 * b:128 * b + 128]
        top = torch.nan_to_num(v.abs(), nan=0.0).amax(1, keepdim=True)
        e = torch.full_like(top, -127.0)
        for k in range(-126, 128):
            e = torch.where(top > 448.0 * 2.0 ** (k - 1), float(k), e)
        v = (v / torch.exp2(e)).clamp(-448.0, 448.0)
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3.0)
        codes[:, 128 * b:128 * b + v.shape[1]] = torch.round(v / step) * step
        scales[:, b:b + 1] = (e + 127).to(torch.uint8)
    return codes, scales


def same_codes(got, want):
    g = got.double()
    assert torch.equal(torch.isnan(g), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(g), torch.nan_to_num(want))


def check_scores(out, q, base, dim, alpha, bias):
    a, b = decode(*q, dim), decode(*base, dim)
    want = alpha * (a @ b.T)
    mag = abs(alpha) * (a.abs() @ b.abs().T)
    if bias is not None:
        want = want + bias.double()
        mag = mag + bias.double().abs()
    fi = torch.finfo(out.dtype)
    tol = (dim + 2) * 2.0 ** -23 * mag + fi.eps / 2 * (want.abs() * (1 + 2.0 ** -10) + fi.smallest_normal) + 1e-37
    err = (out.double() - want).abs()
    assert bool((err <= tol).all()), f"largest error / tolerance {float((err / tol).max()):.3g}"


def plain_rules(scores, seen, pen, bias_ids, bias, excluded):
    """(values in 64 bits, magnitudes of what was summed)."""
    x = scores.double().cpu().numpy().copy()
    Q, n = x.shape
    mag = np.abs(np.where(np.isfinite(x), x, 0.0))
    for q in range(Q):
        if seen is not None:
            ids, cnt = np.unique(seen[q].cpu().numpy(), return_counts=True)
            rho, phi, pi = (float(v) for v in pen[q].double())
            for j, c in zip(ids, cnt):
                if 0 <= j < n:
                    s = x[q, j]
                    x[q, j] = (s / rho if s > 0 else s * rho) - phi * c - pi
                    mag[q, j] = mag[q, j] * max(rho, 1 / rho) + abs(phi) * c + abs(pi)
        if bias_ids is not None:
            for j, v in zip(bias_ids[q].tolist(), bias[q].double().tolist()):
                if 0 <= j < n:
                    x[q, j] += v
                    mag[q, j] += abs(v)
        if excluded is not None:
            w = excluded[0 if excluded.shape[0] == 1 else q].cpu().numpy().view(np.uint32)
            bits = (w[np.arange(n) // 32] >> (np.arange(n) % 32).astype(np.uint32)) & 1
            x[q, bits != 0] = -np.inf
    return torch.from_numpy(x).to(scores.device), torch.from_numpy(mag).to(scores.device)


def check_rules(ix, scores, seen=None, pen=None, bias_ids=None, bias=None, excluded=None, out=None):
    want, mag = plain_rules(scores, seen, pen, bias_ids, bias, excluded)
    got = ix.adjust_scores(scores, seen, pen, bias_ids, bias, excluded, out=out)
    nb = 0 if bias_ids is None else bias_ids.shape[1]
    fi = torch.finfo(scores.dtype)
    g = got.double()
    assert torch.equal(torch.isnan(g), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(g[inf], want[inf])
    there = torch.isfinite(want)
    tol = (5 + nb) * 2.0 ** -24 * mag + fi.eps / 2 * want.abs() * (1 + 2.0 ** -10) + fi.smallest_normal * fi.eps
    assert bool(((g - want).abs()[there] <= tol[there]).all())
    return got


def plain_topk(scores, k, id_base=0):
    x = scores.float().cpu().numpy()
    Q, n = x.shape
    ids, best = np.full((Q, k), -1, np.int32), np.full((Q, k), -FLT_MAX, np.float32)
    for q in range(Q):
        there = np.nonzero(x[q] > -np.inf)[0]
        top = there[np.argsort(-x[q][there].astype(np.float64), kind="stable")][:k]
        ids[q, :len(top)] = top + id_base
        best[q, :len(top)] = x[q][top]
    return ids, best


def check_topk(ix, scores, k, id_base=0):
    ids, best = ix.topk_scores(scores, k, id_base)
    want_ids, want = plain_topk(scores, k, id_base)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    assert np.array_equal(best.cpu().numpy(), want)      # as numbers: +0 for either zero


# -------------------------------------------------------------------------------------- compression
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim,extra", [(1, 1, 0), (1, 512, 0), (3, 127, 0), (5, 128, 0), (7, 129, 3), (33, 200, 56),
                                            (64, 513, 0), (2, 4096, 8), (1000, 36, 0), (1, 65536, 0)])
def test_quantize(ix, dtype, rows, dim, extra):
    g = gen(rows * 7919 + dim)
    x = torch.randn(rows, dim + extra, generator=g, device="cuda")
    x *= torch.exp2(torch.randint(-12, 5, (rows, 1), generator=g, device="cuda").float())
    x = x.to(dtype)[:, :dim]
    codes, scales = ix.fp8_quantize(x)
    want, want_scales = plain_quantize(x)
    same_codes(codes, want)
    assert torch.equal(scales.view(torch.uint8), want_scales)


def test_quantize_edges(ix):
    inf, nan = float("inf"), float("nan")
    x = torch.zeros(16, 256, device="cuda")
    x[1, 5] = 448.0                      # the largest code, scale 1
    x[2, 5] = 448.0 * (1 + 2.0 ** -23)   # just above it
    x[3] = 2.0 ** -149                   # the smallest subnormal
    x[4, 0] = FLT_MAX
    x[4, 1] = 1.0
    x[5, 7], x[5, 8] = nan, 3.0
    x[6, 9], x[6, 10] = inf, 1.0
    x[7, 9] = -inf
    x[8] = nan
    x[9, 130] = -5.0                     # one block empty, the other not
    x[10, :17] = torch.arange(17, device="cuda") / 16.0 + 1     # ties between codes
    x[10, 20] = 448.0
    x[11, 0] = 2.0 ** -130
    x[12, 0], x[12, 1] = 448.0, 2.0 ** -10      # half the smallest code: ties to zero
    x[12, 2] = 1.5 * 2.0 ** -9
    x[13, 0] = -0.0
    x[14, 0], x[14, 1] = 2.0 ** 127, -(2.0 ** 100)
    codes, scales = ix.fp8_quantize(x)
    want, want_scales = plain_quantize(x)
    same_codes(codes, want)
    assert torch.equal(scales.view(torch.uint8), want_scales)
    assert bool(torch.isnan(codes.float()[6:8, 9]).all()) and codes.float()[6, 10] == 256.0      # 1 = 256 * 2^-8


def test_quantize_writes_its_rows_only(ix):
    x = torch.randn(5, 200, generator=gen(3), device="cuda")
    codes = torch.full((9, 208), 1.0, device="cuda").to(torch.float8_e4m3fn)
    scales = torch.full((9, 4), 7, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    ix.fp8_quantize(x, out=(codes[2:7], scales[2:7]))
    want, want_scales = plain_quantize(x)
    same_codes(codes[2:7], want)
    assert torch.equal(scales.view(torch.uint8)[2:7], want_scales)
    for r in (0, 1, 7, 8):
        assert bool((codes[r].float() == 1.0).all()) and bool((scales.view(torch.uint8)[r] == 7).all())


# ----------------------------------------------------------------------------------------- product
def rows8(ix, rows, dim, seed, spread=6):
    g = gen(seed)
    x = torch.randn(rows, dim, generator=g, device="cuda")
    # a scale of its own for every block, so that a misplaced one shows
    x *= torch.exp2(torch.randint(-spread, spread + 1, (rows, -(-dim // 128)), generator=g, device="cuda").float()
                    ).repeat_interleave(128, 1)[:, :dim]
    return ix.fp8_quantize(x)


@pytest.mark.parametrize("Q,n,dim,dtype,biased", [
    (1, 1, 1, F32, False), (1, 1, 128, F32, True), (1, 256, 128, F32, False), (128, 256, 128, F32, False),
    (128, 256, 512, F32, True), (1, 257, 512, F32, False), (129, 300, 200, F32, True), (3, 100, 17, BF16, False),
    (64, 1000, 640, F16, True), (300, 700, 1100, BF16, True), (128, 512, 65536, F32, False),
    (257, 40000, 64, F32, True), (5, 100_001, 96, BF16, False), (2000, 999, 130, F16, False), (16, 512, 8192, F32, True),
    (1, 1000, 16384, BF16, False), (17, 4096, 4096, F32, True), (200, 256, 20000, F32, False),
])
def test_scores(ix, Q, n, dim, dtype, biased):
    q, base = rows8(ix, Q, dim, 1, 3), rows8(ix, n, dim, 2, 3)
    if dtype == F16:
        alpha = 2.0 ** -8           # inside fp16's range
    else:
        alpha = -1.25
    bias = torch.randn(n, generator=gen(5), device="cuda") if biased else None
    out = ix.fp8_scores(q, base, dim, alpha, bias, dtype)
    assert out.shape == (Q, n) and out.dtype == dtype
    check_scores(out, q, base, dim, alpha, bias)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,lead,ld", [(256, 0, 256), (256, 1, 300), (999, 0, 999), (1000, 3, 1003), (1000, 8, 1008), (64, 0, 4096),
                                       (999, 0, 1000), (1001, 8, 1032), (257, 0, 264), (250, 16, 512), (1, 0, 8), (5, 8, 24),
                                       (767, 0, 768), (770, 0, 776)])
def test_scores_into_slices(ix, dtype, n, lead, ld):
    """Any alignment of the output rows, and nothing outside them is written."""
    Q, dim = 130, 256
    q, base = rows8(ix, Q, dim, 3, 2), rows8(ix, n, dim, 4, 2)
    whole = torch.full((Q + 2, ld), 77.0, dtype=dtype, device="cuda")
    out = whole[1:Q + 1, lead:lead + n]
    assert ix.fp8_scores(q, base, dim, 2.0 ** -6, out=out) is out
    check_scores(out, q, base, dim, 2.0 ** -6, None)
    out.fill_(77.0)
    assert bool((whole == 77.0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Q,n,dim,lead,pad", [(1, 1, 1, 0, 0), (1, 255, 40, 1, 0), (15, 257, 128, 3, 5), (16, 60_001, 200, 0, 7),
                                              (16, 60_000, 70, 8, 8), (17, 60_001, 200, 0, 7), (2, 40_000, 700, 5, 1),
                                              (9, 38_000, 513, 2, 0), (32, 40_003, 200, 1, 0), (31, 39_000, 513, 0, 8),
                                              (24, 300, 16, 3, 2), (33, 40_000, 130, 0, 0), (32, 90_000, 1300, 0, 3)])
def test_scores_of_few_queries(ix, dtype, Q, n, dim, lead, pad):
    """Around the number of queries at which base rows and queries change sides."""
    q, base = rows8(ix, Q, dim, 16, 3), rows8(ix, n, dim, 17, 3)
    bias = torch.randn(n, generator=gen(18), device="cuda")
    whole = torch.full((Q + 2, lead + n + pad), 77.0, dtype=dtype, device="cuda")
    out = whole[1:Q + 1, lead:lead + n]
    ix.fp8_scores(q, base, dim, 2.0 ** -9, bias, out=out)
    check_scores(out, q, base, dim, 2.0 ** -9, bias)
    out.fill_(77.0)
    assert bool((whole == 77.0).all())
    check_scores(ix.fp8_scores(q, base, dim, 0.5 ** 9, dtype=dtype), q, base, dim, 0.5 ** 9, None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Q,n,dim", [(3, 700, 2100), (130, 513, 4096), (40, 257, 1100), (128, 300, 8200), (33, 1999, 3000)])
@pytest.mark.parametrize("lead,pad", [(0, 0), (1, 2), (4, 4)])
def test_scores_of_few_tiles(ix, dtype, Q, n, dim, lead, pad):
    """Few tiles with many k-blocks are shared by clusters: any alignment of the output, nothing outside it."""
    q, base = rows8(ix, Q, dim, 13, 2), rows8(ix, n, dim, 14, 2)
    bias = torch.randn(n, generator=gen(15), device="cuda")
    whole = torch.full((Q + 2, lead + n + pad), 77.0, dtype=dtype, device="cuda")
    out = whole[1:Q + 1, lead:lead + n]
    ix.fp8_scores(q, base, dim, 2.0 ** -9, bias, out=out)
    check_scores(out, q, base, dim, 2.0 ** -9, bias)
    first = out.clone()
    ix.fp8_scores(q, base, dim, 2.0 ** -9, bias, out=out)
    assert torch.equal(first, out)
    out.fill_(77.0)
    assert bool((whole == 77.0).all())


def test_scores_extreme_scales_and_values(ix):
    dim = 512
    q = rows8(ix, 4, dim, 11, 0)
    x = torch.zeros(8, dim, device="cuda")
    x[1] = 1e30
    x[2] = 1e-30
    x[3, 0] = float("nan")
    x[4, 0] = float("inf")
    x[5, 128:256] = -2.0 ** 100
    x[6] = 2.0 ** -140
    base = ix.fp8_quantize(x)
    out = ix.fp8_scores(q, base, dim)
    a, b = decode(*q, dim), decode(*base, dim)
    want = a @ b.T
    ok = [0, 1, 2, 5, 6, 7]
    tol = 514 * 2.0 ** -23 * (a.abs() @ b.abs().T) + 2.0 ** -126
    assert bool(((out.double() - want).abs()[:, ok] <= tol[:, ok]).all())
    assert bool(torch.isnan(out[:, 3]).all())
    assert bool(torch.isnan(out[:, 4]).all())


# ------------------------------------------------------------------------------------------- rules
def words(g, rows, n, share):
    w = torch.zeros(rows, -(-n // 32), dtype=torch.int32, device="cuda")
    for b in range(32):
        w |= (torch.rand(w.shape, generator=g, device="cuda") < share).to(torch.int32) << b
    return w


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Q,n,n_seen,n_bias,share,shared", [
    (1, 1, 1, 1, 0.0, False), (1, 1, 0, 0, 1.0, False), (3, 31, 5, 0, 0.5, False), (2, 33, 0, 4, 0.9, True),
    (4, 8192, 100, 10, 0.3, False), (2, 8193, 300, 1024, 0.0, False), (3, 30000, 5000, 50, 0.95, True),
    (70, 1000, 64, 3, 1.0, False), (1, 100_003, 20_000, 0, 0.02, False), (2, 40_000, 0, 0, 0.5, True),
])
def test_rules(ix, dtype, Q, n, n_seen, n_bias, share, shared):
    g = gen(Q + n + n_seen)
    x = (torch.randn(Q, n, generator=g, device="cuda") * 3).to(dtype)
    seen = pen = bids = bias = ex = None
    if n_seen:
        seen = torch.randint(-2, n + 3, (Q, n_seen), generator=g, device="cuda", dtype=torch.int32)
        seen[:, : n_seen // 3] = seen[:, :1]            # one id many times
        pen = torch.rand(Q, 3, generator=g, device="cuda") + torch.tensor([0.6, -0.3, -0.5], device="cuda")
    if n_bias:
        bids = torch.randint(-2, n + 2, (Q, n_bias), generator=g, device="cuda", dtype=torch.int32)
        bids[:, : n_bias // 2] = bids[:, -1:]
        bias = torch.randn(Q, n_bias, generator=g, device="cuda")
    if share:
        ex = words(g, 1 if shared else Q, n, share)
    got = check_rules(ix, x, seen, pen, bids, bias, ex)
    again = x.clone()
    assert ix.adjust_scores(again, seen, pen, bids, bias, ex, out=again) is again
    assert torch.equal(again.view(torch.int16), got.contiguous().view(torch.int16))     # in place: the same bits


def test_rules_values(ix):
    """Excluded columns may hold anything; what is not excluded keeps infinities and NaN."""
    inf, nan = float("inf"), float("nan")
    for dtype in TYPES:
        low = torch.finfo(dtype).min
        row = torch.tensor([[nan, inf, -inf, low, 0.0, -0.0, 1.0, nan, inf, -inf, low, 5.0]], device="cuda").to(dtype)
        ex = torch.tensor([[0b1100_1000_0111]], dtype=torch.int32, device="cuda")
        seen = torch.tensor([[3, 4, 5, 6, 8, 9, 8, 0, -1, 12, 2 ** 31 - 1, -2 ** 31]], dtype=torch.int32, device="cuda")
        pen = torch.tensor([[2.0, 0.0, 0.0]], device="cuda")
        got = ix.adjust_scores(row, seen, pen, excluded=ex).float()[0].tolist()
        assert got[0] == got[1] == got[2] == got[7] == got[10] == got[11] == -inf
        assert got[3] == -inf and got[4] == 0.0 and got[5] == 0.0 and got[6] == 0.5     # lowest * 2 overflows by the formula
        assert got[8] == inf and got[9] == -inf
        seen.fill_(-1)
        bits = ix.adjust_scores(row, seen, pen)           # nothing applies: the same bits
        assert torch.equal(bits.view(torch.int16), row.view(torch.int16))


@pytest.mark.parametrize("dtype", TYPES)
def test_rules_strided(ix, dtype):
    """Rows apart by an odd number of elements, output rows between the input's."""
    g = gen(9)
    n, Q = 1001, 5
    whole = torch.randn(Q, 2 * n + 1, generator=g, device="cuda").to(dtype)
    keep = whole.clone()
    ex = words(g, Q, n, 0.4)
    check_rules(ix, whole[:, :n], excluded=ex, out=whole[:, n:2 * n])
    assert torch.equal(whole[:, :n], keep[:, :n]) and torch.equal(whole[:, 2 * n], keep[:, 2 * n])


# ------------------------------------------------------------------------------------------ choice
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Q,n,k", [(1, 1, 1), (2, 5, 8), (1, 1000, 10), (3, 8192, 1), (2, 8193, 100), (1, 20000, 1024),
                                   (5, 50_001, 37), (1, 1_000_003, 1000), (300, 700, 64), (2, 300_000, 1)])
def test_topk(ix, dtype, Q, n, k):
    x = torch.randn(Q, n, generator=gen(n + k), device="cuda").to(dtype)
    x[torch.rand(Q, n, generator=gen(n), device="cuda") < 0.3] = -float("inf")
    check_topk(ix, x, k, 5)


@pytest.mark.parametrize("n,k", [(40_000, 100), (200_000, 1024), (9000, 7)])
def test_topk_orders(ix, n, k):
    """Ascending scores beat the threshold at every column; equal ones go by the id."""
    up = torch.arange(n, device="cuda", dtype=F32)[None]
    for x in (up, -up, up * 0, (up % 7) - 3, torch.full((1, n), -float("inf"), device="cuda"),
              torch.full((1, n), -FLT_MAX, device="cuda"), torch.full((1, n), float("nan"), device="cuda"),
              torch.where(up % 2 == 0, 0.0, -0.0)):
        check_topk(ix, x, k)


def test_topk_values(ix):
    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[nan, -inf, inf, -FLT_MAX, 0.0, -0.0, 2.0 ** -149, -2.0 ** -149, FLT_MAX, inf, 1.0, 1.0]], device="cuda")
    ids, best = ix.topk_scores(x, 12)
    assert ids[0].tolist() == [2, 9, 8, 10, 11, 6, 4, 5, 7, 3, -1, -1]
    assert best[0].tolist()[:3] == [inf, inf, FLT_MAX] and best[0].tolist()[-2:] == [-FLT_MAX, -FLT_MAX]
    ids, best = ix.topk_scores(torch.empty(3, 0, device="cuda"), 2)
    assert ids.tolist() == [[-1, -1]] * 3
    ids, best = ix.topk_scores(torch.zeros(2, 9, device="cuda")[:, 2:], 3, id_base=2 ** 31 - 8)
    assert ids.tolist() == [[2 ** 31 - 8, 2 ** 31 - 7, 2 ** 31 - 6]] * 2


# ----------------------------------------------------------------------------- together, and around
def run_all(ix, x, base, dim, bias, seen, pen, ex, k):
    q = ix.fp8_quantize(x)
    s = ix.fp8_scores(q, base, dim, 1.0, bias)
    s = ix.adjust_scores(s, seen, pen, excluded=ex, out=s)
    return ix.topk_scores(s, k)


def chain_inputs(ix, Q, n, dim, seed):
    g = gen(seed)
    x = torch.randn(Q, dim, generator=g, device="cuda")
    rows = torch.randn(n, dim, generator=g, device="cuda")
    base = ix.fp8_quantize(rows)
    bias = -0.5 * rows.square().sum(1)
    seen = torch.randint(-1, n, (Q, 40), generator=g, device="cuda", dtype=torch.int32)
    pen = torch.tensor([[1.3, 0.2, 0.1]], device="cuda").repeat(Q, 1)
    ex = words(g, 1, n, 0.2)
    ex[0, -1] &= 1
    return x, base, bias, seen, pen, ex


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k", [(1500, 1000), (5000, 800), (70_000, 1024), (70_000, 400), (300, 300), (9000, 40)])
def test_topk_crowded_ranges(ix, dtype, n, k):
    """Rows whose best scores crowd parts of their range: all equal, few values, one far away, infinities,
    both signs, exponents apart, the largest and the smallest numbers."""
    g = gen(91)
    fi = torch.finfo(dtype)
    r = torch.randn(n, generator=g, device="cuda").to(dtype)
    far = r.clone()
    far[n // 2] = fi.max
    inf = r.clone()
    inf[::3] = float("inf")
    ends = torch.where(r > 0, torch.full_like(r, fi.max), torch.full_like(r, -fi.max))
    tiny = r * fi.smallest_normal
    spread = torch.exp2(torch.randint(-14, 15, (n,), generator=g, device="cuda").double()).to(dtype) * torch.sign(r)
    few = torch.randint(0, 4, (n,), generator=g, device="cuda").to(dtype)
    one = torch.zeros_like(r)
    one[n - 1] = 1
    check_topk(ix, torch.stack([torch.full_like(r, 2.5), few, far, inf, ends, tiny, spread, one, torch.zeros_like(r)]), k)


def test_the_operators_together(ix):
    """Compressed rows, rules and choice as one search, and the same over two chunks of the base."""
    Q, n, dim, k = 37, 5000, 200, 50
    x, base, bias, seen, pen, ex = chain_inputs(ix, Q, n, dim, 21)
    ids, best = run_all(ix, x, base, dim, bias, seen, pen, ex, k)
    a, b = decode(*ix.fp8_quantize(x), dim), decode(*base, dim)
    want, _ = plain_rules(a @ b.T + bias.double(), seen, pen, None, None, ex)
    got = best.double()
    top = torch.sort(want, dim=1, descending=True).values[:, :k]
    # scores within the product's and the rules' error of the true ones at every rank
    tol = (dim + 9) * 2.0 ** -23 * 1.5 * (a.abs() @ b.abs().T + bias.double().abs()).amax()
    assert bool(((got - top).abs() <= tol).all())
    assert bool(((want.gather(1, ids.long()) - got).abs() <= tol).all())
    # two chunks, each with its own slice of the rules, merged as shards are
    half = 2560
    parts_i, parts_s = [], []
    for lo, hi in ((0, half), (half, n)):
        part = tuple(t[lo:hi] for t in base)
        sl = torch.where((seen >= lo) & (seen < hi), seen - lo, -1)
        i, s = ix.fp8_quantize(x), None
        s = ix.fp8_scores(i, part, dim, 1.0, bias[lo:hi])
        s = ix.adjust_scores(s, sl, pen, excluded=ex[:, lo // 32:(hi + 31) // 32].contiguous())
        i, s = ix.topk_scores(s, k, id_base=lo)
        parts_i.append(i)
        parts_s.append(s)
    mi, ms = ix.merge_shards(torch.stack(parts_i), torch.stack(parts_s), stream=torch.cuda.current_stream().cuda_stream or 1)
    torch.cuda.synchronize()
    assert torch.equal(ms, best) and torch.equal(mi, ids)


def test_results_do_not_depend_on_the_run(ix):
    x, base, bias, seen, pen, ex = chain_inputs(ix, 5, 70_000, 128, 31)
    first = run_all(ix, x, base, 128, bias, seen, pen, ex, 200)
    for _ in range(5):
        again = run_all(ix, x, base, 128, bias, seen, pen, ex, 200)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_captured_and_replayed(ix):
    """Two graphs of the whole chain, replayed on two streams, with inputs changed between replays."""
    dim, k = 256, 20
    sets = [chain_inputs(ix, 6, 30_000, dim, s) for s in (41, 42)]
    want = [run_all(ix, *s[:2], dim, *s[2:], k) for s in sets]
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs, fed = [], [], []
    for s, st in zip(sets, side):
        x = torch.zeros_like(s[0])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(run_all(ix, x, s[1], dim, *s[2:], k))
        graphs.append(g)
        fed.append(x)
    for turn in range(3):
        for i in (0, 1):
            with torch.cuda.stream(side[i]):
                fed[i].copy_(sets[i][0] if turn != 1 else -sets[i][0])
                graphs[i].replay()
        torch.cuda.synchronize()
        if turn != 1:
            for i in (0, 1):
                assert torch.equal(outs[i][0], want[i][0]) and torch.equal(outs[i][1], want[i][1])
    ix.scores_check()
    del graphs


def test_other_streams(ix):
    x, base, bias, seen, pen, ex = chain_inputs(ix, 9, 50_000, 384, 51)
    want = run_all(ix, x, base, 384, bias, seen, pen, ex, 33)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for st in streams:
        with torch.cuda.stream(st):
            got.append(run_all(ix, x, base, 384, bias, seen, pen, ex, 33))
    torch.cuda.synchronize()
    for ids, best in got:
        assert torch.equal(ids, want[0]) and torch.equal(best, want[1])


def test_two_threads_at_once(ix):
    """The chain from two threads, each with its stream and inputs, on one handle."""
    import threading
    sets = [chain_inputs(ix, 6, 30_000 + 1000 * i, 256, 95 + i) for i in range(2)]
    want = [run_all(ix, x, base, 256, bias, seen, pen, ex, 20) for x, base, bias, seen, pen, ex in sets]
    torch.cuda.synchronize()
    got, wrong = [None, None], []

    def work(i):
        x, base, bias, seen, pen, ex = sets[i]
        stream = torch.cuda.Stream()
        try:
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got[i] = run_all(ix, x, base, 256, bias, seen, pen, ex, 20)
                    stream.synchronize()
                    assert torch.equal(got[i][0], want[i][0]) and torch.equal(got[i][1], want[i][1])
        except BaseException as e:
            wrong.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong


def test_launches_are_counted(ix):
    before = ix.launch_count
    run_all(ix, *chain_inputs(ix, 2, 100, 64, 61)[:2], 64, None, None, None, None, 5)
    assert ix.launch_count - before >= 4


# ---------------------------------------------------------------------------------------- refusals
def refused(code, f, *a, **kw):
    with pytest.raises(capi.CoralError) as e:
        f(*a, **kw)
    assert e.value.code == code and len(str(e.value)) > 20


def test_refusals(ix):
    x = torch.randn(4, 64, device="cuda")
    q = ix.fp8_quantize(x)
    s = torch.zeros(4, 100, device="cuda")
    A, L = capi.ERR_ARG, capi.ERR_LIMIT
    refused(A, ix.fp8_quantize, x.double())
    refused(A, ix.fp8_quantize, x.cpu())
    refused(A, ix.fp8_quantize, x.t())
    refused(A, ix.fp8_quantize, x[0])
    refused(A, ix.fp8_quantize, x[:, :0])
    refused(A, ix.fp8_quantize, x, out=(q[0][:3], q[1]))
    refused(A, ix.fp8_quantize, x, out=(q[1], q[0]))
    refused(A, ix.fp8_quantize, x[:1].expand(4, 64))
    refused(A, ix.fp8_scores, q, q, 63 - 20)
    refused(A, ix.fp8_scores, q, q, 0)
    refused(A, ix.fp8_scores, q, (q[0], q[1][:3]), 64)
    refused(A, ix.fp8_scores, q, q, 64, bias=torch.zeros(5, device="cuda"))
    refused(A, ix.fp8_scores, q, q, 64, bias=torch.zeros(4))
    refused(A, ix.fp8_scores, q, q, 64, out=torch.zeros(4, 5, device="cuda"))
    refused(A, ix.fp8_scores, q, q, 64, dtype=torch.bfloat16, out=torch.zeros(4, 4, device="cuda"))
    ids = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    pen = torch.ones(4, 3, device="cuda")
    refused(A, ix.adjust_scores, s, ids)
    refused(A, ix.adjust_scores, s, None, pen)
    refused(A, ix.adjust_scores, s, ids.long(), pen)
    refused(A, ix.adjust_scores, s, ids[:3], pen)
    refused(A, ix.adjust_scores, s, None, None, ids)
    refused(A, ix.adjust_scores, s, None, None, None, pen)
    refused(A, ix.adjust_scores, s, None, None, ids, pen)
    refused(A, ix.adjust_scores, s, excluded=torch.zeros(4, 3, dtype=torch.int32, device="cuda"))
    refused(A, ix.adjust_scores, s, excluded=torch.zeros(2, 4, dtype=torch.int32, device="cuda"))
    refused(A, ix.adjust_scores, s, out=s.half())
    refused(A, ix.adjust_scores, s[:, :50], out=s[:, 20:70])
    refused(A, ix.adjust_scores, s.view(-1)[:200].view(2, 100), out=s.view(-1)[100:300].view(2, 100))
    refused(L, ix.adjust_scores, s, None, None, torch.zeros(4, 1025, dtype=torch.int32, device="cuda"),
            torch.zeros(4, 1025, device="cuda"))
    refused(A, ix.topk_scores, s, 0)
    refused(L, ix.topk_scores, s, 1025)
    refused(A, ix.topk_scores, s, 5, id_base=-1)
    refused(A, ix.topk_scores, s, 5, id_base=2 ** 31 - 100)
    refused(A, ix.topk_scores, s.int(), 5)


def test_c_refusals(ix):
    """What the binding cannot hand over: misaligned and host pointers, short workspaces."""
    lib, h = ix._lib, ix._h
    buf = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    host = torch.zeros(1 << 16, dtype=torch.uint8)
    d, p = buf.data_ptr(), host.data_ptr()
    A, L, OK = capi.ERR_ARG, capi.ERR_LIMIT, capi.OK
    assert lib.coral_fp8_quantize(h, d, 0, 4, 64, 64, d + 4096, d + 65536, 1) == OK
    for args in ((p, 0, 4, 64, 64, d, d), (d, 0, 4, 64, 64, p, d), (d, 0, 4, 64, 64, d, p), (d + 2, 0, 4, 64, 64, d, d),
                 (d, 0, 4, 64, 64, d + 8, d), (d, 0, 4, 64, 64, d, d + 2), (d, 3, 4, 64, 64, d, d), (d, 0, -1, 64, 64, d, d),
                 (d, 0, 4, 64, 63, d, d), (d, 0, 4, 65537, 65537, d, d), (None, 0, 4, 64, 64, d, d)):
        assert lib.coral_fp8_quantize(h, *args, 1) == A
    assert lib.coral_fp8_quantize(h, None, 0, 0, 64, 64, None, None, 1) == OK
    ok = [d, d + 4096, 4, d, d + 4096, 4, 64, 1.0, None, d + 65536, 0, 4]
    assert lib.coral_fp8_scores(h, *ok, 1) == OK
    for i, v in ((0, d + 8), (0, p), (0, None), (1, d + 2), (2, -1), (3, d + 1), (4, d + 1), (5, 1 << 31), (6, 0), (8, p),
                 (8, d + 2), (9, d + 2), (9, p), (10, 7), (11, 3)):
        bad = list(ok)
        bad[i] = v
        assert lib.coral_fp8_scores(h, *bad, 1) == A, i
    for i in (2, 5):
        none = list(ok)
        none[i] = 0
        assert lib.coral_fp8_scores(h, *none, 1) == OK
    ok = [d, 0, 4, 100, 100, None, 0, None, None, None, 0, None, 0, d + 65536, 100]
    assert lib.coral_adjust_scores(h, *ok, 1) == OK
    for i, v in ((0, p), (0, d + 2), (1, 3), (2, -1), (3, -1), (4, 99), (6, 5), (6, -1), (10, 5), (11, p), (13, None), (13, p),
                 (13, d + 400), (14, 99)):
        bad = list(ok)
        bad[i] = v
        assert lib.coral_adjust_scores(h, *bad, 1) == A, i
    assert lib.coral_adjust_scores(h, d, 0, 4, 100, 100, None, 0, None, None, None, 0, d, 3, d, 100, 1) == A
    assert lib.coral_adjust_scores(h, d, 0, 4, 100, 100, None, 0, None, None, None, 0, None, 0, d, 101, 1) == A
    assert lib.coral_adjust_scores(h, d, 0, 2 ** 31 - 1, 2 ** 30, 2 ** 30, None, 0, None, None, None, 0, None, 0, d, 2 ** 30, 1) == L
    need = capi.C.c_int64(0)
    assert lib.coral_topk_workspace(h, 1, 200_000, 10, capi.C.byref(need)) == OK and 0 < need.value < 1 << 16
    ok = [d, 0, 1, 200_000, 200_000, 10, 0, d + 900_000, d + 901_000, d + 910_000, need.value]
    assert lib.coral_topk_scores(h, *ok, 1) == OK
    for i, v, code in ((0, p, A), (0, d + 1, A), (1, 5, A), (4, 1000, A), (5, 0, A), (5, 2000, L), (6, -5, A), (7, p, A), (8, None, A),
                       (9, None, A), (9, d + 4, A), (10, need.value - 1, L)):
        bad = list(ok)
        bad[i] = v
        assert lib.coral_topk_scores(h, *bad, 1) == code, i
    torch.cuda.synchronize()
    assert lib.coral_scores_check(h) == OK


def test_overlaps_are_refused(ix):
    """An output that shares memory with another array of its call, at both ends; side by side is allowed."""
    lib, h = ix._lib, ix._h
    buf = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    d = buf.data_ptr()
    A, L, OK = capi.ERR_ARG, capi.ERR_LIMIT, capi.OK
    x, far = d + 65536, d + 131072

    def quantize(codes, scales):      # 4 rows of 64 floats, 128 apart: bytes [0, 256) of every 512
        return lib.coral_fp8_quantize(h, x, 0, 4, 64, 128, codes, scales, 1)
    assert quantize(far, far + 256) == OK
    assert quantize(x + 3 * 512 + 256, far) == OK and quantize(x - 256, far) == OK
    assert quantize(far, x + 256) == OK      # 16 bytes of scales between two rows
    for codes, scales in ((x, far), (x - 240, far), (x + 3 * 512 + 240, far), (far, x + 252), (far, x + 512 - 12), (far, far + 252), (far, far)):
        assert quantize(codes, scales) == A

    def scores(qc, qs, c, s, bias, out):      # 4 x 8 scores of 64 columns, 16 floats apart: bytes [0, 32) of every 64
        return lib.coral_fp8_scores(h, qc, qs, 4, c, s, 8, 64, 1.0, bias, out, 0, 16, 1)
    ok = [d, d + 256, d + 512, d + 1024, d + 1056]
    assert scores(*ok, x) == OK and scores(*ok[:4], x + 32, x) == OK
    for i, size in enumerate((256, 16, 512, 32, 32)):
        for at in (x, x - size + 16, x + 3 * 64 + 16, x + 64 - size + 16 if size <= 64 else x + 64):
            bad = list(ok)
            bad[i] = at
            assert scores(*bad, x) == A, (i, at - x)

    def adjust(seen, pen, ids, bias, ex):     # 4 x 64 floats, 5 of history, 3 biases
        return lib.coral_adjust_scores(h, x, 0, 4, 64, 64, seen, 5, pen, ids, bias, 3, ex, 2, far, 64, 1)
    ok = [d, d + 256, d + 512, d + 768, d + 1024]
    assert adjust(*ok) == OK
    for i, size in enumerate((80, 48, 48, 48, 32)):
        for at, code in ((far - size, OK), (far - size + 4, A), (far + 1020, A), (far + 1024, OK)):
            bad = list(ok)
            bad[i] = at
            assert adjust(*bad) == code, (i, at - far)
    assert lib.coral_adjust_scores(h, x, 0, 1, 64, 64, d, (1 << 24) + 1, d, None, None, 0, None, 0, far, 64, 1) == L

    need = capi.C.c_int64(0)
    assert lib.coral_topk_workspace(h, 1, 100_000, 10, capi.C.byref(need)) == OK and need.value > 0

    def topk(ids, best, ws):
        return lib.coral_topk_scores(h, d, 0, 1, 100_000, 100_000, 10, 0, ids, best, ws, need.value, 1)
    f = d + 400_000
    assert topk(f, f + 40, f + 80) == OK
    for args in ((f - 4, f + 40, f + 80), (f, f - 4, f + 80), (f, f + 36, f + 80), (f, f + 40, f + 72), (f + 8, f + 48, f - 8),
                 (f + 8, f + 48, f + 16), (d, f, f + 80)):
        assert topk(*args) == A
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------ far and empty
def test_offsets_past_32_bits(ix):
    """Rows 1.2e9 elements apart: the third row starts past 2^31 elements (and 2^32 bytes)."""
    ld, n, dim = 1_200_000_000, 1003, 200
    g = gen(71)
    whole = torch.zeros(3, ld, dtype=BF16, device="cuda")
    x = whole[:, :dim]
    x.copy_(torch.randn(3, dim, generator=g, device="cuda").to(BF16))
    codes, scales = ix.fp8_quantize(x)
    want, want_scales = plain_quantize(x)
    same_codes(codes, want)
    assert torch.equal(scales.view(torch.uint8), want_scales)
    base = rows8(ix, n, dim, 72, 2)
    out = whole[:, 5000:5000 + n]                                     # 16-byte rows: tensor stores
    ix.fp8_scores((codes, scales), base, dim, out=out)
    check_scores(out, (codes, scales), base, dim, 1.0, None)
    odd = whole[:, 20_001:20_001 + n]
    ix.fp8_scores((codes, scales), base, dim, out=odd)
    assert torch.equal(odd, out)
    ex = words(g, 3, n, 0.3)
    seen = torch.randint(0, n, (3, 50), generator=g, device="cuda", dtype=torch.int32)
    pen = torch.tensor([[1.2, 0.1, 0.2]], device="cuda").repeat(3, 1)
    there = whole[:, 30_000:30_000 + n]
    check_rules(ix, out, seen, pen, excluded=ex, out=there)
    check_topk(ix, there, 30)
    del whole
    torch.cuda.empty_cache()


def test_many_rows(ix):
    """More rows than a grid's second dimension has: row offsets and block indexes."""
    x = torch.randn(300_000, 7, generator=gen(73), device="cuda")
    check_topk(ix, x[:70_000], 2)
    ids, best = ix.topk_scores(x, 1)
    assert torch.equal(best[:, 0], x.amax(1)) and torch.equal(ids[:, 0].long(), x.argmax(1))
    ex = torch.zeros(300_000, 1, dtype=torch.int32, device="cuda")
    ex[::2] = 5
    got = ix.adjust_scores(x, excluded=ex)
    want = x.clone()
    want[::2, 0] = want[::2, 2] = -float("inf")
    assert torch.equal(got, want)


def test_empty_sizes(ix):
    for dtype in TYPES:
        codes, scales = ix.fp8_quantize(torch.zeros(0, 200, dtype=dtype, device="cuda"))
        assert codes.shape == (0, 208) and scales.shape == (0, 4)
        some = ix.fp8_quantize(torch.ones(5, 200, dtype=dtype, device="cuda"))
        assert ix.fp8_scores((codes, scales), some, 200, dtype=dtype).shape == (0, 5)
        none = ix.fp8_scores(some, (codes, scales), 200, dtype=dtype)
        assert none.shape == (5, 0)
        assert ix.adjust_scores(none, excluded=torch.zeros(1, 0, dtype=torch.int32, device="cuda")).shape == (5, 0)
        x = torch.randn(4, 9, device="cuda").to(dtype)
        got = ix.adjust_scores(x, torch.zeros(4, 0, dtype=torch.int32, device="cuda"), torch.ones(4, 3, device="cuda"),
                               torch.zeros(4, 0, dtype=torch.int32, device="cuda"), torch.zeros(4, 0, device="cuda"))
        assert torch.equal(got, x)
        ids, best = ix.topk_scores(x[:0], 3)
        assert ids.shape == (0, 3) and best.shape == (0, 3)


@pytest.mark.parametrize("dtype", TYPES)
def test_topk_of_slices(ix, dtype):
    """Rows that start anywhere between two 16-byte boundaries, long and short."""
    for n, k in ((1, 1), (5, 3), (37, 40), (9001, 50), (70_003, 300)):
        whole = torch.randn(5, n + 11, generator=gen(n), device="cuda").to(dtype)
        for lead in (0, 1, 3, 6):
            check_topk(ix, whole[:, lead:lead + n], k)


def test_topk_bounds(ix):
    """Ranges far apart, so that the bound takes its coarser steps, and few scores above the rest."""
    n = 30_000
    j = torch.arange(n, device="cuda", dtype=F32)
    for x in (torch.exp2(j % 250 - 125) * torch.where(j % 2 == 0, 1.0, -1.0), torch.exp2(-(j % 140)), -torch.exp2(j % 120),
              torch.where(j % 3000 == 7, 1e30, j * 1e-6), torch.where(j % 3000 == 7, float("inf"), -j)):
        for k in (1, 20, 300, 1000):
            check_topk(ix, x[None].contiguous(), k)


def test_first_use_inside_a_capture():
    """A process whose very first operator calls are captured (no warm-up that loads the kernels)."""
    import os
    import subprocess
    import sys
    code = """
import torch
from coral_b200 import capi
ix = capi.Index(1, 4, 32, "ip")
x = torch.randn(6, 3000, device="cuda"); rows = torch.randn(700, 3000, device="cuda")
ex = torch.zeros(1, 22, dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    base = ix.fp8_quantize(rows)
    s = ix.fp8_scores(ix.fp8_quantize(x), base, 3000)
    ids, best = ix.topk_scores(ix.adjust_scores(s, excluded=ex), 5)
g.replay(); torch.cuda.synchronize(); ix.scores_check()
want = torch.topk(ix.fp8_scores(ix.fp8_quantize(x), ix.fp8_quantize(rows), 3000), 5)
torch.cuda.synchronize()
assert torch.equal(best, want.values) and torch.equal(ids.long(), want.indices)
print("captured")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]
