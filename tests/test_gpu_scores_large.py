"""Score operators at their far ends: output rows past 2^31 elements, several chunks of the tile order, long
rows with exact sums, scales far apart, and as many columns as there are ids.

Exact sums: codes are small integers and scales powers of two whose product is 1, 2 or 4, so that every
partial sum of at most 65536 products of at most 4 * 4 is an integer below 2^24 in magnitude, whatever the
order: the product has to equal the one in 64 bits."""
import pytest
import torch

from tests.test_gpu_scores import BF16, F16, F32, FLT_MAX, check_scores, decode, gen, rows8
from tests.test_gpu_scores_state import ix  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype,n,lead", [(BF16, 1000, 5000), (BF16, 1003, 5000), (BF16, 1003, 20_001), (F32, 1003, 5000),
                                          (F16, 1000, 9_999_992)])
def test_query_tiles_past_32_bits(ix, dtype, n, lead):  # noqa: F811
    """More queries than change sides, output rows 60M elements apart: tensor stores, with an odd end, and plain
    ones whose last rows start past 2^31 elements; nothing is written beside them."""
    Q, ld, dim = 40, 60_000_000, 200
    assert (Q - 1) * ld > 2 ** 31
    q, base = rows8(ix, Q, dim, 1, 2), rows8(ix, n, dim, 2, 2)
    whole = torch.zeros(Q, ld, dtype=dtype, device="cuda")
    out = whole[:, lead:lead + n]
    ix.fp8_scores(q, base, dim, 2.0 ** -8, out=out)
    check_scores(out, q, base, dim, 2.0 ** -8, None)
    assert torch.equal(out, ix.fp8_scores(q, base, dim, 2.0 ** -8, dtype=dtype))
    out.zero_()
    assert all(not bool(row.view(torch.int16).any()) for row in whole)


@pytest.mark.parametrize("Q,n,dim,dtype,biased", [
    (130, 100_003, 384, BF16, True),      # two chunks, the second of 50 row tiles; the query tile is kept
    (130, 100_003, 1000, F32, False),     # three chunks, the last of 95
    (300, 60_001, 2100, F16, True),       # three query tiles, two chunks, the last of 87
    (257, 200_000, 200, BF16, False),     # the last chunk of 152 tiles, about as many as CTAs
])
def test_several_chunks(ix, Q, n, dim, dtype, biased):  # noqa: F811
    """Row tiles in more than one chunk, for several query tiles, and a narrower last chunk."""
    pitch, tiles = -(-dim // 16) * 16, -(-n // 256)
    chunk = max(148, (32 << 20) // (256 * pitch))
    assert tiles > chunk and tiles % chunk and Q > 128
    q, base = rows8(ix, Q, dim, 3, 2), rows8(ix, n, dim, 4, 2)
    bias = torch.randn(n, generator=gen(5), device="cuda") if biased else None
    out = ix.fp8_scores(q, base, dim, 2.0 ** -8, bias, dtype)
    for j in range(0, n, 20_000):
        part = tuple(t[j:j + 20_000] for t in base)
        check_scores(out[:, j:j + 20_000], q, part, dim, 2.0 ** -8, None if bias is None else bias[j:j + 20_000])


def exact_rows(rows, dim, exponents, seed):
    """Codes -2 .. 2 and the given exponents, plus 0 or 1 a row and block."""
    g = gen(seed)
    codes = torch.zeros(rows, -(-dim // 16) * 16, device="cuda")
    codes[:, :dim] = torch.randint(-2, 3, (rows, dim), generator=g, device="cuda").float()
    blocks = -(-dim // 128)
    scales = torch.zeros(rows, 4 * -(-dim // 512), dtype=torch.int32, device="cuda")
    scales[:, :blocks] = 127 + exponents + torch.randint(0, 2, (rows, blocks), generator=g, device="cuda")
    assert int(scales.min()) >= 0 and int(scales.max()) < 255
    return codes.to(torch.float8_e4m3fn), scales.to(torch.uint8).view(torch.float8_e8m0fnu)


def exact_scores(q, base, dim, exponents):
    """In 64 bits, with each block's own exponent taken out of both sides (their product has none)."""
    e = torch.exp2(exponents.double())[torch.arange(dim, device="cuda") // 128]
    return (decode(*q, dim) / e) @ (decode(*base, dim) * e).T


EXACT = [(3, 40_000, 5000), (20, 38_000, 5300), (200, 20_000, 5000), (40, 20_000, 8200),     # over all SMs
         (1, 1000, 16384), (128, 512, 65536), (2, 300, 65536), (200, 256, 20000), (130, 513, 4224), (33, 1999, 65533),
         (17, 4096, 4096), (5, 1300, 1), (130, 1300, 97), (300, 700, 1100)]


@pytest.mark.parametrize("Q,n,dim", EXACT)
@pytest.mark.parametrize("spread", [0, 40])
def test_exact_sums(ix, Q, n, dim, spread):  # noqa: F811
    """A lost or misplaced piece of a row shows at any length."""
    exponents = torch.randint(-spread, spread + 1, (-(-dim // 128),), generator=gen(dim), device="cuda")
    q, base = exact_rows(Q, dim, exponents, 6), exact_rows(n, dim, -exponents, 7)
    want = exact_scores(q, base, dim, exponents)
    assert float(want.abs().max()) < 2 ** 24
    out = ix.fp8_scores(q, base, dim)
    assert torch.equal(out.double(), want)


@pytest.mark.parametrize("Q,n,dim", [(2, 300, 65536), (130, 300, 20000), (3, 40_000, 5000), (130, 20_000, 1100)])
def test_every_piece_of_a_long_row(ix, Q, n, dim):  # noqa: F811
    """Base row j holds numbers in its 32-column slice j alone (modulo their count)."""
    none = torch.zeros(-(-dim // 128), dtype=torch.int64, device="cuda")
    q = exact_rows(Q, dim, none, 8)
    codes, scales = exact_rows(n, dim, none, 9)
    slices = -(-dim // 32)
    own = (torch.arange(codes.shape[1], device="cuda") // 32)[None] == (torch.arange(n, device="cuda") * 7 % slices)[:, None]
    base = (torch.where(own, codes.float(), 0.0).to(torch.float8_e4m3fn), scales)
    assert torch.equal(ix.fp8_scores(q, base, dim).double(), exact_scores(q, base, dim, none))


@pytest.mark.parametrize("Q,n", [(3, 300), (20, 40_000), (130, 700)])
@pytest.mark.parametrize("far", [60, 100, 119])
def test_scales_far_apart(ix, Q, n, far):  # noqa: F811
    """Scales near both ends of their range whose products are near one."""
    dim = 640
    for sign in (1, -1):
        exponents = torch.full((5,), sign * far, dtype=torch.int64, device="cuda")
        q, base = exact_rows(Q, dim, exponents, 10), exact_rows(n, dim, -exponents, 11)
        out = ix.fp8_scores(q, base, dim)
        assert torch.equal(out.double(), exact_scores(q, base, dim, exponents))


def test_as_many_columns_as_ids(ix):  # noqa: F811
    """2^31 - 1 rows of one column through all four operators: the first, the last, and some between."""
    n = 2 ** 31 - 1
    at = torch.tensor([0, 1, 255, 256, 2 ** 30 - 1, 2 ** 30, 2 ** 31 - 300, 2 ** 31 - 257, 2 ** 31 - 256, 2 ** 31 - 3, 2 ** 31 - 2],
                      device="cuda")
    val = torch.tensor([3.0, 5.0, 8.0, -2.0, 9.0, 13.0, 4.0, 7.0, 14.0, 6.0, 15.0], device="cuda")
    x = torch.zeros(n, 1, dtype=BF16, device="cuda")
    x[at, 0] = val.to(BF16)
    base = ix.fp8_quantize(x)
    del x
    some = tuple(t[at] for t in base)
    assert torch.equal(decode(*some, 1)[:, 0].float(), val)
    q = ix.fp8_quantize(torch.ones(1, 1, device="cuda"))
    s = ix.fp8_scores(q, base, 1, dtype=BF16)
    del base, some
    assert s.shape == (1, n) and torch.equal(s[0, at].float(), val)
    assert sum(int(torch.count_nonzero(s[0, j:j + 2 ** 28])) for j in range(0, n, 2 ** 28)) == len(at)
    seen = torch.tensor([[2 ** 31 - 2, 0, -1, 2 ** 30, 2 ** 30]], dtype=torch.int32, device="cuda")
    pen = torch.tensor([[1.0, 1.0, 0.5]], device="cuda")
    ids = torch.tensor([[2 ** 31 - 3, -5]], dtype=torch.int32, device="cuda")
    bias = torch.tensor([[10.0, 99.0]], device="cuda")
    ex = torch.zeros(1, -(-n // 32), dtype=torch.int32, device="cuda")
    ex[0, (2 ** 31 - 256) // 32] = 1
    s = ix.adjust_scores(s, seen, pen, ids, bias, ex, out=s)
    want = {0: 1.5, 1: 5.0, 255: 8.0, 256: -2.0, 2 ** 30 - 1: 9.0, 2 ** 30: 10.5, 2 ** 31 - 300: 4.0, 2 ** 31 - 257: 7.0,
            2 ** 31 - 256: -float("inf"), 2 ** 31 - 3: 16.0, 2 ** 31 - 2: 13.5}
    assert s[0, at].tolist() == [want[j] for j in at.tolist()]
    ids, best = ix.topk_scores(s, 9)
    order = sorted((j for j in want if want[j] > 0), key=lambda j: -want[j])
    assert ids[0].tolist() == order and best[0].tolist() == [want[j] for j in order]
    ids, best = ix.topk_scores(s, 1000)      # the rest: zeros, by id
    zeros = [j for j in range(1100) if j not in want][:1000 - len(order)]
    assert ids[0].tolist() == order + zeros
    s[0] = -float("inf")
    s[0, n - 1] = -FLT_MAX / 2
    ids, best = ix.topk_scores(s, 2)
    assert ids[0].tolist() == [n - 1, -1]
