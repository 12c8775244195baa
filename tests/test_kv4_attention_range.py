"""Attention over the paged 4-bit cache at the ends of its number ranges, against the formula in 64 bits: caches of one
request, written as codes and parameters, so that every score and value is known."""
import pytest
import torch

pytestmark = pytest.mark.gpu


class Cache:
    """A request's K and V rows: codes [2, length, hd], step and low [2, length], one kv head."""

    def __init__(self, length, hd, page=64):
        self.page, self.hd = page, hd
        self.code = torch.zeros(2, length, hd, dtype=torch.uint8)
        self.step, self.low = torch.zeros(2, 2, length, dtype=torch.float16)

    def values(self):
        k, v = (self.code.double() * self.step.double()[..., None] + self.low.double()[..., None]).cuda()
        return k, v

    def pages(self):
        length, hd, page = self.code.shape[1], self.hd, self.page
        n = -(-length // page)
        par = torch.full((2, n * page, 2), float("nan"), dtype=torch.float16)  # rows past the length: NaN
        par[:, :length, 0], par[:, :length, 1] = self.step, self.low
        codes = torch.zeros(2, n * page, hd // 2, dtype=torch.uint8)
        codes[:, :length] = self.code[..., 0::2] | (self.code[..., 1::2] << 4)
        codes = codes.view(2, n, -1).transpose(0, 1)
        par = par.view(2, n, -1).transpose(0, 1).contiguous().view(torch.uint8)
        return torch.cat([codes.reshape(n, -1), par.reshape(n, -1)], 1).contiguous().cuda()


def _attend(dev, cache, q, scale, workspace=None, copies=1):
    """The rows of `copies` requests that share the cache's pages.  Where there are many, an item's tiles follow each other
    in one run; a lone request is cut into pieces of a few tiles."""
    (length, hd), rows, heads, i32 = cache.code.shape[1:], len(q), q.shape[1], dict(dtype=torch.int32, device="cuda")
    c = dev.KV4Cache(cache.pages(), cache.page, 1, hd)
    table = torch.arange(c.n_pages, **i32).repeat(copies, 1)
    ws = workspace or dev.KV4Workspace(copies, rows * copies, heads, 1, hd)
    q = q.repeat(copies, 1, 1)
    out = c.attention(q, rows * torch.arange(copies + 1, **i32), torch.full((copies,), length, **i32), table, scale, rows, ws,
                      out=torch.full_like(q, 77.0))
    torch.cuda.synchronize()
    assert dev.device_status() == 0
    return out.double().view(copies, rows, heads, hd)


def _exact(cache, q, scale, weight_bits):
    """The result and its bound.  The output's rounding: 2^-11 of it.  The weights': 2^-weight_bits of the sum of the
    products.  32-bit scores (a sum of head_dim terms of magnitude S in all), statistics and sums: 2^-18 (1 + S) of the
    greatest value that the row sees."""
    k, v = cache.values()
    n, length = len(q), len(k)
    seen = torch.arange(length, device="cuda") < (length - n + 1 + torch.arange(n, device="cuda"))[:, None]
    q = q.double()
    z = torch.einsum("thd,jd->htj", q, k) * scale
    p = torch.softmax(z.masked_fill(~seen, float("-inf")), -1)
    size = torch.einsum("thd,jd->htj", q.abs(), k.abs()).mul(abs(scale)).masked_fill(~seen, 0).amax(-1).t()
    most = (v.abs().amax(-1) * seen).amax(-1)
    out = torch.einsum("htj,jd->thd", p, v)
    bound = (2.0 ** -11 * out.abs() + 2.0 ** -weight_bits * torch.einsum("htj,jd->thd", p, v.abs()) +
             (2.0 ** -18 * (1 + size) * most[:, None])[..., None] + 2.0 ** -24)
    return out, bound


def _check(dev, cache, q, scale, weight_bits, copies=1, rows=slice(None)):
    got = _attend(dev, cache, q, scale, copies=copies)
    want, bound = _exact(cache, q, scale, weight_bits)
    assert torch.isfinite(got[:, rows]).all()
    off = ((got - want).abs() / bound)[:, rows]
    assert (off <= 1).all(), float(off.max())


def _bits(rows):
    return 22 if rows <= 16 else 11


def _octaves(cache, z):
    """K rows of one value each, so that a query of ones has the scores z ln 2 (scale ln 2)."""
    cache.step[0], cache.low[0] = 0, (z / cache.hd).half()


LN2 = 0.6931471805599453


@pytest.mark.parametrize("octaves", [9.0, 11.5, 12.9, 13.5, 14.0, 14.5, 14.9, 20.0])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("step", [1.0, 3.75, 7.5, 8.0])
def test_large_steps_under_a_late_maximum(dev, hd, step, octaves):
    """Values whose steps grow to four times the first tile's unit, with one late key far above the scores before it."""
    gen = torch.Generator().manual_seed(5)
    length, n = 400, 40
    c = Cache(length, hd)
    z = torch.zeros(length)
    z[300] = octaves
    _octaves(c, z)
    c.code[1] = torch.randint(0, 16, (length, hd), generator=gen, dtype=torch.uint8)
    c.step[1], c.low[1] = step, -7.5 * step
    c.step[1, :128], c.low[1, :128] = 1.0, -7.5
    _check(dev, c, torch.ones(n, 1, hd, dtype=torch.float16, device="cuda"), LN2, 11,
           copies=300)


@pytest.mark.parametrize("hd", [32, 64])
@pytest.mark.parametrize("rows", [1, 300])
def test_calls_of_every_head_dim_share_a_workspace(dev, hd, rows):
    """What a call of head_dim 128 leaves in the records is no ticket of another head_dim's: items that several warps or
    CTAs share are joined as on a workspace of their own."""
    gen = torch.Generator().manual_seed(8)

    def cache(d, length):
        c = Cache(length, d)
        c.code[:] = torch.randint(0, 16, c.code.shape, generator=gen, dtype=torch.uint8)
        c.step[:], c.low[:] = 0.1, -0.75
        return c

    big, small = cache(128, 3000), cache(hd, 9000)
    qb, qs = (torch.randn(n, 1, d, generator=gen).half().cuda() for n, d in ((1, 128), (rows, hd)))
    ws = dev.KV4Workspace(40, 40 * 300, 1, 1, 128)
    alone = _attend(dev, small, qs, 0.1, copies=40)
    assert not (alone == 77).any()
    for _ in range(2):
        _attend(dev, big, qb, 0.1, ws, copies=40)
        assert torch.equal(_attend(dev, small, qs, 0.1, ws, copies=40), alone)


def _strong_key(dev, hd, rows, drop, copies):
    """60,000 keys `drop` octaves below the first: each weighs little, together they are most of the result, whose first
    value is 0."""
    length = 60000
    c = Cache(length, hd)
    z = torch.full((length,), -drop)
    z[0] = 0
    _octaves(c, z)
    c.code[1], c.step[1], c.low[1] = 15, 0.125, -1.0  # 0.875, in a row that is centred on 0
    c.code[1, 0] = 8  # 0
    _check(dev, c, torch.ones(rows, 1, hd, dtype=torch.float16, device="cuda"), LN2, _bits(rows), copies)


@pytest.mark.parametrize("drop", [12.0, 18.0, 21.0, 23.4, 25.0])
@pytest.mark.parametrize("rows,copies", [(1, 3000), (4, 3000), (7, 1600), (16, 1600)])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_one_strong_key_before_a_long_cache(dev, hd, rows, copies, drop):
    _strong_key(dev, hd, rows, drop, copies)


@pytest.mark.parametrize("rows", [4, 16])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("size", [30.0, 3e3, 6e4])
@pytest.mark.parametrize("part", [0, 1])
def test_a_large_row_moves_none_that_does_not_see_it(dev, hd, rows, size, part):
    _large_row(dev, hd, rows, size, part)


def _large_row(dev, hd, rows, size, part):
    """The last token's K (part 0) or V is far larger than all others: only the last row sees it."""
    gen = torch.Generator().manual_seed(7)
    length = 300
    c = Cache(length, hd)
    x = torch.randn(2, length, hd, generator=gen)
    x[part, -1] = torch.randn(hd, generator=gen).sign() * size
    lo, hi = x.amin(-1), x.amax(-1)
    c.low[:], c.step[:] = lo.half(), ((hi - lo) / 15).half()
    c.code[:] = ((x - c.low.float()[..., None]) / c.step.float()[..., None]).round().clamp(0, 15).to(torch.uint8)
    q = torch.randn(rows, 1, hd, generator=gen).half().cuda()
    _check(dev, c, q, hd ** -0.5, _bits(rows), copies=300, rows=slice(0, rows - 1))


@pytest.mark.parametrize("drop", [12.0, 18.0, 21.0, 23.4, 25.0])
@pytest.mark.parametrize("rows", [40, 200])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_one_strong_key_before_a_long_cache_of_a_prompt(dev, hd, rows, drop):
    _strong_key(dev, hd, rows, drop, 200)


@pytest.mark.parametrize("rows", [40, 200])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("size", [30.0, 3e3, 6e4])
@pytest.mark.parametrize("part", [0, 1])
def test_a_large_row_moves_none_of_a_prompt_that_does_not_see_it(dev, hd, rows, size, part):
    _large_row(dev, hd, rows, size, part)


def _long_sums(dev, hd, rows, copies):
    """60,000 keys whose values are positive; or whose greatest code stands for 0, in a channel that has no other: what a
    kernel sums does not cancel, the result does, and shows it.  An item's sums are long where it is one run.  The bound:
    the result's rounding, the weights' to 11 bits (each by chance, so 2^-11 / sqrt(10,000 keys that count) of the
    values), and 2^-14 for sums of 8,192 keys in steps of 16 that are cut off at 24 bits, 2^-24 each at most on average, in
    one part or two (1,024 2^-24)."""
    gen = torch.Generator().manual_seed(6)
    length = 60000
    c = Cache(length, hd)
    _octaves(c, torch.rand(length, generator=gen) * 2 - 1)
    c.code[1] = torch.randint(0, 16, (length, hd), generator=gen, dtype=torch.uint8)
    c.code[1, :, 0], c.code[1, :, 1] = 15, 0
    c.code[1, :, 2] = torch.randint(12, 16, (length,), generator=gen)
    c.step[1] = (torch.rand(length, generator=gen) * 0.02 + 0.05).half()
    q = torch.ones(rows, 1, hd, dtype=torch.float16, device="cuda")
    for low in (1.1, -15.0):
        c.low[1] = (torch.full((length,), low) if low > 0 else low * c.step[1].float()).half()
        got = _attend(dev, c, q, LN2, copies=copies)
        want, _ = _exact(c, q, LN2, 22)
        size = (c.values()[1].abs().mean(0) + 8 * 0.06)  # of a channel's terms, in values or centred codes
        bound = 2.0 ** -11 * want.abs() + (2.0 ** -11 * 0.01 + 2.0 ** -14) * size
        off = (got - want).abs() / bound
        assert (off <= 1).all(), (low, float(off.max()))


@pytest.mark.parametrize("rows,copies", [(1, 1), (1, 64), (1, 3000), (4, 1200), (7, 1600), (16, 1600)])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_long_sums_of_one_sign(dev, hd, rows, copies):
    _long_sums(dev, hd, rows, copies)


@pytest.mark.parametrize("rows,copies", [(40, 1), (40, 20), (40, 200), (200, 30), (300, 150)])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_long_sums_of_one_sign_of_a_prompt(dev, hd, rows, copies):
    _long_sums(dev, hd, rows, copies)
