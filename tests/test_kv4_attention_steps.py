"""Whole steps of the attention over the paged 4-bit cache: many requests of every size in one call, and scores that keep
rising, against the formula in 64 bits on the GPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _pages(gen, n_pages, page, kvh, hd, steps):
    """Random codes, steps in [0, steps) and lows as fp16, in the documented layout, and what they stand for."""
    codes = torch.randint(0, 256, (n_pages, kvh, 2, page, hd // 2), generator=gen, dtype=torch.uint8)
    par = torch.empty(n_pages, kvh, 2, page, 2)
    par[..., 0] = torch.rand(par.shape[:-1], generator=gen) * steps
    par[..., 1] = torch.randn(par.shape[:-1], generator=gen) - 7.5 * par[..., 0]
    par = par.half()
    raw = torch.cat([codes.reshape(n_pages, kvh, -1), par.view(torch.uint8).reshape(n_pages, kvh, -1)], -1)
    c = torch.stack([codes & 15, codes >> 4], -1).reshape(n_pages, kvh, 2, page, hd).double()
    return raw.reshape(n_pages, -1).contiguous().cuda(), (c * par[..., :1].double() + par[..., 1:].double()).cuda()


def _plain(values, table, q, q_start, kv_len, prefix, scale):
    n_pages, kvh, _, page, hd = values.shape
    heads = q.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for i, length in enumerate(kv_len):
        a, b = q_start[i], q_start[i + 1]
        if a == b:
            continue
        rows = table[i, :-(-length // page)].long()
        there = ((rows >= 0) & (rows < n_pages)).repeat_interleave(page)[:length]
        kv = values[rows.clamp(0, n_pages - 1)].permute(1, 2, 0, 3, 4).reshape(kvh, 2, -1, hd)[:, :, :length]
        k, v = (kv[:, j].repeat_interleave(heads // kvh, 0) for j in (0, 1))
        z = torch.einsum("thd,hjd->htj", q[a:b].double(), k) * scale
        limit = length - (b - a) + torch.arange(b - a, device="cuda") + 1
        limit = limit.clamp(min=prefix[i]).clamp(max=length)
        seen = (torch.arange(length, device="cuda") < limit[:, None]) & there
        p = torch.softmax(z.masked_fill(~seen, -torch.inf), -1).nan_to_num(0.0)
        out[a:b] = torch.einsum("htj,hjd->thd", p, v)
    return out


def _run(dev, values, raw, table, q, q_start, kv_len, prefix, scale, page):
    n_pages, kvh, _, _, hd = values.shape
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    cache = dev.KV4Cache(raw, page, kvh, hd)
    ws = dev.KV4Workspace(len(kv_len), len(q), q.shape[1], kvh, hd)
    out = cache.attention(q, i32(q_start), i32(kv_len), table, scale, max(b - a for a, b in zip(q_start, q_start[1:])), ws,
                          prefix=i32(prefix))
    torch.cuda.synchronize()
    assert dev.device_status() == 0
    return out.double()


def _close(got, want, steps, most, scores):
    """The output's rounding; the weights' to fp16 against codes centred within 8 steps; 32-bit sums, statistics and
    exponentials, and the scores' own rounding, 2^-18 each of the greatest value."""
    bound = 2.0 ** -11 * want.abs() + 2.0 ** -11 * 8 * steps + 2.0 ** -18 * (2 + scores) * most
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("hd,kvh,group,page", [(32, 2, 4, 16), (64, 2, 4, 32), (128, 2, 4, 32), (64, 3, 1, 64), (128, 1, 1, 128)])
@pytest.mark.parametrize("seed", [1, 2, 3])
def test_steps_of_many_requests(dev, hd, kvh, group, page, seed):
    """Single tokens, drafts and prompts side by side; blocks of one and of two groups of rows follow each other."""
    gen = torch.Generator().manual_seed(seed)
    pick = lambda lo, hi: int(torch.randint(lo, hi + 1, (), generator=gen))  # noqa: E731
    new = [pick(0, 3) if i % 4 == 3 else pick(60 // group, 700 // group) for i in range(24)]
    kv_len = [n + pick(0, 1500) for n in new]
    prefix = [pick(0, k) for k in kv_len]
    blocks = [-(-k // page) for k in kv_len]
    raw, values = _pages(gen, sum(blocks) + 1, page, kvh, hd, 0.2)
    order = torch.randperm(sum(blocks), generator=gen).to(torch.int32)
    table = torch.full((24, max(blocks)), -1, dtype=torch.int32)
    for i, b in enumerate(blocks):
        table[i, :b] = order[sum(blocks[:i]):sum(blocks[:i]) + b]
    table = table.cuda()
    q_start = [sum(new[:i]) for i in range(25)]
    q = torch.randn(q_start[-1], kvh * group, hd, generator=gen).half().cuda()
    args = (table, q, q_start, kv_len, prefix, hd ** -0.5)
    want = _plain(values, *args)
    got = _run(dev, values, raw, *args, page)
    _close(got, want, 0.2, float(values.abs().max()), 16 * 3 * hd ** 0.5)
    for _ in range(3):
        assert torch.equal(_run(dev, values, raw, *args, page), got)


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("rise", [0.05, 0.4, 3.0, 40.0])
@pytest.mark.parametrize("missing", [0, 3, 5])
def test_scores_that_keep_rising(dev, hd, rise, missing):
    """Every key outdoes the ones before by `rise` octaves, or falls behind them (half of the heads), or they rise at one
    key alone; the first pages may be missing, so that rows start late."""
    gen = torch.Generator().manual_seed(7)
    page, n, length = 32, 160, 700
    raw, values = _pages(gen, -(-length // page), page, 1, hd, 0.1)
    # dimension 0 of K: a constant row there gives the position's score
    j = torch.arange(length, dtype=torch.float64)
    z = torch.stack([j * rise, -j * rise, torch.where(j >= 331, rise * 60.0, 0.0)])
    q = torch.zeros(n, 3, hd, dtype=torch.float16)
    q[:, 0], q[:, 1], q[:, 2] = 1.0, -1.0, 1.0
    b = raw.view(-1, page * (hd + 8))
    par = b[:, page * hd:].view(torch.float16).view(-1, 2, page, 2)
    for head in (0, 2):  # K rows of one value each: step 0, low = score / (hd q scale)
        low = (z[head] / hd).half()
        flat = torch.zeros(par.shape[0] * page, dtype=torch.float16)
        flat[:length] = low
        par[:, 0, :, 0] = 0
        par[:, 0, :, 1] = flat.view(-1, page).cuda()
        values[:, 0, 0] = par[:, 0, :, 1].double()[..., None]
        rows = [0, 1] if head == 0 else [2]
        table = torch.arange(par.shape[0], dtype=torch.int32, device="cuda")[None].clone()
        table[:, :missing] = -1
        qq = q[:, rows].contiguous().cuda()
        args = (table, qq, [0, n], [length], [0], 0.6931471805599453)
        got, want = _run(dev, values, raw, *args, page), _plain(values, *args)
        top = float((values[:, 0, 0].abs().max() * hd) * 0.7)
        _close(got, want, 0.1, float(values[:, 0, 1].abs().max()), top)
