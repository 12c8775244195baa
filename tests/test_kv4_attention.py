"""Attention over the paged 4-bit cache (gsvk_kv4_attention) against the formula in 64 bits."""
import ctypes

import numpy as np
import pytest
import torch

import kv4_ref as ref


def _case(rng, hd, kvh, group, page, kv_len, new, stale=255, scale=None, spread=1.0):
    """Pages of random rows (stale ones hold NaN parameters), a shuffled block table, packed queries."""
    kv_len, new = np.array(kv_len), np.array(new)
    blocks = -(-np.maximum(kv_len, 0) // page)
    n_pages = int(blocks.sum()) + 3
    order = rng.permutation(n_pages)
    table = np.full((len(kv_len), int(blocks.max(initial=0)) + 2), -1, np.int32)
    pages = ref.Pages(n_pages, page, kvh, hd, fill=stale)
    at = 0
    for i, n in enumerate(kv_len):
        table[i, :blocks[i]] = order[at:at + blocks[i]]
        at += blocks[i]
        for j in range(max(n, 0)):
            k = (rng.standard_normal((kvh, hd)) * spread + rng.standard_normal((kvh, 1))).astype(np.float16)
            v = (rng.standard_normal((kvh, hd)) + 0.5).astype(np.float16)
            pages.put(int(table[i, j // page]) * page + j % page, k, v)
    q_start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = rng.standard_normal((int(q_start[-1]), kvh * group, hd)).astype(np.float16)
    return pages, table, q_start, kv_len.astype(np.int32), q, scale if scale is not None else hd ** -0.5


def _run(dev, pages, table, q_start, kv_len, q, scale, prefix=None, max_q=None, extra=0, workspace=None, stream=None):
    """The call on strided rows between guard values; also checks that nothing beside the requests' rows is written."""
    n, heads, hd = q.shape
    wide = torch.zeros(n + extra, 3, heads, hd, dtype=torch.float16)
    wide[:n, 0] = torch.from_numpy(q)
    wide = wide.cuda()
    out = torch.full((n + extra, 2, heads, hd), 77.0, dtype=torch.float16).cuda()
    c = dev.KV4Cache(torch.from_numpy(pages.bytes).cuda(), pages.page, pages.heads, hd)
    cu = lambda a: None if a is None else torch.from_numpy(np.asarray(a, np.int32)).cuda()  # noqa: E731
    ws = workspace or dev.KV4Workspace(len(kv_len), n + extra, heads, pages.heads, hd)
    new = np.diff(q_start)
    args = (wide[:, 0], cu(q_start), cu(kv_len), cu(table), scale)
    if stream is not None:
        stream.wait_stream(torch.cuda.current_stream())
    c.attention(*args, max_q=int(new.max()) if max_q is None else max_q, workspace=ws, prefix=cu(prefix), out=out[:, 0],
                stream=stream)
    torch.cuda.synchronize()
    assert dev.device_status() == 0
    got = out.cpu().numpy()
    assert (got[:, 1] == 77).all()
    return got[:, 0].astype(np.float64)


def _check(dev, case, prefix=None, **kw):
    got = _run(dev, *case, prefix=prefix, **kw)
    pages, table, q_start, kv_len, q, scale = case
    want, tol = ref.attention(pages, q, q_start, kv_len, table, scale, prefix)
    n = len(q)
    assert (got[n:] == 77).all()
    for i in range(n):
        if np.isnan(want[i]).all():
            assert (got[i] == 77).all()  # a row of no request
    fine = ~np.isnan(want)
    off = np.abs(got[:n] - want)
    assert np.isfinite(got[:n][fine]).all()
    assert (off <= tol)[fine].all(), (off / np.maximum(tol, 1e-30))[fine].max()
    return got


DECODE = [0, 1, 2, 15, 16, 17, 31, 33, 64, 100, 127, 129, 300]


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("kvh,group,page", [(3, 1, 16), (2, 4, 32), (1, 7, 64), (2, 8, 128), (1, 16, 16), (1, 20, 32)])
def test_single_tokens(dev, hd, kvh, group, page):
    rng = np.random.default_rng(hd + group)
    _check(dev, _case(rng, hd, kvh, group, page, DECODE, [1] * len(DECODE)), extra=3)


@pytest.mark.gpu
@pytest.mark.parametrize("hd,kvh,group,page", [(32, 4, 1, 16), (64, 1, 3, 32), (128, 1, 2, 64), (64, 2, 1, 128)])
@pytest.mark.parametrize("with_prefix", [False, True])
def test_ragged_rows_and_prefixes(dev, hd, kvh, group, page, with_prefix):
    """Requests of 0 to 150 new rows behind caches of 0 to 260 tokens, some with more rows than keys (rows that see
    nothing), a prefix below, inside and past the length."""
    rng = np.random.default_rng(hd * 2 + page)
    new = [1, 0, 5, 17, 150, 40, 1, 64, 129, 3, 2, 30]
    kv = [77, 40, 5, 260, 150, 25, 0, 65, 200, 0, 1, 31]
    prefix = [0, 10, 3, 200, 150, 30, 5, 64, 1, 0, 9, 15] if with_prefix else None
    _check(dev, _case(rng, hd, kvh, group, page, kv, new), prefix=prefix, extra=2)


@pytest.mark.gpu
@pytest.mark.parametrize("hd,kvh,group,page,n,kv", [(64, 1, 1, 64, 700, 900), (128, 1, 1, 16, 300, 513),
                                                    (32, 1, 2, 32, 260, 260), (64, 1, 4, 128, 130, 1100)])
def test_prompts(dev, hd, kvh, group, page, n, kv):
    rng = np.random.default_rng(n)
    case = _case(rng, hd, kvh, group, page, [kv, 10, n + 1], [n, 2, n])
    _check(dev, case, prefix=[n // 3, 0, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("max_q", [0, 1, 10000])
def test_max_q_is_only_a_hint(dev, max_q):
    rng = np.random.default_rng(9)
    _check(dev, _case(rng, 64, 2, 2, 16, [40, 200, 9], [33, 140, 1]), max_q=max_q)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 40])
def test_long_caches_split_and_join(dev, n):
    """A single long request over the whole GPU, beside short ones."""
    rng = np.random.default_rng(11)
    _check(dev, _case(rng, 32, 1, 1, 16, [9000, 3, 700], [n, 1, 1]))


@pytest.mark.gpu
@pytest.mark.parametrize("scale,spread", [(0.0, 1.0), (3.0, 3.0), (-1.0, 1.0), (1e-4, 100.0)])
def test_scores_of_every_size(dev, scale, spread):
    rng = np.random.default_rng(12)
    case = _case(rng, 64, 2, 1, 16, [50, 333, 40], [1, 1, 30], scale=scale, spread=spread)
    _check(dev, case)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 150])
def test_pages_outside_the_pool_are_not_seen(dev, n):
    rng = np.random.default_rng(13)
    pages, table, q_start, kv_len, q, scale = _case(rng, 32, 2, 2, 16, [200, 170, 40, 160], [n, n, 1, n])
    table[0, 3], table[1, 0], table[2, :] = 10**6, -7, -1
    table[3, 9] = 2**31 - 1
    _check(dev, (pages, table, q_start, kv_len, q, scale))
    # a length past the table's last column: the keys there are not seen either
    kv_len = kv_len + np.array([0, 0, 0, 10**6], np.int32)
    _check(dev, (pages, table, q_start, kv_len, q, scale))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 130])
def test_a_nan_row_reaches_only_those_who_see_it(dev, n):
    rng = np.random.default_rng(14)
    case = pages, table, q_start, kv_len, q, scale = _case(rng, 64, 2, 1, 16, [150, 150], [n, 1])
    clean = _run(dev, *case)
    at = int(table[0, 140 // 16]) * 16 + 140 % 16
    k = np.full((2, 64), np.nan, np.float16)
    k[1] = 1
    v = np.ones((2, 64), np.float16)
    v[0] = np.nan
    pages.put(at, k, v)
    got = _run(dev, *case)
    first = max(0, 140 - (150 - n))  # the first row of request 0 that sees position 140
    assert np.isnan(got[first:n, 0]).all() and np.isfinite(got[:, 1]).all()
    np.testing.assert_array_equal(got[:first], clean[:first])
    np.testing.assert_array_equal(got[n:], clean[n:])


@pytest.mark.gpu
def test_nan_and_infinite_queries_stay_in_their_rows(dev):
    rng = np.random.default_rng(15)
    case = pages, table, q_start, kv_len, q, scale = _case(rng, 32, 2, 2, 16, [50, 90], [3, 1])
    clean = _run(dev, *case)
    q[1, 2, 5], q[3, 0, 0] = np.nan, np.inf
    got = _run(dev, *case)
    hit = np.zeros(got.shape[:2], bool)
    hit[1, 2] = hit[3, 0] = True
    assert np.isnan(got[hit]).all()
    np.testing.assert_array_equal(got[~hit], clean[~hit])


@pytest.mark.gpu
def test_the_same_call_gives_the_same_bits_on_any_stream(dev):
    rng = np.random.default_rng(16)
    case = _case(rng, 64, 2, 4, 16, [700, 33, 1200, 5], [1, 3, 1, 1])
    first = _run(dev, *case)
    ws = dev.KV4Workspace(64, 5000, 8, 2, 64)
    for _ in range(3):
        np.testing.assert_array_equal(_run(dev, *case, workspace=ws), first)
    np.testing.assert_array_equal(_run(dev, *case, workspace=ws, stream=torch.cuda.Stream()), first)


@pytest.mark.gpu
def test_a_captured_call_follows_its_inputs(dev):
    """Lengths, tables and pages are read on the device: a graph replays with new ones."""
    rng = np.random.default_rng(17)
    pages, table, q_start, kv_len, q, scale = _case(rng, 32, 2, 1, 16, [300, 40, 77], [1, 1, 1])
    c = dev.KV4Cache(torch.from_numpy(pages.bytes).cuda(), 16, 2, 32)
    cu = lambda a: torch.from_numpy(np.asarray(a)).cuda()  # noqa: E731
    tq, ts, tl, tt = cu(q), cu(q_start), cu(kv_len), cu(table)
    ws, out = dev.KV4Workspace(3, 3, 2, 2, 32), torch.zeros_like(tq)
    g = torch.cuda.CUDAGraph()
    c.attention(tq, ts, tl, tt, scale, 1, ws, out=out)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        c.attention(tq, ts, tl, tt, scale, 1, ws, out=out)
    kv_len = np.array([17, 40, 1], np.int32)
    tl.copy_(cu(kv_len))
    g.replay()
    torch.cuda.synchronize()
    want, tol = ref.attention(pages, q, q_start, kv_len, table, scale)
    assert (np.abs(out.cpu().numpy().astype(np.float64) - want) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 200])
def test_pages_past_32_bits_of_bytes(dev, n):
    rng = np.random.default_rng(18)
    pages, table, q_start, kv_len, q, scale = _case(rng, 128, 8, 1, 16, [230], [n])
    size = ref.page_bytes(16, 8, 128)
    n_pages = 2**32 // size + len(pages.bytes) + 5
    far = torch.zeros(n_pages, size, dtype=torch.uint8, device="cuda")
    far[-len(pages.bytes):] = torch.from_numpy(pages.bytes).cuda()
    moved = np.where(table >= 0, table + (n_pages - len(pages.bytes)), table).astype(np.int32)
    c = dev.KV4Cache(far, 16, 8, 128)
    cu = lambda a: torch.from_numpy(np.asarray(a)).cuda()  # noqa: E731
    out = c.attention(cu(q), cu(q_start), cu(kv_len), cu(moved), scale, n, dev.KV4Workspace(1, n, 8, 8, 128))
    want, tol = ref.attention(pages, q, q_start, kv_len, table, scale)
    assert (np.abs(out.cpu().numpy().astype(np.float64) - want) <= tol).all()


@pytest.mark.gpu
def test_wrapper_checks(dev):
    c = dev.KV4Cache.empty(4, 16, 2, 32)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.zeros(2, 4, 32, dtype=torch.float16, device="cuda")
    ws = dev.KV4Workspace(2, 2, 4, 2, 32)
    ok = dict(q=q, q_start=i32(3), kv_len=i32(2), block_table=i32(2, 4), scale=1.0, max_q=1, workspace=ws)
    c.attention(**ok)
    for over in (dict(q=q[:, :, :16]), dict(q_start=i32(2)), dict(kv_len=i32(1)), dict(block_table=i32(8)),
                 dict(prefix=i32(1)), dict(out=q[:1]), dict(q=q.transpose(0, 1))):
        with pytest.raises(ValueError):
            c.attention(**{**ok, **over})
    for over in (dict(q=q.float()), dict(kv_len=torch.zeros(2, dtype=torch.int64, device="cuda"))):
        with pytest.raises(TypeError):
            c.attention(**{**ok, **over})
    with pytest.raises(dev.GsvkError):  # 3 query heads over 2
        c.attention(**{**ok, "q": q[:, :3].contiguous()})
    with pytest.raises(ValueError):
        dev.KV4Workspace(2, 2, 3, 2, 32)


def _args(gsv, **over):
    from gsv_b200.quant import KV4AttentionArgs, KV4CacheArgs

    c = dict(pages=256, n_pages=4, page_size=16, kv_heads=2, head_dim=32)
    a = dict(q=256, q_stride=128, out=256, out_stride=128, heads=4, n_tokens=2, n_seq=2, max_blocks=4, max_q=1,
             q_start=256, kv_len=256, prefix=None, block_table=256, scale=1.0, workspace=256, workspace_bytes=1 << 40)
    for k, v in over.items():
        (c if k in c else a)[k] = v
    return gsv.lib().gsvk_kv4_attention(ctypes.byref(KV4AttentionArgs(cache=KV4CacheArgs(**c), **a)), None)


@pytest.mark.parametrize("over,rc", [
    (dict(pages=None), -1), (dict(q=None), -1), (dict(out=None), -1), (dict(q_start=None), -1), (dict(kv_len=None), -1),
    (dict(block_table=None), -1), (dict(workspace=None), -1), (dict(heads=0), -1), (dict(n_seq=0), -1),
    (dict(max_blocks=0), -1), (dict(heads=3), -1), (dict(workspace_bytes=0), -1), (dict(q_stride=64), -1),
    (dict(out_stride=120), -1), (dict(page_size=20), -5), (dict(head_dim=96), -5), (dict(n_seq=16385), -5),
    (dict(max_blocks=2**40), -5), (dict(heads=2**20), -5), (dict(n_tokens=2**40), -5), (dict(q=264), -2),
    (dict(out=8), -2), (dict(q_stride=132), -2), (dict(workspace=272), -2), (dict(n_tokens=0), 0)])
def test_bad_arguments_are_refused_before_any_launch(gsv, over, rc):
    assert _args(gsv, **over) == rc
