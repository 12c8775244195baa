"""Rows into and out of the paged 4-bit cache (gsvk_kv4_append, gsvk_kv4_read): bytes and values against the rule."""
import ctypes

import numpy as np
import pytest
import torch

import kv4_ref as ref


def _rows(rng, n, heads, hd, dtype):
    x = rng.standard_normal((n, heads, hd)) * rng.choice([1e-3, 1, 30], (n, heads, 1)) + rng.standard_normal((n, heads, 1))
    return x.astype(dtype)


def _special(x):
    """Rows at the edges: constant, zero, one outlier, ties, subnormal steps, the greatest fp16, NaN, infinities."""
    n, hd = x.shape[0], x.shape[2]
    for i, f in enumerate((lambda r: r.fill(3.25), lambda r: r.fill(0), lambda r: (r.fill(0), r.__setitem__(5, 1000)),
                           lambda r: r.__setitem__(slice(None), (np.arange(hd) % 31) * 0.5),
                           lambda r: r.__setitem__(slice(None), np.arange(hd) * 6e-8),
                           lambda r: (r.__setitem__(0, 65504), r.__setitem__(1, -65504)),
                           lambda r: r.__setitem__(3, np.nan), lambda r: r.__setitem__(7, np.inf),
                           lambda r: r.__setitem__(hd - 1, -np.inf))):
        if i < n:
            f(x[i, i % x.shape[1]])
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("n,heads,hd,page", [(1, 1, 32, 16), (13, 16, 32, 16), (40, 3, 64, 32), (33, 1, 128, 64),
                                             (70, 5, 128, 128), (257, 2, 64, 16)])
def test_append_writes_the_rules_bytes(dev, n, heads, hd, page, dtype):
    rng = np.random.default_rng(n + hd)
    n_pages = n // page + 4
    slots = rng.permutation(n_pages * page)[:n].astype(np.int64)
    if n > 12:
        slots[[10, 11, 12]] = [-1, n_pages * page, 2**40]  # outside the cache: skipped
    k, v = _special(_rows(rng, n, heads, hd, dtype)), _special(_rows(rng, n, heads, hd, dtype)[::-1].copy())
    want = ref.Pages(n_pages, page, heads, hd, fill=170)
    for t in range(n):
        if 0 <= slots[t] < n_pages * page:
            want.put(slots[t], k[t], v[t])
    c = dev.KV4Cache(torch.full((n_pages, ref.page_bytes(page, heads, hd)), 170, dtype=torch.uint8).cuda(), page, heads, hd)
    # K and V as slices of wider rows
    wide = torch.zeros(n, 3, heads, hd, dtype=torch.from_numpy(k).dtype)
    wide[:, 1], wide[:, 2] = torch.from_numpy(k), torch.from_numpy(v)
    wide = wide.cuda()
    s = torch.from_numpy(slots).cuda()
    c.append(wide[:, 1], wide[:, 2], s)
    got = c.pages.cpu().numpy()
    bad = np.flatnonzero((got != want.bytes).any(1))
    # NaN parameters may carry any NaN
    a, b = got.copy().view(np.float16), want.bytes.copy().view(np.float16)
    assert ((got.view(np.uint16) == want.bytes.view(np.uint16)) | (np.isnan(a) & np.isnan(b))).all(), bad
    rk, rv = c.read(s)
    for t in range(n):
        if 0 <= slots[t] < n_pages * page:
            w = want.get(slots[t])
            for x, y in ((rk, w[0]), (rv, w[1])):
                x = x[t].cpu().numpy().astype(np.float64)
                assert (np.isnan(x) == np.isnan(y)).all()
                fine = ~np.isnan(y)
                # one fp32 rounding, then one to fp16, which keeps to its range
                tol = 2**-11 * np.abs(y) + 2**-25 + 2**-24 * np.abs(y)
                assert (np.abs(x - np.clip(y, -65504, 65504)) <= tol)[fine].all()
        else:
            assert not rk[t].any() and not rv[t].any()


@pytest.mark.gpu
def test_a_row_is_within_half_a_step(dev):
    """What comes back is within half a step of the row (and the roundings of step and low to fp16)."""
    rng = np.random.default_rng(5)
    k = _rows(rng, 64, 4, 128, np.float16)
    c = dev.KV4Cache(torch.zeros(4, ref.page_bytes(16, 4, 128), dtype=torch.uint8).cuda(), 16, 4, 128)
    s = torch.randperm(64).cuda()
    c.append(torch.from_numpy(k).cuda(), torch.from_numpy(k).cuda(), s)
    got = c.read(s)[0].cpu().numpy().astype(np.float64)
    x = k.astype(np.float64)
    span = x.max(-1, keepdims=True) - x.min(-1, keepdims=True)
    # half a step; a step that fp16 rounds by 2^-11 shifts the 15th level by as much of the span; output rounding
    assert (np.abs(got - x) <= span / 30 + span * 2**-11 + np.abs(x) * 2**-11 + 1e-6).all()


@pytest.mark.gpu
def test_read_into_strided_rows_and_one_side_only(dev):
    rng = np.random.default_rng(6)
    c = dev.KV4Cache(torch.zeros(3, ref.page_bytes(16, 2, 32), dtype=torch.uint8).cuda(), 16, 2, 32)
    x = torch.from_numpy(_rows(rng, 20, 2, 32, np.float16)).cuda()
    s = torch.arange(20).cuda() + 7
    c.append(x, -x, s)
    k, v = c.read(s)
    wide = torch.full((20, 2, 2, 32), 7.0, dtype=torch.float16).cuda()
    assert c.read(s, v=wide[:, 1])[0] is None
    assert torch.equal(wide[:, 1], v) and (wide[:, 0] == 7).all()
    c.read(s, k=wide[:, 0])
    assert torch.equal(wide[:, 0], k)
    empty = torch.empty(0, dtype=torch.int64).cuda()
    assert c.read(empty)[0].shape == (0, 2, 32)
    c.append(x[:0], x[:0], empty)


@pytest.mark.gpu
def test_slots_past_32_bits_of_bytes(dev):
    """A cache of over 4 GiB: the last slots are where they should be."""
    page, heads, hd = 16, 8, 128
    size = ref.page_bytes(page, heads, hd)
    n_pages = 2**32 // size + 40
    c = dev.KV4Cache(torch.zeros(n_pages, size, dtype=torch.uint8, device="cuda"), page, heads, hd)
    rng = np.random.default_rng(8)
    x = torch.from_numpy(_rows(rng, 3, heads, hd, np.float16)).cuda()
    s = torch.tensor([n_pages * page - 1, 5, (2**32 // size + 2) * page]).cuda()
    c.append(x, x + 1, s)
    want = ref.Pages(3, page, heads, hd, fill=0)
    for i in range(3):
        want.put(i * page + int(s[i]) % page, x[i].cpu().numpy(), (x[i] + 1).cpu().numpy())
    assert (c.pages[s // page].cpu().numpy() == want.bytes).all()
    assert int(c.pages[6:2**32 // size].count_nonzero()) == 0


@pytest.mark.gpu
def test_wrapper_checks(dev):
    c = dev.KV4Cache.empty(2, 16, 2, 32)
    x = torch.zeros(4, 2, 32, dtype=torch.float16, device="cuda")
    s = torch.zeros(4, dtype=torch.int64, device="cuda")
    for bad in (lambda: c.append(x, x[:, :1], s), lambda: c.append(x[:3], x, s), lambda: c.append(x, x, s[:2]),
                lambda: c.append(x.cpu(), x, s), lambda: c.append(x.transpose(0, 1), x, s),
                lambda: dev.KV4Cache(c.pages, 24, 2, 32), lambda: dev.KV4Cache(c.pages.view(-1)[:-1], 16, 2, 32),
                lambda: dev.KV4Cache.empty(2, 16, 2, 48), lambda: c.read(s, k=x[:2])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: c.append(x.double(), x.double(), s), lambda: c.append(x, x.float(), s),
                lambda: c.append(x, x, s.int())):
        with pytest.raises(TypeError):
            bad()
    odd = torch.zeros(4 * 68, dtype=torch.float16, device="cuda").as_strided((4, 2, 32), (68, 32, 1))
    with pytest.raises(dev.GsvkError) as e:
        c.append(odd, x, s)
    assert e.value.code == -2


def test_page_bytes(gsv):
    assert gsv.kv4_page_bytes(16, 16, 32) == 16 * 16 * 40
    for bad in ((24, 1, 32), (16, 0, 32), (16, 1025, 32), (16, 1, 96), (-16, 1, 32), (16, 1, 0)):
        assert gsv.kv4_page_bytes(*bad) == 0


def _cache(**over):
    from gsv_b200.quant import KV4CacheArgs

    a = dict(pages=256, n_pages=4, page_size=16, kv_heads=2, head_dim=32)
    a.update(over)
    return ctypes.byref(KV4CacheArgs(**a))


@pytest.mark.parametrize("over,rc", [(dict(pages=None), -1), (dict(n_pages=0), -1), (dict(page_size=8), -5),
                                     (dict(kv_heads=0), -5), (dict(head_dim=40), -5), (dict(n_pages=2**31), -5),
                                     (dict(pages=264), -2)])
def test_bad_caches_are_refused_before_any_launch(gsv, over, rc):
    L = gsv.lib()
    assert L.gsvk_kv4_append(_cache(**over), 256, 64, 256, 64, 0, 256, 1, None) == rc
    assert L.gsvk_kv4_read(_cache(**over), 256, 1, 256, 64, 256, 64, None) == rc


def test_bad_rows_are_refused_before_any_launch(gsv):
    L = gsv.lib()
    assert L.gsvk_kv4_append(None, 256, 64, 256, 64, 0, 256, 1, None) == -1
    assert L.gsvk_kv4_append(_cache(), None, 64, 256, 64, 0, 256, 1, None) == -1
    assert L.gsvk_kv4_append(_cache(), 256, 64, 256, 64, 0, None, 1, None) == -1
    assert L.gsvk_kv4_append(_cache(), 256, 32, 256, 64, 0, 256, 2, None) == -1
    assert L.gsvk_kv4_append(_cache(), 256, 68, 256, 64, 0, 256, 2, None) == -2
    assert L.gsvk_kv4_append(_cache(), 258, 64, 256, 64, 0, 256, 2, None) == -2
    assert L.gsvk_kv4_append(_cache(), 256, 64, 256, 64, 0, 256, 2**40, None) == -5
    assert L.gsvk_kv4_append(_cache(), 256, 64, 256, 64, 0, 256, 0, None) == 0
    assert L.gsvk_kv4_read(_cache(), 256, 1, None, 0, None, 0, None) == -1
    assert L.gsvk_kv4_read(_cache(), 256, 2, 256, 68, None, 0, None) == -2
    assert L.gsvk_kv4_read(_cache(), 256, 0, 256, 64, None, 0, None) == 0
