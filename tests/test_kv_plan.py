"""The page planner (gsvk_kv_plan) and the return of pages (gsvk_kv_release) against the request-by-request rule."""
import ctypes

import numpy as np
import pytest
import torch

import kv4_ref as ref


def _state(rng, n_seq, page, ctx, new, spare, count=None, max_blocks=None):
    blocks = np.maximum(0, -(-(ctx + np.maximum(new, 0)) // page))
    have = np.maximum(0, -(-ctx // page))
    max_blocks = max_blocks or int(max(blocks.max(), have.max())) + 1
    n_pages = int(blocks.sum() + have.sum()) + spare
    order = rng.permutation(n_pages).astype(np.int32)
    table = np.full((n_seq, max_blocks), -1, np.int32)
    used = 0
    for i in range(n_seq):
        h = min(int(have[i]), max_blocks)
        table[i, :h] = order[used:used + h]
        used += h
    free = np.full(n_pages, -1, np.int32)
    free[:n_pages - used] = order[used:]
    return table, free, n_pages, (n_pages - used if count is None else count)


def _run(dev, ctx, new, table, free, count, n_pages, page, max_tokens, in_place=False):
    t = [torch.from_numpy(np.array(x)).cuda() for x in (ctx, new, table, free, np.array([count], np.int32))]
    p = dev.KVPlan(len(ctx), table.shape[1], page, n_pages, max_tokens)
    p.run(*t, in_place=in_place)
    return p, t


def _same(p, t, want, in_place=False):
    q_start, kv_len, table, slots, left, refused = want
    np.testing.assert_array_equal(p.q_start.cpu().numpy(), q_start)
    np.testing.assert_array_equal((t[0] if in_place else p.kv_len).cpu().numpy(), kv_len)
    np.testing.assert_array_equal(t[2].cpu().numpy(), table)
    np.testing.assert_array_equal(p.slots.cpu().numpy(), slots)
    assert int(t[4] if in_place else p.free_left) == left
    assert int(p.refused) == refused


@pytest.mark.gpu
@pytest.mark.parametrize("n_seq,page,ctx_hi,new_hi,share,in_place", [
    (1, 16, 1, 1, 1.0, False), (1, 128, 1000, 3000, 1.0, False), (64, 16, 1024, 1, 1.0, True),
    (63, 32, 70, 200, 1.0, False), (1025, 64, 300, 33, 1.0, False), (1500, 16, 100, 40, 0.4, False),
    (300, 16, 64, 300, 0.5, True), (16384, 16, 20, 2, 0.7, False), (7, 16, 0, 5000, 0.9, True)])
def test_plan_matches_the_rule(dev, n_seq, page, ctx_hi, new_hi, share, in_place):
    rng = np.random.default_rng(n_seq * 7 + page)
    ctx = rng.integers(0, ctx_hi + 1, n_seq).astype(np.int32)
    new = rng.integers(0, new_hi + 1, n_seq).astype(np.int32)
    table, free, n_pages, count = _state(rng, n_seq, page, ctx, new, 3)
    need = int((-(-(ctx + new) // page) - -(-ctx // page)).sum())
    count = min(count, int(need * share) + (share == 1.0))
    max_tokens = int(new.sum()) + 9
    want = ref.plan(ctx, new, table, free, count, page, table.shape[1], max_tokens)
    p, t = _run(dev, ctx, new, table, free, count, n_pages, page, max_tokens, in_place)
    _same(p, t, want, in_place)
    if not in_place:  # inputs kept: the same call gives the same
        p.run(*t)
        _same(p, t, want)


@pytest.mark.gpu
def test_plan_refuses_what_does_not_fit(dev):
    """Negative lengths, tables that are too short, rows past max_tokens, and requests behind the first shortage."""
    ctx = np.array([5, -3, 30, 0, 16, 40, 2**31 - 1, 3, 0], np.int32)
    new = np.array([3, 2, 40, 20, 0, -7, 2**31 - 1, 1, 0], np.int32)
    page, max_blocks, max_tokens = 16, 4, 70
    table = np.full((9, max_blocks), -1, np.int32)
    table[0, 0], table[2, :2], table[4, 0], table[5, :3], table[7, 0] = 9, (8, 7), 6, (5, 4, 3), 2
    free = np.array([1, 0, 10, 11] + [-1] * 8, np.int32)
    want = ref.plan(ctx, new, table, free, 4, page, max_blocks, max_tokens)
    assert want[5] == 6  # the negative ones, the table, and all behind the row bound
    p, t = _run(dev, ctx, new, table, free, 4, 12, page, max_tokens)
    _same(p, t, want)


@pytest.mark.gpu
def test_a_plan_in_place_steps_on_and_pages_come_back(dev):
    """Steps in place until the pool is short, release, and the pool holds every page once again."""
    rng = np.random.default_rng(3)
    n_seq, page, n_pages = 40, 16, 200
    dev_i = lambda a: torch.from_numpy(np.asarray(a, np.int32)).cuda()  # noqa: E731
    length, count = dev_i(np.zeros(n_seq)), dev_i([n_pages])
    free, table = dev_i(rng.permutation(n_pages)), dev_i(np.full((n_seq, 30), -1))
    p = dev.KVPlan(n_seq, 30, page, n_pages, 4000)
    total = np.zeros(n_seq, np.int64)
    refused = 0
    for step in range(14):
        new = rng.integers(0, 30, n_seq).astype(np.int32)
        before = length.cpu().numpy()
        p.run(length, dev_i(new), table, free, count, in_place=True)
        after = length.cpu().numpy()
        refused += int(p.refused)
        assert ((after == before + new) | (after == before)).all()
        total = after
        held = table.cpu().numpy()
        ids = np.concatenate([held[i, :-(-int(total[i]) // page)] for i in range(n_seq)] +
                             [free.cpu().numpy()[:int(count)]])
        assert sorted(ids.tolist()) == list(range(n_pages))
    assert refused > 0
    done = rng.integers(0, 2, n_seq).astype(np.int32)
    want_free = free.cpu().numpy()[:int(count)].tolist()
    for i in np.flatnonzero(done):
        want_free += held[i, :-(-int(total[i]) // page)].tolist()
    p.release(dev_i(done), length, table, free, count)
    assert free.cpu().numpy()[:int(count)].tolist() == want_free
    np.testing.assert_array_equal(length.cpu().numpy(), np.where(done, 0, total))
    assert (table.cpu().numpy()[done == 1][:, 0] == -1).all()
    p.release(dev_i(np.ones(n_seq)), length, table, free, count)
    assert sorted(free.cpu().numpy()[:int(count)].tolist()) == list(range(n_pages))
    p.release(dev_i(np.ones(n_seq)), length, table, free, count)  # nothing is returned twice
    assert int(count) == n_pages


@pytest.mark.gpu
def test_release_keeps_to_the_pool(dev):
    """Entries outside the pool stay out, and a list that is full takes no more."""
    dev_i = lambda a: torch.from_numpy(np.asarray(a, np.int32)).cuda()  # noqa: E731
    p = dev.KVPlan(2, 3, 16, 4, 8)
    table, length = dev_i([[7, 2, -1], [3, 1, 0]]), dev_i([40, 200])
    free, count = dev_i([0, 1, -5, -5, 99]), dev_i([2])
    p.release(dev_i([1, 1]), length, table, free, count)
    assert free.cpu().tolist() == [0, 1, 2, 3, 99] and int(count) == 4
    assert length.cpu().tolist() == [0, 0]


@pytest.mark.gpu
def test_plan_on_another_stream(dev):
    s = torch.cuda.Stream()
    ctx, new = np.array([3, 100], np.int32), np.array([2, 30], np.int32)
    rng = np.random.default_rng(0)
    table, free, n_pages, count = _state(rng, 2, 16, ctx, new, 2)
    t = [torch.from_numpy(np.array(x)).cuda() for x in (ctx, new, table, free, np.array([count], np.int32))]
    p = dev.KVPlan(2, table.shape[1], 16, n_pages, 40)
    s.wait_stream(torch.cuda.current_stream())
    p.run(*t, stream=s)
    s.synchronize()
    _same(p, t, ref.plan(ctx, new, table, free, count, 16, table.shape[1], 40))


def _args(gsv, **over):
    from gsv_b200.quant import KVPlanArgs

    a = dict(n_seq=2, max_blocks=4, n_pages=8, max_tokens=8, page_size=16)
    a.update({n: 256 for n in ("ctx_len", "new_len", "block_table", "free_pages", "free_count", "q_start", "kv_len",
                               "slots", "free_left", "refused", "workspace")})
    a.update(over)
    return gsv.lib().gsvk_kv_plan(ctypes.byref(KVPlanArgs(**a)), None)


@pytest.mark.parametrize("over,rc", [
    (dict(n_seq=0), -1), (dict(max_blocks=0), -1), (dict(n_pages=0), -1), (dict(max_tokens=0), -1),
    (dict(slots=None), -1), (dict(workspace=None), -1), (dict(free_count=None), -1), (dict(page_size=24), -5),
    (dict(page_size=0), -5), (dict(n_seq=16385), -5), (dict(max_blocks=2**60), -5), (dict(max_tokens=2**31), -5),
    (dict(n_pages=2**31), -5)])
def test_plan_refuses_bad_arguments_before_any_launch(gsv, over, rc):
    assert _args(gsv, **over) == rc
    assert "kv_plan" in gsv.last_error()


def test_release_refuses_bad_arguments_before_any_launch(gsv):
    L = gsv.lib()
    assert L.gsvk_kv_plan(None, None) == -1
    assert L.gsvk_kv_release(1, 1, 1, 16, None, 256, 256, 256, 256, None) == -1
    assert L.gsvk_kv_release(0, 1, 1, 16, 256, 256, 256, 256, 256, None) == -1
    assert L.gsvk_kv_release(1, 1, 1, 17, 256, 256, 256, 256, 256, None) == -5
    assert L.gsvk_kv_release(20000, 1, 1, 16, 256, 256, 256, 256, 256, None) == -5
