"""The return of pages at the end of what 32 bits count."""
import pytest
import torch


@pytest.mark.gpu
def test_a_full_list_of_2_31_pages_takes_no_more(dev):
    """Places past the last entry are past 2^31 - 1 too: nothing is written, least of all before the list."""
    n_pages = 2**31 - 1
    guard, blocks = 1024, 70
    memory = torch.full((n_pages + 2 * guard,), -3, dtype=torch.int32, device="cuda")
    free = memory[guard:guard + n_pages]
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    p = dev.KVPlan(3, blocks, 16, n_pages, 8)
    for held, back in ((n_pages, 0), (n_pages - 2, 2), (n_pages - 100, 100)):
        table = torch.arange(3 * blocks, dtype=torch.int32, device="cuda").view(3, blocks).contiguous()
        length, count = i32(16 * blocks, 16 * blocks, 5), i32(held)
        p.release(i32(1, 1, 1), length, table, free, count)
        assert int(count) == n_pages and (table[:2] == -1).all() and length.tolist() == [0, 0, 0]
        want = torch.arange(2 * blocks + 1, dtype=torch.int32, device="cuda")[:back]
        assert torch.equal(free[held:], want)
        assert int((memory != -3).sum()) == back
        free[held:] = -3
