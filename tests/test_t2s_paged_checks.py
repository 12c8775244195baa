"""What T2SPaged refuses, and that a refused call leaves the requests as they were."""
import types

import pytest
import torch


def _host(gsv, rows=0):
    """A T2SPaged without a device: the checks come before anything runs."""
    t2s = object.__new__(gsv.T2SPaged)
    t2s.plan = types.SimpleNamespace(q_start=torch.tensor([0, rows, rows], dtype=torch.int32))
    return t2s


def test_no_rows_have_no_logits(gsv):
    """An index into no rows would be a device assertion."""
    for call in ("logits", "greedy"):
        with pytest.raises(ValueError, match="rows"):
            getattr(_host(gsv), call)(torch.zeros(0, 8))


def test_a_refused_step_plans_nothing(gsv):
    t2s = _host(gsv)
    t2s.d_model, t2s.max_tokens, t2s.max_seq, t2s.layers = 8, 4, 2, []
    t2s.length = t2s.block_table = t2s.free_pages = t2s.free_count = None
    t2s.plan.run = lambda *a, **k: pytest.fail("a step was planned")
    for x in (torch.zeros(4, 8, dtype=torch.float16), torch.zeros(4, 7), torch.zeros(4), torch.zeros(8).expand(4, 8)):
        with pytest.raises((ValueError, TypeError)):
            t2s.step(x, None, 1)


@pytest.mark.gpu
def test_a_refused_step_leaves_the_lengths(dev):
    import test_t2s_paged as paged

    m = paged._model(dev, 9)
    t2s = dev.T2SPaged(m, max_seq=2, max_tokens=64, max_len=64, n_pages=8, page_size=16)
    x = torch.randn(5, m["d_model"], device="cuda")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    new = i32(2, 3)
    first = t2s.step(x, new, 3)
    for bad in (dict(x=x.half()), dict(x=x[:, :-1]), dict(x=x[:1].expand(5, -1)), dict(x=x.cpu()), dict(prefix=i32(1)),
                dict(prefix=torch.zeros(2, dtype=torch.int64, device="cuda")), dict(x=torch.zeros(65, m["d_model"], device="cuda"))):
        with pytest.raises((ValueError, TypeError)):
            t2s.step(**{**dict(x=x, new_len=new, max_q=3), **bad})
        assert t2s.length.tolist() == [2, 3] and int(t2s.free_count) == 6
    # a step in which every request rests
    assert t2s.step(x[:0], i32(0, 0), 0).shape == (0, m["d_model"])
    assert t2s.length.tolist() == [2, 3] and int(t2s.plan.refused) == 0
    # rows apart from each other are rows
    t2s.release(i32(1, 1))
    wide = torch.zeros(5, m["d_model"] + 4, device="cuda")
    wide[:, :-4] = x
    assert torch.equal(t2s.step(wide[:, :-4], new, 3), first)
