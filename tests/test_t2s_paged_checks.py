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
