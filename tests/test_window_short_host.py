"""Host-side checks of how many launches short sequences beside longer ones take; no GPU."""

from __future__ import annotations

import torch

from gdn2_sm120_b200.attention import _apart, _keeps_rest, _launches


def _bounds(lengths):
    return tuple(sum(lengths[:i]) for i in range(len(lengths) + 1))


def test_launches_of_short_sequences_apart():
    assert _launches(None, True) == 1 and _launches((0, 0, 0), True) == 0
    assert _launches(_bounds((128, 1, 0)), True) == _launches(_bounds((129, 700)), True) == 1
    assert _launches(_bounds((128, 129)), True) == 2 and _launches(_bounds((128, 129))) == 1
    assert _launches(_bounds((3,) * 256 + (300,)), True) == 2 and _launches(_bounds((3,) * 255 + (300,) * 2), True) == 3


def test_a_window_over_everything():
    q = torch.zeros(1, 30, 1, 8)
    assert _apart(q, None, (30, 0)) and not _apart(q, None, (29, 0)) and not _apart(q, None, (0, 0))
    assert _apart(q, (0, 10, 10, 30), (20, 5)) and not _apart(q, (0, 10, 10, 30), (19, 5))


def test_what_is_kept_for_the_backward():
    q, long = torch.zeros(1, 30, 1, 8), torch.zeros(1, 300, 1, 8)
    assert _keeps_rest(q, None, (29, 0)) and _keeps_rest(q, None, (2 ** 30, 0)) and not _keeps_rest(q, None, (0, 0))
    assert _keeps_rest(long, None, (299, 0)) and not _keeps_rest(long, None, (300, 0))
    assert _keeps_rest(long, (0, 128, 300), (200, 0)) and _keeps_rest(long, (0, 129, 300), (170, 0))
    assert not _keeps_rest(long, (0, 129, 129, 300), (171, 0)) and not _keeps_rest(long, (0, 300, 300), (300, 7))
