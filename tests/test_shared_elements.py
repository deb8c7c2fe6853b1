"""Which strided tensors share elements (checked before a call writes into given tensors), against all their addresses."""

from __future__ import annotations

import itertools
import random

import pytest
import torch

from gdn2_sm120_b200 import _validate


def _bytes(x):
    places = [0]
    for n, s in zip(x.shape, x.stride()):
        places = [p + i * s for p in places for i in range(n)]
    lo, es = x.data_ptr(), x.element_size()
    return [lo + p * es + b for p in places for b in range(es)]


def test_random_views_against_all_addresses():
    rng = random.Random(0)
    base = torch.zeros(4000, dtype=torch.int16)
    seen = {True: 0, False: 0}
    for _ in range(3000):
        views = []
        for _ in range(2):
            shape = [rng.choice([1, 1, 2, 3, 4, 5]) for _ in range(4)]
            stride = [rng.choice([0, 1, 2, 3, 4, 6, 8, 12, 24, 48, 96]) for _ in range(4)]
            x = base.view(rng.choice([torch.int16, torch.int32])) if rng.random() < 0.5 else base
            views.append(x.as_strided(shape, stride, rng.randrange(300)))
        a, b = (_bytes(x) for x in views)
        want = bool(set(a) & set(b))
        assert _validate.share_elements(*views) == want and _validate.share_elements(*views[::-1]) == want
        assert _validate.shares_with_itself(views[0]) == (len(set(a)) < len(a))
        seen[want] += 1
    assert min(seen.values()) > 300


def test_slices_of_one_projection():
    fused = torch.zeros(3, 1000, 48 * 128 + 8, dtype=torch.bfloat16)
    q, k, v = (fused[..., a * 128:b * 128].unflatten(-1, (-1, 128)) for a, b in ((0, 32), (32, 40), (40, 48)))
    for a, b in itertools.combinations((q, k, v), 2):
        assert not _validate.share_elements(a, b)
    assert not any(_validate.shares_with_itself(x) for x in (q, k, v, q.transpose(1, 2)))
    assert _validate.share_elements(q, fused[..., 31 * 128 + 127:].as_strided(k.shape, k.stride(), 31 * 128 + 127))
    # heads of q and k by turns
    pairs = torch.zeros(3, 100, 8, 2, 64)
    assert not _validate.share_elements(pairs[..., 0, :], pairs[..., 1, :])
    assert _validate.share_elements(pairs[..., 0, :], pairs[:, 99:, 7:, 0])
    assert not _validate.share_elements(pairs[:2], pairs[2:]) and not _validate.share_elements(pairs[:0], pairs)


@pytest.mark.parametrize("size,stride,shared", [((4, 5), (5, 1), False), ((4, 5), (4, 1), True), ((4, 5), (0, 1), True), ((1, 5), (0, 1), False),
                                                ((2, 2), (3, 2), False), ((3, 3), (3, 2), False), ((3, 4), (3, 2), True), ((3, 4, 2), (8, 2, 1), False)])
def test_one_tensor(size, stride, shared):
    assert _validate.shares_with_itself(torch.zeros(100).as_strided(size, stride)) == shared


def test_heads_in_place_against_all_addresses():
    """What is refused of random pairs of [B, T, H, D] views is what shares an element."""

    rng = random.Random(1)
    base = torch.zeros(3000, dtype=torch.int16)
    apart = torch.zeros(4)
    seen = {True: 0, False: 0}
    for _ in range(4000):
        batch, time, dim = rng.choice([1, 2, 3]), rng.choice([1, 2, 4]), rng.choice([1, 2, 4])
        heads = [rng.choice([1, 2, 3]) for _ in range(2)]
        if rng.random() < 0.7:       # slices of one projection, cut at places that need not be right
            row = max(1, rng.choice([sum(heads) * dim, sum(heads) * dim + rng.randrange(-3, 8)]))
            strides = [(rng.choice([time * row, time * row + 3, max(1, time * row - 2)]), row, dim, 1)] * 2
            at = [0, rng.choice([heads[0] * dim, heads[0] * dim + rng.randrange(-2, 3)])]
        else:
            strides = [tuple(rng.choice([0, 1, 2, 4, 8, 16, 48]) for _ in range(4)) for _ in range(2)]
            at = [0, rng.randrange(200)]
        if rng.random() < 0.5:
            at.reverse()
        views = [base.as_strided((batch, time, h, dim), s, max(0, x)) for h, s, x in zip(heads, strides, at)]
        places = [_bytes(x) for x in views]
        want = len(set(places[0] + places[1])) < len(places[0]) + len(places[1])
        if want:
            with pytest.raises(ValueError, match="places of their own"):
                _validate.heads_in_place(*views, (apart, apart, None))
        else:
            _validate.heads_in_place(*views, (apart, apart, None))
            inside = base[views[1].storage_offset():views[1].storage_offset() + 1]
            with pytest.raises(ValueError, match="do not lie in"):
                _validate.heads_in_place(*views, (apart, inside, None))
        seen[want] += 1
    assert min(seen.values()) > 500
