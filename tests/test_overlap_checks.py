"""The overlap checks of the in-place and strided outputs against the sets of elements
themselves, on small layouts: what they accept shares no element.  No GPU."""

from __future__ import annotations

import itertools
import random

import torch


def _elements(t):
    offsets = [t.storage_offset()]
    for n, stride in zip(t.shape, t.stride()):
        offsets = [o + i * stride for o, i in itertools.product(offsets, range(n))]
    return offsets



def _apart(a, b):
    return not set(_elements(a)) & set(_elements(b))


def test_interleaved_slices_of_unequal_batch_and_token_spacing():
    """Batch entries that are no multiple of a token apart: the second part's rows of
    entry 0 reach into the first part's rows of entry 1."""
    from hilberta_b200.prep import _interleaved

    base = torch.empty(4096, dtype=torch.float16)
    for (a_shape, a_strides, a_at), (b_shape, b_strides, b_at) in (
            (((2, 2, 1, 2), (100, 8, 4, 1), 44), ((2, 2, 3, 2), (100, 8, 2, 1), 142)),
            (((3, 1, 2, 2), (72, 32, 2, 1), 88), ((3, 1, 1, 2), (72, 32, 2, 1), 16))):
        a, b = base.as_strided(a_shape, a_strides, a_at), base.as_strided(b_shape, b_strides, b_at)
        assert not _apart(a, b) and not _interleaved(a, b) and not _interleaved(b, a)


def test_interleaved_accepts_nothing_shared():
    from hilberta_b200.prep import _interleaved

    rng = random.Random(1)
    base = torch.empty(4096, dtype=torch.float16)
    accepted = 0
    for _ in range(20000):
        shape = rng.randint(1, 3), rng.randint(1, 4)
        strides = rng.choice([8, 16, 24, 32, 40, 48, 64, 72, 100]), rng.choice([8, 16, 24, 32])
        a, b = (base.as_strided((*shape, rng.randint(1, 3), 2), (*strides, rng.choice([2, 4]), 1), 2 * rng.randint(0, 80))
                for _ in range(2))
        if _interleaved(a, b):
            accepted += 1
            assert _apart(a, b), (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
    assert accepted > 1000


def test_interleaved_accepts_parts_of_one_projection():
    from hilberta_b200.prep import _interleaved

    joint = torch.empty(2, 9, 3, 4, 32, dtype=torch.float16)
    q, k, v = joint.unbind(2)
    for a, b in itertools.permutations((q, k, v), 2):
        assert _interleaved(a, b) and _interleaved(a[:, 3:], b[:, 3:]) and _interleaved(a[:1], b[:1])
        assert _interleaved(a[:, :1], b[:, :1])
    assert not _interleaved(q, q) and not _interleaved(joint[:, :, 0, :3], joint[:, :, 0, 2:])
    padded = torch.empty(2, 9 * 96 + 40, dtype=torch.float16)  # entries further apart than their tokens
    a, b = (padded.as_strided((2, 9, 1, 32), (9 * 96 + 40, 96, 32, 1), at) for at in (0, 64))
    assert _interleaved(a, b) and _interleaved(b, a)


def test_apart_and_self_overlap_accept_nothing_shared():
    from hilberta_b200.int8 import _apart as checked
    from hilberta_b200.int8 import _overlaps_itself

    rng = random.Random(2)
    base = torch.empty(4096, dtype=torch.float16)
    accepted = 0
    for _ in range(20000):
        n = rng.choice([2, 3])
        a, b = (base.as_strided([rng.randint(1, 3) for _ in range(n - 1)] + [rng.choice([1, 2, 4])],
                                [rng.choice([0, 4, 8, 12, 16, 20, 24, 36, 48]) for _ in range(n - 1)] + [1], rng.randint(0, 60))
                for _ in range(2))
        if rng.random() < 0.7:
            b = base.as_strided(b.shape, a.stride(), b.storage_offset())
        if checked(a, b):
            accepted += 1
            assert _apart(a, b), (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
        if not _overlaps_itself(a):
            assert len(set(_elements(a))) == a.numel()
    assert accepted > 1000


def test_norms_and_rotation_inside_an_in_place_output_are_refused():
    import pytest

    from hilberta_b200.prep import _check_qk_out

    joint = torch.zeros(1, 9, 3, 4, 64, dtype=torch.float16)
    q, k, v = joint.unbind(2)
    cos, sin, weight = torch.zeros(9, 64), torch.zeros(9, 64), torch.zeros(64, dtype=torch.float16)
    _check_qk_out(q, k, (q, k), [cos, sin, weight, weight])
    for bad in (q[0, 4, 1], k[0, 0, 0], q.view(torch.float32)[0, 1, 0]):  # rewritten while other rows read them
        with pytest.raises(ValueError, match="must not overlap"):
            _check_qk_out(q, k, (q, k), [cos, sin, bad, weight])
        with pytest.raises(ValueError, match="must not overlap"):
            _check_qk_out(q, k, (q, k), [cos, sin, weight, bad])


def test_parts_that_follow_each_other_in_every_batch_entry():
    """Queries and keys of [B, 3, S, H, D] or [B, 3, H, S, D] storage, in place."""
    from hilberta_b200.prep import _check_qk_out, _interleaved

    small = [torch.zeros(9, 32), torch.zeros(32, dtype=torch.float16)]
    blocks = torch.zeros(3, 3, 9, 4, 32, dtype=torch.float16)
    heads_first = torch.zeros(3, 3, 4, 9, 32, dtype=torch.float16).transpose(2, 3)
    for joint in (blocks, heads_first):
        q, k, v = joint.unbind(1)
        assert _interleaved(q, k) and _interleaved(k, q) and _interleaved(v, q) and not _interleaved(q, q)
        _check_qk_out(q, k, (q, k), small)
        _check_qk_out(q[:, :4], k[:, :4], (v[:, :4], k[:, :4]), small)
        assert not _interleaved(joint[:, 0, :6], joint[:, 0, 5:])
    q, k, v = blocks.unbind(1)
    _check_qk_out(q[:, :4], k[:, :4], (q[:, 4:8], v[:, :4]), small)


def test_one_tensor_for_both_outputs_is_refused():
    import pytest

    from hilberta_b200.prep import _check_qk_out

    small = [torch.zeros(9, 32), torch.zeros(32, dtype=torch.float16)]
    q, k, out = (torch.zeros(2, 9, 4, 32, dtype=torch.float16) for _ in range(3))
    for args in ((q, q, (q, q)), (q, k, (out, out)), (q, k, (q, q)), (q, k, (k, k)), (q, k, (k, q)), (q, q, (out, q)), (q, q, (q, out)),
                 (q, q.view(q.shape), (q, q.view(q.shape)))):
        with pytest.raises(ValueError, match="must not overlap"):
            _check_qk_out(*args, small)
    _check_qk_out(q, q, (out, k), small)
    _check_qk_out(q, k, (q, out), small)
    _check_qk_out(q, k, (out, k), small)
