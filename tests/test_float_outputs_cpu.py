"""CompressedCache.read_float's outputs, without a GPU: which pairs of tensors share an element's memory."""

import random

import pytest
import torch

from insitu_amd.cache import _overlaps


def _cells(x):
    """The element numbers of x in its storage."""
    at = torch.arange(x.untyped_storage().nbytes() // x.element_size())
    return set(at.as_strided(x.shape, x.stride(), x.storage_offset()).reshape(-1).tolist())


@pytest.mark.parametrize("make,bad", [
    (lambda z: (z[:30], z[15:]), True), (lambda z: (z[15:], z[:30]), True), (lambda z: (z[:30], z[:30]), True),
    (lambda z: (z[:30], z[30:]), False), (lambda z: (z[29:59], z[:30]), True), (lambda z: (z[30:], z[:30]), False),
    (lambda z: (z[::2], z[1::2]), False), (lambda z: (z[:40:2], z[2:42:2]), True), (lambda z: (z[:, :1], z[:, 1:2]), False),
    (lambda z: (z[:, :, :4], z[:, :, 4:]), False), (lambda z: (z[:, :, :4], z[:, :, 3:7]), True),
    (lambda z: (z[:3].transpose(0, 1), z[3:6].transpose(0, 1)), False), (lambda z: (z[:3].transpose(0, 1)[:, :3], z[:3]), True),
    (lambda z: (z[:0], z[:0]), False)])
def test_two_outputs_in_one_place(make, bad):
    x, y = make(torch.zeros(60, 3, 8))
    assert _overlaps(x, y) is _overlaps(y, x) is bad
    assert not bad or _cells(x) & _cells(y)


def test_half_an_element_apart():
    raw = torch.zeros(82, dtype=torch.uint8)
    x = raw[:80].view(torch.float32).view(5, 1, 4)
    y = raw[2:82].clone().view(torch.float32).view(5, 1, 4)
    assert not _overlaps(x, y)
    y = torch.frombuffer(memoryview(raw.numpy())[1:81], dtype=torch.uint8).view(torch.float16).view(10, 1, 4)
    assert _overlaps(raw[:80].view(torch.float16).view(10, 1, 4), y)


def test_no_pair_that_shares_an_element_passes():
    """Random slices of one tensor, dimensions turned: what passes is apart, what is contiguous and apart passes."""
    rng = random.Random(0)
    passed = refused = 0
    for _ in range(4000):
        z = torch.zeros([rng.randint(1, 6) for _ in range(3)] + [8])
        d = rng.choice([4, 8])
        shape = [rng.randint(1, n) for n in z.shape[:3]]
        step = [rng.choice([1, 1, 2]) for _ in shape]
        shape = [min(n, (m + s - 1) // s) for n, m, s in zip(shape, z.shape, step)]
        def view():
            idx = []
            for n, m, s in zip(shape, z.shape, step):
                lo = rng.randint(0, m - (n - 1) * s - 1)
                idx.append(slice(lo, lo + (n - 1) * s + 1, s))
            c = rng.randint(0, 8 - d)
            return z[tuple(idx)][..., c:c + d]
        x, y = view(), view()
        order = rng.sample(range(3), 3) + [3]
        x, y = x.permute(order), y.permute(order)
        if _overlaps(x, y):
            refused += 1
        else:
            passed += 1
            assert not _cells(x) & _cells(y)
    assert passed > 500 and refused > 500
