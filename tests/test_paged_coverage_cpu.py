"""The decisive rows of tests/paged_coverage.py are decisive: one position lost or counted twice, or a tile in another's
place, is beyond the tolerance over the range of lengths that the GPU tests use them at (the change falls with the length)."""
import numpy as np
import pytest

from tests import paged_coverage as cover

LENGTHS = [2, 17, 64, 129, 777, 2000, 5000, 7000, 12000, 16003, 20011]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", LENGTHS)
@pytest.mark.parametrize("layout", ["stripes", "random"])
def test_every_single_position_counts(n, hd, layout):
    classes = cover.value_classes(n, 1, hd, layout, n)
    want = cover.even(classes, np.ones(n), hd)
    assert cover.off(want.astype(np.float16).astype(np.float64), want, cover.EVEN) <= 1  # a right answer passes
    sizes = np.bincount(classes[:, 0], minlength=hd)
    for change in (-1, 1):
        for size in np.unique(sizes[sizes > 0]):  # positions of equally large classes are alike
            p = np.nonzero(sizes[classes[:, 0]] == size)[0][0]
            counts = np.ones(n)
            counts[p] += change
            got = cover.even(classes, counts, hd).astype(np.float16).astype(np.float64)
            assert cover.off(got, want, cover.EVEN) > 1, (change, size)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [n for n in LENGTHS if n >= 256])
def test_a_tile_in_another_ones_place_counts(n, hd):
    classes = cover.value_classes(n, 1, hd, "random", n)
    want = cover.even(classes, np.ones(n), hd)
    for tile in (16, 64):
        for i in range(0, n - 2 * tile + 1, tile):
            counts = np.ones(n)
            counts[i : i + tile] += 1
            counts[i + tile : i + 2 * tile] -= 1
            assert cover.off(cover.even(classes, counts, hd).astype(np.float16).astype(np.float64), want, cover.EVEN) > 1, (tile, i)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", LENGTHS)
def test_chosen_positions_count(n, hd):
    """Of the positions of a key class, each one lost or counted twice; and two positions' values exchanged."""
    classes, keys = cover.value_classes(n, 1, hd, "random", n), cover.key_classes(n, 1, hd)
    step = max(1, n // 40)
    for p in range(0, n, step):
        wanted = [keys[p, 0]]
        want = cover.chosen(classes, keys, np.ones(n), hd, wanted)
        assert cover.off(want.astype(np.float16).astype(np.float64), want, cover.CHOSEN) <= 1
        alone = (keys == keys[p]).sum() == 1
        for change in (-1, 1):
            counts = np.ones(n)
            counts[p] += change
            got = cover.chosen(classes, keys, counts, hd, wanted).astype(np.float16).astype(np.float64)
            # (twice the only one of its class leaves it with all the weight)
            assert (alone and change == 1) or cover.off(got, want, cover.CHOSEN) > 1, (p, change)
        if p + 1 < n and classes[p, 0] != classes[p + 1, 0]:
            other = classes.copy()
            other[[p, p + 1]] = other[[p + 1, p]]
            got = cover.chosen(other, keys, np.ones(n), hd, wanted).astype(np.float16).astype(np.float64)
            assert cover.off(got, want, cover.CHOSEN) > 1, p
