"""Batches of the paged 8-bit attention in which requests that see nothing stand between others, against the row-by-row
definition (tests/kv8_ref.py) within the bounds of tests/test_kv8_gpu.py."""
import random

import pytest

from test_kv8_gpu import Batch, T, ref  # noqa: F401  (T and ref are fixtures)

pytestmark = pytest.mark.gpu

# 4 query heads per KV head: more than 12 new tokens are more than 48 rows. 30 rows are one group of 120, seen by nobody;
# with an odd number of KV heads an odd number of such units follow one another.
KINDS = [(1, 64, 0), (1, 128, 1), (1, 128, 0), (1, 256, 2), (5, 64, 1), (5, 128, 0), (5, 128, 2), (3, 256, 1)]


@pytest.mark.parametrize("hkv,hd,type", KINDS)
@pytest.mark.parametrize("fmt", [0, 1])
def test_prompts_not_placed_between_prompts(fb, T, ref, hkv, hd, type, fmt):  # noqa: F811
    """Short prompts, every other one not placed: a CTA's run of tiles crosses several units without tiles."""
    rng = random.Random(hkv * hd + type)
    lens = []
    for _ in range(300 // hkv):
        n = rng.choice([30, 32, 64])
        lens.append((rng.randint(n, 400), n))
        lens.append((0, 30))
    Batch(fb, T, lens, 4 * hkv, hkv, hd, 64, fmt, type).check(ref)


@pytest.mark.parametrize("hkv,hd,type", KINDS)
def test_long_prompts_with_gaps_of_every_length(fb, T, ref, hkv, hd, type):  # noqa: F811
    """Units of many tiles with none, one, two or three requests that were not placed between them, decode rows among them."""
    rng = random.Random(7 * hkv + hd)
    lens = []
    for i in range(28 // hkv):
        lens.append((rng.randint(1500, 4000), rng.choice([60, 130, 256])))
        lens += [(0, rng.choice([30, 60, 70])) for _ in range(i % 4)] + [(rng.randint(1, 300), 1)]
    Batch(fb, T, lens, 4 * hkv, hkv, hd, 32, 0, type).check(ref)


@pytest.mark.parametrize("hkv,hd,type", KINDS)
def test_rows_before_the_first_position(fb, T, ref, hkv, hd, type):  # noqa: F811
    """More rows than positions: the first groups of rows of a request see nothing, the later ones do."""
    lens = []
    for i in range(120 // hkv):
        lens += [(50 + i % 7, 120 + i % 5), (60, 60), (40, 200)]
    Batch(fb, T, lens, 4 * hkv, hkv, hd, 16, 1, type).check(ref)


@pytest.mark.parametrize("n", [1, 5, 60])
@pytest.mark.parametrize("type", [0, 2])
def test_windows_longer_than_any_request(fb, T, ref, n, type):  # noqa: F811
    """Up to the largest int the window hides nothing, with requests that are not placed or have more rows than positions."""
    b = Batch(fb, T, [(500, n), (0, n + 2), (max(1, n - 3), n), (40, 200 if n == 60 else n)], 8, 2, 128, 16, 0, type)
    b.check(ref)
    want = [x.clone() for x in b.run()]
    for window in (2 ** 31 - 1, 2 ** 31 - 64, 2 ** 30, 16 * b.max_pages, 16 * b.max_pages - 1):
        b.window = window
        for x in (b.out, b.lse):
            x.fill_(7)
        got = b.run()
        assert T.equal(got[0], want[0]) and T.equal(got[1], want[1])


@pytest.mark.parametrize("n", [1, 5, 60, 300])
@pytest.mark.parametrize("hd,type", [(64, 0), (128, 1), (256, 2)])
@pytest.mark.parametrize("page", [16, 64])
def test_table_entries_before_the_window_are_not_used(fb, T, ref, n, hd, type, page):  # noqa: F811
    """Pages that the window has left behind may be given away: their entries in the table hold no page."""
    b = Batch(fb, T, [(900, n), (500, n)], 8, 2, hd, page, 0, type, window=70)
    want = [x.clone() for x in b.run()]
    for r, (kv, m) in enumerate(b.lens):
        b.d_table[r, :max(0, kv - m + 1 - 70) // page] = -1
    got = b.run()
    assert fb.lib().fence_device_error() == 0
    assert T.equal(got[0], want[0]) and T.equal(got[1], want[1])
