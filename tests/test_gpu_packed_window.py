"""attention.packed_attention on windowed layers whose pages behind the window have left the block table: entries that no row
reaches are not looked at, wherever the window starts, and nothing of the page read in their place gets into a result."""
import pytest
import torch

from nanochat_amd.attention import decode_attention, packed_attention

from .test_gpu_packed_attention import PAGE, check, reference, setup

pytestmark = pytest.mark.gpu


def poison(cache, page):
    """A page whose every code and scale is NaN."""
    cache.k_pages[page] = cache.v_pages[page] = 0x7F
    cache.kv_scale[page] = float("nan")


def first_keys(n, ctx, window):
    return [max(ctx + t - window, 0) for t in range(n)]


def drop(table, b, first):
    """The table as a server keeps it once the pages below position `first` of sequence b are given back."""
    table[b, :first // PAGE] = -1


def without_page_zero(table, cache):
    """Page 0 swapped out of every row of the table (for one that is nobody's), so that it can hold anything."""
    used = set(table.flatten().tolist())
    spare = next(p for p in range(cache.num_pages) if p not in used)
    for t in (cache.k_pages, cache.v_pages, cache.kv_scale):
        t[spare] = t[0].clone()
    table[table == 0] = spare


@pytest.mark.parametrize("n", [1, 5, 16, 17, 40, 150, 600])
@pytest.mark.parametrize("window", [0, 7, 15, 16, 100, 2900])
def test_pages_behind_the_window(device, n, window):
    """Narrow, alone and wide items, cut and uncut, at windows that start anywhere in even and odd pages."""
    for ctx in (4000, 4007, 4016, 4021, window + 3):
        q, cache, table, cu, lens, cu_l, lens_l = setup(device, [n], [ctx], 4, 2, seed=n + ctx, spare=2)
        without_page_zero(table, cache)
        want, size = reference(q, cache, table, cu_l, lens_l, window)
        drop(table, 0, first_keys(n, ctx, window)[0])
        poison(cache, 0)
        got = packed_attention(q, cache, table, cu, lens, lens_l[0], window)
        check(got, want, size, cu_l)
        if n == 1:
            assert not bool(torch.isnan(decode_attention(q, cache, table, lens, lens_l[0], window=window)).any())


@pytest.mark.parametrize("window", [5, 31, 40, 200])
def test_an_entry_that_some_rows_reach(device, window):
    """A wide sequence, and pages at its window's start missing: NaN for the rows that reach them; right for every row of a
    wave (16 rows of two heads) none of whose rows does."""
    n, ctx, wave = 600, 3000, 16
    q, cache, table, cu, lens, cu_l, lens_l = setup(device, [n], [ctx], 4, 2, seed=window, spare=2)
    without_page_zero(table, cache)
    want, size = reference(q, cache, table, cu_l, lens_l, window)
    lows = first_keys(n, ctx, window)
    for missing in (lows[0] // PAGE, lows[0] // PAGE + 1, lows[300] // PAGE):
        bad = table.clone()
        bad[0, missing] = -1
        poison(cache, 0)
        got = packed_attention(q, cache, bad, cu, lens, lens_l[0], window)
        reach = [lo // PAGE <= missing <= (ctx + t) // PAGE for t, lo in enumerate(lows)]
        assert any(reach)
        for t0 in range(0, n, wave):
            rows = slice(t0, min(t0 + wave, n))
            if not any(reach[rows]):
                check(got[rows], want[rows], size[rows], [0, rows.stop - rows.start])
        assert bool(torch.isnan(got[torch.tensor(reach)]).all())


def test_a_batch_behind_its_windows(device):
    new, ctx, window = [1, 3, 0, 70, 1, 200], [2500, 777, 100, 1234, 40, 0], 333
    q, cache, table, cu, lens, cu_l, lens_l = setup(device, new, ctx, 8, 2, seed=3, spare=2)
    without_page_zero(table, cache)
    want, size = reference(q, cache, table, cu_l, lens_l, window)
    for b, (n, c) in enumerate(zip(new, ctx)):
        drop(table, b, max(c - window, 0))
    poison(cache, 0)
    check(packed_attention(q, cache, table, cu, lens, max(lens_l), window), want, size, cu_l)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5])
def test_a_window_past_every_position_hides_nothing(device, window):
    q, cache, table, cu, lens, _, lens_l = setup(device, [1, 60], [3000, 200], 4, 2, seed=4)
    assert torch.equal(packed_attention(q, cache, table, cu, lens, max(lens_l), window),
                       packed_attention(q, cache, table, cu, lens, max(lens_l)))
