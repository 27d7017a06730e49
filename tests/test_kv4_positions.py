"""Every position counts, once, in every way through the attention over the 4-bit cache: queries that look at one position each, all positions
in turn; and plain averages of values that rise with the position, which show a piece that is lost or taken twice."""
import numpy as np
import pytest

import ternary_llm_amd as tl
from tests import kv4_plain as plain
from tests.test_kv4 import HALF_STEP, TINY, torch_, up, upload  # noqa: F401
from tests.test_kv4_precision import check_exact, run, set_scales

WAYS = [
    # length, batch, rows, heads, kv heads, dim, page, bound of the lengths (0: the length)
    (5000, 32, 1, 4, 1, 128, 64, 0),      # 4 rows, in line
    (4300, 32, 1, 8, 2, 64, 16, 0),
    (1030, 40, 1, 4, 1, 128, 32, 0),      # ... alone
    (517, 16, 1, 3, 1, 64, 16, 0),
    (4100, 16, 2, 4, 1, 128, 16, 0),      # 8 rows
    (900, 16, 1, 8, 1, 64, 64, 0),
    (5000, 8, 5, 4, 1, 128, 32, 0),       # 20 rows: tiles of 32, in line
    (700, 16, 11, 2, 1, 64, 16, 0),       # ... alone
    (4500, 6, 16, 4, 1, 128, 64, 0),      # 64 rows: two tiles
    (3000, 2, 90, 1, 1, 128, 16, 0),      # prompts, in line
    (700, 2, 333, 1, 1, 64, 256, 0),
    (1500, 1, 1500, 1, 1, 128, 64, 1 << 15),
    (600, 3, 200, 2, 1, 128, 32, 0),      # ... alone
]


def one_page_table(rng, length, page, kv, dim):
    """A cache of one sequence's pages in random order (garbage behind its end), and its table."""
    n = -(-length // page)
    cache = plain.Cache(n + 1, page, kv, dim, rng)
    return cache, rng.permutation(n + 1)[:n].astype(np.int32)


def fill(cache, table, length, which, codes, step, low):
    """Positions 0..length-1 of all heads: codes [length, heads, dim], step and minimum [length, heads, groups]."""
    t = np.arange(length)
    page, slot = table[t // cache.page], t % cache.page
    words = np.zeros(codes.shape[:2] + (cache.dim // 8,), np.uint32)
    for d in range(cache.dim):
        at, shift = plain.k_word_of(d, cache.dim) if which == "k" else (d // 8, 4 * (d % 8))
        words[:, :, at] |= codes[:, :, d].astype(np.uint32) << np.uint32(shift)
    if which == "k":
        cache.kc[page, :, slot] = words
    else:
        cache.vc[page, :, slot // 4, :, slot % 4] = words
    s = cache.ks if which == "k" else cache.vs
    both = np.stack([step, low], -1).astype(np.float16).view(np.uint16)   # [length, heads, groups, 2]
    s[page, :, :, slot] = both


def case_of(way, seed):
    length, batch, rows, heads, kv, dim, page, bound = way
    rng = np.random.default_rng(seed)
    cache, table = one_page_table(rng, length, page, kv, dim)
    signs = rng.integers(0, 2, (length, kv, dim))
    groups = (length, kv, dim // 32)
    fill(cache, table, length, "k", signs * 15, np.full(groups, 1.0), np.full(groups, -7.5))   # +-7.5
    step = rng.uniform(0.05, 0.3, groups)
    codes = rng.integers(0, 16, (length, kv, dim))
    fill(cache, table, length, "v", codes, step, -7.5 * step)
    # the sequences of the batch share the pages and end at different positions
    lens = length - (np.arange(batch) * 37) % max(1, min(length - rows, 300))
    starts = np.arange(batch + 1) * rows
    return rng, cache, table, 2 * signs - 1, starts.astype(np.int32), lens.astype(np.int32)


@pytest.mark.gpu
@pytest.mark.parametrize("way", WAYS, ids=range(len(WAYS)))
def test_every_position_in_turn(torch_, way):
    """A query of a position's own signs sees that position and, e^-40 of it, the others: the result is its value. Positions are
    taken in turn until each was looked at."""
    torch = torch_
    length, batch, rows, heads, kv, dim, page, bound = way
    rng, cache, table, signs, starts, lens = case_of(way, length + dim)
    dev, share = upload(torch, cache), heads // kv
    args = (up(torch, starts), up(torch, lens), up(torch, np.tile(table, (batch, 1))))
    values = np.stack([cache.sequence("v", table, length, h)[0] for h in range(kv)], 1)         # [length, kv, dim]
    s = cache.vs[table[np.arange(length) // page], :, :, np.arange(length) % page].view(np.float16).astype(np.float64)
    size = np.repeat(np.abs(s[..., 1]) + 15 * s[..., 0], 32, -1)
    overlap = max(int((np.einsum("td,ud->tu", signs[:, h], signs[:, h]) - 2 * dim * np.eye(length, dtype=int)).max()) for h in range(kv))
    beta = 2.0 ** np.ceil(np.log2(40.0 / (7.5 * dim ** -0.5 * (dim - overlap))))
    pos = (lens[:, None] - rows + np.arange(rows)).reshape(-1)                                # of each row
    few = rows * share <= 8
    left = [set(range(length)) for _ in range(kv)]
    for call in range(80):
        target = np.zeros((batch * rows, heads), int)
        for r in rng.permutation(batch * rows):
            for h in range(heads):
                open_ = left[h // share]
                best = max((t for t in open_ if t <= pos[r]), default=None) if call % 2 else next((t for t in open_ if t <= pos[r]), None)
                target[r, h] = rng.integers(0, pos[r] + 1) if best is None else best
                open_.discard(target[r, h])
        h = np.arange(heads) // share
        q = (signs[target, h] * beta).astype(np.float16)
        got = run(torch, q, dev, args, rows, bound or length).astype(np.float64)
        want = values[target, h]
        allowed = HALF_STEP * np.abs(want) * (1 if few else 2) + 2 * TINY + 2.0 ** -16 * size[target, h]
        wrong = np.abs(got - want) > allowed
        assert not wrong.any(), (call, np.argwhere(wrong)[:3].tolist(), target[wrong.any(-1)][:8].tolist())
        if not any(left):
            break
    assert not any(left)
    # another position in its place would show
    a, b = rng.integers(0, length, (2, 2000))
    other = a != b
    assert (np.abs(values[a] - values[b]) > 2.0 ** -9 * size[a]).any(-1)[other].all()


@pytest.mark.gpu
@pytest.mark.parametrize("way", WAYS, ids=range(len(WAYS)))
def test_averages_of_rising_values(torch_, way):
    """Queries of zero: the mean of what a row sees. Values rise with the position, so that a step's positions more or less move it."""
    torch = torch_
    length, batch, rows, heads, kv, dim, page, bound = way
    rng, cache, table, signs, starts, lens = case_of(way, length)
    t = np.arange(length)[:, None, None]
    groups = (length, kv, dim // 32)
    low = np.broadcast_to(8.0 * t / length, groups)
    fill(cache, table, length, "v", rng.integers(0, 16, (length, kv, dim)), np.full(groups, 0.125), low)
    dev = upload(torch, cache)
    args = (up(torch, starts), up(torch, lens), up(torch, np.tile(table, (batch, 1))))
    q = np.zeros((batch * rows, heads, dim), np.float16)
    got = run(torch, q, dev, args, rows, bound or length)
    values = np.stack([cache.sequence("v", table, length, h)[0] for h in range(kv)], 1)
    upto = (lens[:, None] - rows + np.arange(rows)).reshape(-1) + 1
    mean = np.cumsum(values, 0)[upto - 1] / upto[:, None, None]
    want = np.repeat(mean, heads // kv, 1)
    # half a step of the result; from 9 rows on half a step of each value; fp32 sums of up to 2^12 in one accumulator: 2^-16 of 10
    allowed = HALF_STEP * np.abs(want) * (1 if rows * heads // kv <= 8 else 2) + 10 * 2.0 ** -16
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= allowed).all(), float((err / allowed).max())
    # 16 positions more or less at an end would show
    assert (16 / length * np.abs(values[:16].mean(0) - mean[-1]) > 2 * allowed.max()).any() or length > 2000


@pytest.mark.gpu
@pytest.mark.parametrize("way", [w for w in WAYS if w[2] * w[3] // w[4] <= 8], ids=str)
def test_few_rows_to_the_last_bits(torch_, way):
    """Up to 8 rows with scores of some units, against the bound that knows of no rounding of k, v and p."""
    torch = torch_
    length, batch, rows, heads, kv, dim, page, bound = way
    batch = min(batch, 6)
    rng, cache, table, signs, starts, lens = case_of((length, batch) + way[2:], length + 7)
    low = rng.uniform(-2.0, 0.5, cache.ks.shape[:-1])
    set_scales(cache.ks, rng.uniform(0.05, 0.2, low.shape), low)
    q = rng.standard_normal((batch * rows, heads, dim)).astype(np.float16)
    dev, tables = upload(torch, cache), np.tile(table, (batch, 1))
    got = run(torch, q, dev, (up(torch, starts), up(torch, lens), up(torch, tables)), rows, bound or length)
    check_exact(got, cache, q, starts, lens, tables, dim ** -0.5)
