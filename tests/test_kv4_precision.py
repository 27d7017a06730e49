"""How exact the attention over the 4-bit cache is where values are small, large or of very different sizes."""
import numpy as np
import pytest

import ternary_llm_amd as tl
from tests import kv4_plain as plain
from tests.test_kv4 import check_attention, torch_, up  # noqa: F401
from tests.test_kv4_serving import on_device, random_batch

pytestmark = pytest.mark.gpu


def run(torch, q, dev, batch, max_query, max_length, **how):
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
    tl.attention_kv4(up(torch, q), out, *dev, *batch, max_query, max_length, **how)
    return out.cpu().numpy()


def set_scales(held, step, low):
    """Steps and minima (float64 [pages, heads, groups, page], or what broadcasts to it)."""
    held[..., 0] = np.broadcast_to(step, held.shape[:-1]).astype(np.float16).view(np.uint16)
    held[..., 1] = np.broadcast_to(low, held.shape[:-1]).astype(np.float16).view(np.uint16)


@pytest.mark.parametrize("size", [1e-2, 1e-3, 2e-4, 1e-4, 1e-5, 1e-6, 1e-7])
@pytest.mark.parametrize("rows,heads,bound", [(1, 4, 150), (2, 4, 5000), (3, 4, 150), (16, 4, 5000), (80, 1, 150), (80, 2, 5000)])
def test_small_values(torch_, size, rows, heads, bound):
    """Steps and minima down to fp16's smallest: the values are those of the cache with one rounding (half a step of a subnormal is
    2^-25), in every kernel. Rows that see one position show a single value."""
    torch = torch_
    rng = np.random.default_rng(rows + heads + bound)
    for dim in (64, 128):
        cache, starts, lens, table = random_batch(rng, [rows, 150], [rows, rows], 16, 1, dim)
        step = size * rng.uniform(0.1, 0.5, cache.vs.shape[:-1])
        set_scales(cache.vs, step, -step * rng.uniform(3, 12, step.shape))
        q = rng.standard_normal((2 * rows, heads, dim)).astype(np.float16)
        dev, batch = on_device(torch, cache, starts, lens, table)
        want, spread, reach = plain.attend(cache, q, starts, lens, table, dim ** -0.5, 0)
        check_attention(run(torch, q, dev, batch, rows, bound), want, spread, reach, q)


@pytest.mark.parametrize("rows,heads,bound", [(3, 4, 150), (16, 4, 5000), (80, 1, 150), (80, 2, 5000)])
def test_values_at_the_end_of_fp16(torch_, rows, heads, bound):
    """m + 15 s may be half a step of s above 65504: kept there (up to 60 less, within two half steps of fp16), beside groups that
    are small and groups that are not finite."""
    torch = torch_
    rng = np.random.default_rng(rows + heads)
    for dim in (64, 128):
        cache, starts, lens, table = random_batch(rng, [rows + 1, 90], [rows, rows], 16, 1, dim)
        step = np.where(rng.integers(0, 4, cache.vs.shape[:-1]) > 0, rng.uniform(0.1, 0.5, cache.vs.shape[:-1]), 8736.0)
        set_scales(cache.vs, step, np.where(step > 1, -65504.0, -7 * step))     # -65504 + 15 * 8736 = 65536
        keys = np.where(rng.integers(0, 4, cache.ks.shape[:-1]) > 0, 0.25, 8736.0)
        set_scales(cache.ks, keys, np.where(keys > 1, -65504.0, -7 * keys))
        cache.vc[...] |= np.where(rng.integers(0, 2, cache.vc.shape), np.uint32(0xFFFFFFFF), np.uint32(0)).astype(np.uint32)
        cache.kc[...] |= np.where(rng.integers(0, 2, cache.kc.shape), np.uint32(0xFFFFFFFF), np.uint32(0)).astype(np.uint32)
        q = (rng.standard_normal((2 * rows, heads, dim)) * 2.0 ** -14).astype(np.float16)
        cache.vs[table[0, 0], 0, 0, 1] = 0x7E00   # position 1 of the first sequence: a value's first group
        dev, batch = on_device(torch, cache, starts, lens, table)
        with np.errstate(invalid="ignore"):
            want, spread, reach = plain.attend(cache, q, starts, lens, table, dim ** -0.5, 0)
        got = run(torch, q, dev, batch, rows, bound)
        np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
        bad = np.isnan(want)
        check_attention(np.where(bad, 0, got), np.where(bad, 0, want), np.where(bad, 0, spread), reach, q)


# ---------------------------------------------------------------------------------------------------------------- up to 8 rows
#
# A bound that knows what these rows are not rounded by. Of the result: half a step of fp16. Of the products p s, in two fp16 pieces: 2^-22
# of each, or 2^-29 of the largest of the row and group, for each of n positions, times codes of 15 at most. Of fp32 sums of p m and p s c: 2^-16
# of the sum of their sizes (2^8 of them after each other in one accumulator). Of the scores: sums of fp32 products, 2^-19 of scale sum |q| (|m| + 15 s),
# which p is off by twice, relative.
def held_sizes(cache, which, table, count, head):
    """(step, |minimum|) float64 [count, groups] of positions 0..count-1."""
    s = cache.ks if which == "k" else cache.vs
    t = np.arange(count)
    both = s[table[t // cache.page], head, :, t % cache.page].view(np.float16).astype(np.float64)
    return both[..., 0], np.abs(both[..., 1])


def exact_bound(cache, q, starts, lens, table, scale, want):
    bound = np.full(want.shape, np.inf)
    x, heads, kv = np.abs(q.astype(np.float64)), q.shape[1], cache.kc.shape[1]
    for b in range(len(lens)):
        for h in range(kv):
            n = int(lens[b])
            ks, km = held_sizes(cache, "k", table[b], n, h)
            vs, vm = held_sizes(cache, "v", table[b], n, h)
            keys, _ = cache.sequence("k", table[b], n, h)
            for r in range(starts[b], starts[b + 1]):
                upto = n - (starts[b + 1] - 1 - r)
                for head in range(h * heads // kv, (h + 1) * heads // kv):
                    score = keys[:upto] @ q[r, head].astype(np.float64) * scale
                    p = np.exp(score - score.max())
                    p /= p.sum()
                    reach = (np.repeat(km[:upto] + 15 * ks[:upto], 32, 1) @ x[r, head]).max() * abs(scale)
                    size = p @ (vm[:upto] + 15 * vs[:upto])
                    largest = (p[:, None] * vs[:upto]).max(0)
                    group = size * (2.0 ** -16 + 2.0 ** -22 + 2 * 2.0 ** -19 * reach) + 15 * upto * 2.0 ** -29 * largest
                    bound[r, head] = 2.0 ** -11 * np.abs(want[r, head]) + 2.0 ** -25 + np.repeat(group, 32)
    return bound


def check_exact(got, cache, q, starts, lens, table, scale):
    want, _, _ = plain.attend(cache, q, starts, lens, table, scale, 0)
    err, bound = np.abs(got.astype(np.float64) - want), exact_bound(cache, q, starts, lens, table, scale, want)
    assert np.isfinite(got).all()
    assert (err <= bound).all(), (float((err / bound).max()), float((err - bound).max()))


FEW = [(1, 4, 1), (1, 3, 1), (2, 4, 1), (1, 8, 1), (3, 4, 2), (4, 1, 1)]   # rows, heads, kv heads: up to 8 rows of a kv head


@pytest.mark.parametrize("rows,heads,kv", FEW)
@pytest.mark.parametrize("dim,bound", [(128, 300), (128, 5000), (64, 300), (64, 5000)])
@pytest.mark.parametrize("how", ["alike", "groups", "positions", "any", "falling", "rising", "zeros"])
def test_steps_of_different_sizes(torch_, how, dim, bound, rows, heads, kv):
    """Steps of values of any sizes beside each other: in the groups of a position, from position to position (a large one that hardly counts
    beside small ones that do), for rows that look at different positions, and with the scores that fall or rise."""
    torch = torch_
    rng = np.random.default_rng(dim + rows + heads + len(how))
    page, lengths = 16, [bound if bound < 1000 else 1111, 70, rows]
    cache, starts, lens, table = random_batch(rng, lengths, [rows] * 3, page, kv, dim)
    shape = cache.vs.shape[:-1]
    step = rng.uniform(0.1, 0.3, shape)
    if how == "groups":
        step = step * (2.0 ** np.array([14, -14, 0, -18]))[None, None, :dim // 32, None]
    elif how in ("positions", "any"):
        step = 2.0 ** rng.uniform(-20, 12, shape if how == "any" else shape[:2] + (1,) + shape[3:])
    elif how in ("falling", "rising"):   # with the position: sizes from 2^12 to 2^-12
        for b, n in enumerate(lengths):
            t = np.arange(n)
            power = np.linspace(12, -12, n)[::1 if how == "falling" else -1]
            step[table[b, t // page], :, :, t % page] = (2.0 ** power)[:, None, None]
    elif how == "zeros":
        step = np.where(rng.integers(0, 3, shape) > 0, step, 0.0)
    step = np.minimum(step, 4000.0)   # (m and m + 15 s are fp16 numbers)
    set_scales(cache.vs, step, -step * rng.choice([0.0, 7.0, 15.0], shape))
    # keys: rows prefer positions far apart, so that most of a row's positions hardly count
    low = rng.choice([0.0, -0.3], cache.ks.shape[:-1])
    set_scales(cache.ks, np.full(low.shape, 0.04), low)
    q = (rng.standard_normal((3 * rows, heads, dim)) * rng.choice([1.0, 8.0, 30.0], (3 * rows, heads, 1))).astype(np.float16)
    dev, batch = on_device(torch, cache, starts, lens, table)
    check_exact(run(torch, q, dev, batch, rows, bound), cache, q, starts, lens, table, dim ** -0.5)


@pytest.mark.parametrize("rows,heads,kv", FEW[:4])
@pytest.mark.parametrize("power", [-15, -11, -7, 5])
@pytest.mark.parametrize("dim,bound", [(128, 300), (64, 5000)])
def test_small_queries_and_large_keys(torch_, dim, bound, power, rows, heads, kv):
    """Scores of some units from queries of 2^-15 and keys of 2^15, and the other way round; rows of very different sizes in a tile."""
    torch = torch_
    rng = np.random.default_rng(dim + rows + heads + power)
    lengths = [300, 70]
    cache, starts, lens, table = random_batch(rng, lengths, [rows] * 2, 16, kv, dim)
    step = 2.0 ** (-power - 4) * rng.uniform(0.5, 1.0, cache.ks.shape[:-1])
    set_scales(cache.ks, step, -step * rng.choice([0.0, 7.5, 15.0], step.shape))
    q = rng.standard_normal((2 * rows, heads, dim)) * 2.0 ** power
    q[:, 0] *= 2.0 ** -6
    q = q.astype(np.float16)
    dev, batch = on_device(torch, cache, starts, lens, table)
    check_exact(run(torch, q, dev, batch, rows, bound), cache, q, starts, lens, table, dim ** -0.5)
