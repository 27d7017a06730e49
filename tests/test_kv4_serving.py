"""The 4-bit paged cache and its attention as a server uses them: every way through the attention's kernels (few rows, up to 64,
prompts; alone, in line, both in one batch), values that are not finite, cut bounds, captured steps, streams, workspaces, pages
behind 4 GiB, and rotary, append and attention together over the steps of a conversation."""
import numpy as np
import pytest

import ternary_llm_amd as tl
from tests import kv4_plain as plain
from tests.test_kv4 import HALF_STEP, batch_of, check_attention, rotary_bound, torch_, up, upload  # noqa: F401

pytestmark = pytest.mark.gpu


def random_batch(rng, lengths, rows, page, kv, dim, spare=2):
    """Sequences over pages in random order; any codes, steps of 0.05 to 0.3 and minima around -7.5 steps; garbage and NaN behind
    each sequence's end."""
    need = [-(-n // page) for n in lengths]
    cache = plain.Cache(sum(need) + spare, page, kv, dim, rng)
    table = np.full((len(lengths), max(need + [1])), -1, np.int32)
    order, used = rng.permutation(cache.n), 0
    for b, n in enumerate(need):
        table[b, :n] = order[used:used + n]
        used += n
        for j in range(n):
            upto = min(page, lengths[b] - j * page)
            for s in (cache.ks, cache.vs):
                at = s[table[b, j]]
                step = rng.uniform(0.05, 0.3, at[:, :, :upto, 0].shape)
                at[:, :, :upto, 0] = step.astype(np.float16).view(np.uint16)
                at[:, :, :upto, 1] = (step * rng.uniform(-9, -6, step.shape)).astype(np.float16).view(np.uint16)
    starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    return cache, starts, np.array(lengths, np.int32), table


def on_device(torch, cache, starts, lens, table):
    return upload(torch, cache), (up(torch, starts), up(torch, lens), up(torch, table))


WAYS = [
    # lengths, rows, page, heads, kv, dim, window
    ([5000], [1], 64, 4, 1, 128, 0),                            # 4 rows, in line
    ([2100, 1, 900], [1, 1, 1], 16, 3, 1, 64, 0),
    ([4100, 4100], [1, 1], 128, 2, 2, 128, 3000),
    ([3000, 40, 700], [1, 1, 1], 32, 8, 1, 128, 0),             # 8 rows, in line
    ([1500, 1300], [3, 2], 16, 4, 2, 64, 1400),
    ([3000, 900], [5, 3], 64, 8, 2, 128, 0),                    # 20 rows of a tile of 32, in line
    ([2500], [16], 16, 4, 1, 64, 0),                            # 64 rows: two tiles
    ([600], [16], 256, 4, 1, 128, 0),                           # ... alone
    ([65, 64, 63, 31, 1], [11, 11, 11, 11, 11], 32, 2, 1, 64, 40),
    ([2500], [13], 64, 5, 1, 128, 0),                           # 65 rows: a prompt, in line
    ([700], [600], 16, 1, 1, 64, 0),                            # three row tiles
    ([700, 300], [300, 300], 256, 3, 3, 128, 129),
    ([6000], [70], 64, 2, 1, 64, 0),
    ([3000, 2000, 50, 1200, 1], [100, 1, 50, 4, 1], 64, 4, 1, 128, 0),   # every kind of row count in one batch, in line
    (list(range(100, 1800, 24)), [1] * 71, 64, 2, 1, 64, 0),    # more sequences than a wave has lanes, in line
    ([520] * 40, [1] * 40, 16, 2, 1, 128, 0),                   # ... alone
]


@pytest.mark.parametrize("case", WAYS, ids=range(len(WAYS)))
def test_ways_through_attention(torch_, case):
    torch = torch_
    lengths, rows, page, heads, kv, dim, window = case
    rng = np.random.default_rng(sum(lengths) + sum(rows) + dim)
    cache, starts, lens, table = random_batch(rng, lengths, rows, page, kv, dim)
    q = rng.standard_normal((int(starts[-1]), heads, dim)).astype(np.float16)
    dev, batch = on_device(torch, cache, starts, lens, table)
    want, size, reach = plain.attend(cache, q, starts, lens, table, dim ** -0.5, window)
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
    tl.attention_kv4(up(torch, q), out, *dev, *batch, max(rows), max(lengths), window=window)
    check_attention(out.cpu().numpy(), want, size, reach, q)
    again = torch.full_like(out, 7.0)
    tl.attention_kv4(up(torch, q), again, *dev, *batch, max(rows), max(lengths), window=window)
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))


@pytest.mark.parametrize("scale", [0.0, -0.3, 0.02])
@pytest.mark.parametrize("rows,heads", [(1, 4), (2, 4), (5, 4), (40, 2)])
def test_any_scale(torch_, scale, rows, heads):
    torch = torch_
    rng = np.random.default_rng(rows + heads)
    cache, starts, lens, table = random_batch(rng, [150, 33], [rows, rows], 16, 1, 64)
    q = rng.standard_normal((2 * rows, heads, 64)).astype(np.float16)
    dev, batch = on_device(torch, cache, starts, lens, table)
    want, size, reach = plain.attend(cache, q, starts, lens, table, scale, 0)
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
    tl.attention_kv4(up(torch, q), out, *dev, *batch, rows, 150, scale=scale)
    check_attention(out.cpu().numpy(), want, size, reach, q)


@pytest.mark.parametrize("length,rows,heads,dim,window", [
    (200, 1, 4, 128, 0), (200, 2, 4, 64, 0), (200, 6, 4, 128, 0), (200, 6, 4, 64, 30), (300, 80, 1, 128, 0), (300, 80, 1, 64, 60),
    (2500, 1, 4, 64, 0), (2500, 2, 4, 128, 0), (2500, 6, 4, 128, 0), (2500, 80, 1, 128, 0)])
def test_not_finite(torch_, length, rows, heads, dim, window):
    """A key whose group is NaN makes the rows that see it NaN, a value's group its own dims of them; other rows, dims and heads
    are what they would be."""
    torch = torch_
    rng = np.random.default_rng(length + rows + dim)
    cache, starts, lens, table = random_batch(rng, [length], [rows], 32, 2, dim)
    first = length - rows                                    # position of the first row
    spots = [("v", 0, first, 1), ("k", 1, length - 1, 0)]     # seen by all rows, by the last one
    if rows > 3:
        spots += [("v", 1, length - 3, 0), ("v", 0, length - 2, 1), ("k", 1, length - 2, 1)]
    for which, head, pos, group in spots:
        s = cache.ks if which == "k" else cache.vs
        s[table[0, pos // 32], head, group, pos % 32] = 0x7E00
    cache.vs[table[0, 2], 0, 1, 70 % 32] = 0x7E00             # far from any row's end
    q = rng.standard_normal((rows, 2 * heads, dim)).astype(np.float16)
    dev, batch = on_device(torch, cache, starts, lens, table)
    with np.errstate(invalid="ignore"):
        want, size, reach = plain.attend(cache, q, starts, lens, table, dim ** -0.5, window)
    assert np.isnan(want).any() and not np.isnan(want).all()
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
    tl.attention_kv4(up(torch, q), out, *dev, *batch, rows, length, window=window)
    got = out.cpu().numpy()
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    some = np.isnan(size)
    check_attention(np.where(np.isnan(want), 0, got), np.where(np.isnan(want), 0, want), np.where(some, 0, size), np.nan_to_num(reach), q)


@pytest.mark.parametrize("rows,heads,length", [(1, 4, 90), (1, 8, 90), (5, 4, 90), (40, 2, 90), (1, 4, 2500), (2, 4, 2500), (6, 4, 2500), (80, 1, 2500)])
def test_queries_that_are_not_finite(torch_, rows, heads, length):
    """They make their own row and head NaN and no other."""
    torch = torch_
    rng = np.random.default_rng(rows + heads + length)
    cache, starts, lens, table = random_batch(rng, [length], [rows], 64, 1, 128)
    q = rng.standard_normal((rows, heads, 128)).astype(np.float16)
    dev, batch = on_device(torch, cache, starts, lens, table)
    want, size, reach = plain.attend(cache, q, starts, lens, table, 128 ** -0.5, 0)
    bad = np.zeros((rows, heads), bool)
    bad[0, 0] = bad[rows // 2, heads - 1] = True
    q[bad] = np.where(rng.integers(0, 2, (bad.sum(), 128)), np.inf, -np.inf)
    q[bad, 3] = np.nan
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
    tl.attention_kv4(up(torch, q), out, *dev, *batch, rows, length)
    got = out.cpu().numpy()
    assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()
    want[bad] = np.nan
    check_attention(got, want, size, reach, q)


@pytest.mark.parametrize("bound", [40, 5000])
def test_many_sequences(torch_, bound):
    """A thousand of them, of 0 to 40 positions, each its own row tile; and in line, tens in a wave's piece."""
    torch = torch_
    rng = np.random.default_rng(bound)
    lengths = rng.integers(0, 41, 1000).tolist()
    cache, starts, lens, table = random_batch(rng, lengths, [1] * 1000, 16, 1, 64)
    q = rng.standard_normal((1000, 4, 64)).astype(np.float16)
    dev, batch = on_device(torch, cache, starts, lens, table)
    table_wide = torch.full((1000, 400), -1, dtype=torch.int32, device="cuda")
    table_wide[:, :table.shape[1]] = batch[2]
    want, size, reach = plain.attend(cache, q, starts, lens, table, 0.125, 0)
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
    tl.attention_kv4(up(torch, q), out, *dev, batch[0], batch[1], table_wide, 1, bound)
    check_attention(out.cpu().numpy(), want, size, reach, q)


@pytest.mark.parametrize("rows,heads", [(6, 1), (6, 2), (12, 4), (90, 1)])
def test_bounds_that_cut(torch_, rows, heads):
    """Rows from max_query on are left as they were; positions from max_length on count as absent."""
    torch = torch_
    rng = np.random.default_rng(rows)
    cache, starts, lens, table = random_batch(rng, [200, 90], [rows, rows], 16, 1, 128)
    q = rng.standard_normal((2 * rows, heads, 128)).astype(np.float16)
    dev, batch = on_device(torch, cache, starts, lens, table)
    for max_query, max_length in ((rows - 2, 200), (rows, 75), (1, 1), (2, 150)):
        want, size, reach = plain.attend(cache, q, starts, lens, table, 128 ** -0.5, 0, max_query, max_length)
        out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
        tl.attention_kv4(up(torch, q), out, *dev, *batch, max_query, max_length)
        got = out.cpu().numpy()
        check_attention(got, want, size, reach, q)
        assert (got[np.isnan(want)] == 7).all()


@pytest.mark.parametrize("rows,heads", [(6, 1), (8, 1), (12, 4), (90, 1)])
def test_the_widest_window(torch_, rows, heads):
    """A window of 2^31 - 1 positions is none, also beside rows that lie before the first position."""
    torch = torch_
    rng = np.random.default_rng(rows)
    cache, starts, lens, table = random_batch(rng, [rows - 4, 70], [rows, 4], 16, 1, 128)
    q = up(torch, rng.standard_normal((rows + 4, heads, 128)).astype(np.float16))
    dev, batch = on_device(torch, cache, starts, lens, table)
    for bound in (100, 3000):
        out = [torch.full_like(q, 7.0) for _ in range(2)]
        for o, window in zip(out, (0, 2 ** 31 - 1)):
            tl.attention_kv4(q, o, *dev, *batch, rows, bound, window=window)
        assert torch.equal(out[0].view(torch.int16), out[1].view(torch.int16))
    want, size, reach = plain.attend(cache, q.cpu().numpy(), starts, lens, table, 128 ** -0.5, 0)
    check_attention(out[1].cpu().numpy(), want, size, reach, q)


def test_shared_pages(torch_):
    """Two sequences with the same first pages, and one with a page twice."""
    torch = torch_
    rng = np.random.default_rng(5)
    cache, starts, lens, table = random_batch(rng, [100, 100, 64], [1, 4, 2], 16, 1, 64)
    table[1, :3] = table[0, :3]
    table[2, 2] = table[2, 0]
    q = rng.standard_normal((7, 4, 64)).astype(np.float16)
    dev, batch = on_device(torch, cache, starts, lens, table)
    want, size, reach = plain.attend(cache, q, starts, lens, table, 0.125, 0)
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
    tl.attention_kv4(up(torch, q), out, *dev, *batch, 4, 100)
    check_attention(out.cpu().numpy(), want, size, reach, q)


@pytest.mark.parametrize("rows,heads,length", [(1, 4, 3000), (2, 4, 3000), (5, 4, 3000), (70, 1, 3000), (70, 1, 130)])
def test_own_workspace(torch_, rows, heads, length):
    """Of exactly the bytes that are asked for, whatever they hold; not a byte behind them is written; a byte less is refused."""
    torch = torch_
    rng = np.random.default_rng(rows)
    cache, starts, lens, table = random_batch(rng, [length, 40], [rows, 1], 64, 1, 128)
    q = up(torch, rng.standard_normal((rows + 1, heads, 128)).astype(np.float16))
    dev, batch = on_device(torch, cache, starts, lens, table)
    want = torch.full_like(q, 7.0)
    tl.attention_kv4(q, want, *dev, *batch, rows, length)
    need = tl.attention_kv4_workspace_bytes(heads, *dev, *batch, rows + 1, rows, length)
    assert (need > 0) == (length == 3000)   # (short contexts need none)
    for fill in (0, 255):
        memory = torch.full((need + 256,), fill, dtype=torch.uint8, device="cuda")
        out = torch.full_like(q, 7.0)
        tl.attention_kv4(q, out, *dev, *batch, rows, length, workspace=memory[:need])
        assert torch.equal(out.view(torch.int16), want.view(torch.int16)) and bool((memory[need:] == fill).all())
    if need:
        with pytest.raises(tl.TllmError):
            tl.attention_kv4(q, out, *dev, *batch, rows, length, workspace=memory[:need - 1])


def test_streams(torch_):
    """The same calls on the default stream, and on two others at once, each with its own workspace from torch."""
    torch = torch_
    rng = np.random.default_rng(9)
    work = []
    for rows, length in ((1, 5000), (5, 2500), (40, 700)):
        cache, starts, lens, table = random_batch(rng, [length, 333], [rows, 1], 64, 2, 128)
        q = up(torch, rng.standard_normal((rows + 1, 8, 128)).astype(np.float16))
        dev, batch = on_device(torch, cache, starts, lens, table)
        want = torch.full_like(q, 7.0)
        tl.attention_kv4(q, want, *dev, *batch, rows, length)
        work.append((q, dev, batch, rows, length, want))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for round_ in range(3):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            for q, dev, batch, rows, length, want in work:
                with torch.cuda.stream(s):
                    out = torch.full_like(q, 7.0)
                tl.attention_kv4(q, out, *dev, *batch, rows, length, stream=s)
                outs.append((out, want))
    torch.cuda.synchronize()
    for out, want in outs:
        assert torch.equal(out.view(torch.int16), want.view(torch.int16))


def test_pages_behind_4_gib(torch_):
    """A cache of more than 2^32 bytes of codes each for k and v: rows on its first and last pages are those of a small cache."""
    torch = torch_
    kv, dim, page = 8, 128, 256
    per_page = kv * page * dim // 2
    n = (1 << 32) // per_page + 9
    scale_shape = (n, kv, dim // 32, page, 2)
    big = (torch.empty(n, kv, page, dim // 8, dtype=torch.int32, device="cuda"), torch.empty(scale_shape, dtype=torch.float16, device="cuda"),
           torch.empty(n, kv, page // 4, dim // 8, 4, dtype=torch.int32, device="cuda"), torch.empty(scale_shape, dtype=torch.float16, device="cuda"))
    small = tl.kv4_cache(4, page, kv, dim)
    g = torch.Generator(device="cuda").manual_seed(4)
    lengths = [700, 1]
    k, v = (torch.randn(sum(lengths), kv, dim, dtype=torch.float16, device="cuda", generator=g) for _ in range(2))
    int32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    starts, lens = int32(0, 700, 701), int32(*lengths)
    tables = {True: int32([n - 1, 0, n - 2], [n - 3, -1, -1]), False: int32([0, 1, 2], [3, -1, -1])}
    got = {}
    for is_big, cache in ((True, big), (False, small)):
        tl.kv4_append(k, v, *cache, starts, lens, tables[is_big])
        ko, vo = torch.zeros_like(k), torch.zeros_like(v)
        tl.kv4_read(ko, vo, *cache, starts, lens, tables[is_big])
        results = [ko, vo]
        for rows in (1, 3, 7, 100):   # 4, 12, 28 and 400 rows
            q = torch.randn(rows, 32, dim, dtype=torch.float16, device="cuda", generator=torch.Generator(device="cuda").manual_seed(rows))
            for bound in (700, 1 << 15):
                o = torch.full_like(q, 7.0)
                tl.attention_kv4(q, o, *cache, int32(0, rows), int32(700), tables[is_big][:1], rows, bound)
                results.append(o)
        got[is_big] = results
    torch.cuda.synchronize()
    for a, b in zip(got[True], got[False]):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_append_and_read_on_many_heads(torch_):
    """Enough rows for the launches that take two heads of k and v a wave; an odd head count; the last one alone."""
    torch = torch_
    for kv, dim, rows in ((5, 128, 6000), (3, 64, 12000), (1, 64, 33000), (2, 128, 1000)):
        rng = np.random.default_rng(kv)
        page = 64
        cache = tl.kv4_cache(-(-rows // page) + 1, page, kv, dim)
        table = torch.from_numpy(rng.permutation(-(-rows // page) + 1).astype(np.int32))[None, :].cuda()
        x = (rng.standard_normal((2, rows, kv, dim)) * 3).astype(np.float16)
        k, v = up(torch, x[0]), up(torch, x[1])
        starts, lens = up(torch, np.array([0, rows], np.int32)), up(torch, np.array([rows], np.int32))
        tl.kv4_append(k, v, *cache, starts, lens, table)
        ko, vo = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
        tl.kv4_read(ko, vo, *cache, starts, lens, table)
        for got, rows_ in ((ko, x[0]), (vo, x[1])):
            code, step, low = plain.quantise(rows_)
            want = np.repeat(low.astype(np.float64), 32, -1) + np.repeat(step.astype(np.float64), 32, -1) * code
            assert (np.abs(got.cpu().numpy().astype(np.float64) - want) <= (HALF_STEP + 2.0 ** -23) * np.abs(want) + 2.0 ** -25).all()


class Conversation:
    """Tensors of a batch of sequences in decode: what a step reads and writes lies in one place, as a captured step needs."""

    def __init__(self, torch, rng, lengths, page, heads, kv, dim, most):
        self.torch, self.heads, self.kv, self.dim, self.most, n = torch, heads, kv, dim, most, len(lengths)
        self.cache = tl.kv4_cache(n * most // page, page, kv, dim)
        self.host = plain.Cache(n * most // page, page, kv, dim)
        self.table = rng.permutation(n * most // page).astype(np.int32).reshape(n, -1)
        self.lens = np.array(lengths, np.int32)
        self.dev_table, self.dev_lens = up(torch, self.table), up(torch, self.lens)
        self.starts = {}
        self.how = dict(layout="half", scaling="banded", factor=8.0)

    def begin(self, rows):
        """Tensors for steps of these many rows of each sequence."""
        torch, n = self.torch, sum(rows)
        self.rows = rows
        self.starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.dev_starts = up(torch, self.starts)
        self.positions = torch.zeros(n, dtype=torch.int32, device="cuda")
        self.qkv = torch.zeros(n, self.heads + 2 * self.kv, self.dim, dtype=torch.float16, device="cuda")
        self.out = torch.zeros(n, self.heads, self.dim, dtype=torch.float16, device="cuda")

    def feed(self, x):
        """New rows: the lengths grow, positions follow."""
        self.lens = self.lens + np.array(self.rows, np.int32)
        pos = np.concatenate([np.arange(l - r, l) for l, r in zip(self.lens, self.rows)]).astype(np.int32)
        self.pos, self.x = pos, x
        self.dev_lens.copy_(up(self.torch, self.lens))
        self.positions.copy_(up(self.torch, pos))
        self.qkv.copy_(up(self.torch, x))

    def step(self, stream=None):
        h, kv = self.heads, self.kv
        q, k, v = self.qkv[:, :h], self.qkv[:, h:h + kv], self.qkv[:, h + kv:]
        tl.rotary(q, k, q, k, self.positions, self.dim, 500000.0, stream=stream, **self.how)
        tl.kv4_append(k, v, *self.cache, self.dev_starts, self.dev_lens, self.dev_table, stream=stream)
        tl.attention_kv4(q, self.out, *self.cache, self.dev_starts, self.dev_lens, self.dev_table, max(self.rows), self.most, stream=stream)

    def check(self):
        """Each operator against the plain forms on what the one before it gave."""
        h, kv = self.heads, self.kv
        turned = self.qkv.cpu().numpy()
        x = self.x.astype(np.float64)
        w = plain.rates(self.dim, 500000.0, "banded", 8.0)
        want = plain.turn(x[:, :h + kv], self.pos, self.dim, w, True)
        assert (np.abs(turned[:, :h + kv] - want) <= rotary_bound(x[:, :h + kv], want, self.dim, True, 1.0)).all()
        np.testing.assert_array_equal(turned[:, h + kv:], self.x[:, h + kv:])
        for b in range(len(self.rows)):
            for r in range(self.starts[b], self.starts[b + 1]):
                at, slot = divmod(int(self.pos[r]), self.host.page)
                for g in range(kv):
                    self.host.put(self.table[b, at], slot, g, turned[r, h + g], turned[r, h + kv + g])
        for got, want in zip(self.cache, self.host.arrays()):
            np.testing.assert_array_equal(got.cpu().numpy().view(want.dtype), want)
        q = turned[:, :h]
        want, size, reach = plain.attend(self.host, q, self.starts, self.lens, self.table, self.dim ** -0.5, 0)
        check_attention(self.out.cpu().numpy(), want, size, reach, q)


@pytest.mark.parametrize("heads,kv,dim,page", [(4, 1, 128, 16), (8, 2, 64, 32)])
def test_a_conversation(torch_, heads, kv, dim, page):
    """Prompts, single tokens, drafts of three, again single tokens: rotary, append, attention, in one place after another."""
    torch = torch_
    rng = np.random.default_rng(dim)
    c = Conversation(torch, rng, [0, 0, 0], page, heads, kv, dim, 128)
    for rows in ([70, 33, 1], [1, 1, 1], [1, 1, 1], [3, 3, 3], [1, 0, 1]):
        c.begin(rows)
        c.feed(rng.standard_normal((sum(rows), heads + 2 * kv, dim)).astype(np.float16))
        c.step()
        torch.cuda.synchronize()
        c.check()


@pytest.mark.parametrize("most,rows", [(256, [1, 1, 1]), (2048, [1, 1, 1]), (2048, [5, 5, 5]), (2048, [40, 40, 40])])
def test_captured_steps(torch_, most, rows):
    """One graph of rotary, append and attention, replayed while the sequences grow, with eager work between the replays: every
    replay gives what an eager step gives."""
    torch = torch_
    rng = np.random.default_rng(most + sum(rows))
    heads, kv, dim = 4, 1, 128
    captured = Conversation(torch, rng, [3, 60, 17], 16, heads, kv, dim, most)
    eager = Conversation(torch, np.random.default_rng(1), [3, 60, 17], 16, heads, kv, dim, most)
    eager.table = captured.table
    eager.dev_table = captured.dev_table
    for c in (captured, eager):
        c.begin(rows)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            captured.step(stream=side)
    for t in captured.cache:
        t.zero_()
    for i in range(4):
        x = rng.standard_normal((sum(rows), heads + 2 * kv, dim)).astype(np.float16)
        for c in (captured, eager):
            c.feed(x)
        eager.step()
        torch.cuda.synchronize()
        captured.out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured.out.view(torch.int16), eager.out.view(torch.int16)), i
        for a, b in zip(captured.cache, eager.cache):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16)), i
        torch.randn(1 << 20, device="cuda").sum().item()
