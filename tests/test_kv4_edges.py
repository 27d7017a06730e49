"""The attention over the 4-bit cache at the edges of what a call may hold: starts that are not ascending, positions near 2^31,
pages of 2^29 and 2^30 positions."""
import numpy as np
import pytest

import ternary_llm_amd as tl
from tests import kv4_plain as plain
from tests.test_kv4 import check_attention, torch_, up  # noqa: F401
from tests.test_kv4_serving import on_device, random_batch

pytestmark = pytest.mark.gpu

LOW, HIGH = -2 ** 31, 2 ** 31 - 1


@pytest.mark.parametrize("bound", [90, 5000])
@pytest.mark.parametrize("max_query,heads", [(1, 4), (2, 4), (5, 4), (16, 4), (80, 1)])
def test_starts_that_do_not_ascend(torch_, max_query, heads, bound):
    """Sequences whose starts descend or lie out of range have no rows there: nothing but their rows inside the row arrays is
    written, and the sequences beside them are what they would be."""
    torch = torch_
    rng = np.random.default_rng(max_query + heads + bound)
    n, behind = max_query + 6, 40
    cache, _, lens, table = random_batch(rng, [90] * 8, [1] * 8, 16, 1, 128)
    q = rng.standard_normal((n + 2 * behind, heads, 128)).astype(np.float16)
    dev, (_, dev_lens, dev_table) = on_device(torch, cache, np.zeros(1, np.int32), lens, table)
    dev_q = up(torch, q)[behind:behind + n]
    for middle in ([1 << 30, -3 * (1 << 29), 1, LOW, 1, 0, LOW], [805306368, 0, HIGH, LOW, HIGH, -1, 2], [n, n + 1, -5, n, 7, 7, 3],
                   [HIGH, HIGH, LOW, LOW, 0, -1, HIGH]):
        starts = np.array([0, max_query] + middle, np.int32)
        claimed = np.zeros(n, int)
        sound = [(0, max_query)]
        for s0, s1 in zip(starts[:-1].tolist(), starts[1:].tolist()):
            if 0 <= s0 < min(s1, n):
                claimed[s0:min(s1, n, s0 + max_query)] += 1
        out = torch.full((n + 2 * behind, heads, 128), 7.0, dtype=torch.float16, device="cuda")
        tl.attention_kv4(dev_q, out[behind:behind + n], *dev, up(torch, starts), dev_lens, dev_table, max_query, bound)
        got = out.cpu().numpy()
        assert (got[:behind] == 7).all() and (got[behind + n:] == 7).all() and (got[behind:behind + n][claimed == 0] == 7).all()
        want, size, reach = plain.attend(cache, q[behind:behind + n], sound[0], lens[:1], table[:1], 128 ** -0.5, 0)
        want[claimed != 1] = np.nan
        check_attention(got[behind:behind + n], want, size, reach, q)


@pytest.mark.parametrize("rows,heads", [(1, 4), (2, 4), (5, 4), (80, 1)])
def test_positions_near_two_to_the_31(torch_, rows, heads):
    """The last positions that a page table can have, in a window: those of a short sequence with the same rows."""
    torch = torch_
    rng = np.random.default_rng(rows + heads)
    page, held, width = 16, 13 * 16, (1 << 27) - 1
    cache, starts, lens, table = random_batch(rng, [held], [rows], page, 1, 64)
    q = up(torch, rng.standard_normal((rows, heads, 64)).astype(np.float16))
    dev, batch = on_device(torch, cache, starts, lens, table)
    far = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    far[0, width - table.shape[1]:] = batch[2][0]
    capacity = width * page
    want, size, reach = plain.attend(cache, q.cpu().numpy(), starts, lens, table, 0.125, 50)
    for bound in (capacity, HIGH):
        out = torch.full_like(q, 7.0)
        tl.attention_kv4(q, out, *dev, batch[0], up(torch, np.array([capacity], np.int32)), far, rows, bound, window=50)
        check_attention(out.cpu().numpy(), want, size, reach, q)
    # more positions than the table has: those behind it are not seen, and the window counts from the row
    more = 20
    out = torch.full_like(q, 7.0)
    tl.attention_kv4(q, out, *dev, batch[0], up(torch, np.array([capacity + 14], np.int32)), far, rows, HIGH, window=50 + more)
    moved, size, reach = plain.attend(cache, q.cpu().numpy(), starts, lens + 14, table, 0.125, 50 + more, max_length=held)
    check_attention(out.cpu().numpy(), moved, size, reach, q)


@pytest.mark.parametrize("dim,page", [(128, 1 << 29), (64, 1 << 30)])
def test_the_largest_pages(torch_, dim, page):
    """One page whose groups of steps lie 2^31 and 2^32 bytes apart: rows at its beginning and at its end are those of a small cache."""
    torch = torch_
    need = page * dim + 4 * page * dim // 32 * 2
    if torch.cuda.mem_get_info()[0] < need + (8 << 30):
        pytest.skip("the card has no room for a page of this size")
    scales = (1, 1, dim // 32, page, 2)
    big = (torch.empty(1, 1, page, dim // 8, dtype=torch.int32, device="cuda"), torch.empty(scales, dtype=torch.float16, device="cuda"),
           torch.empty(1, 1, page // 4, dim // 8, 4, dtype=torch.int32, device="cuda"), torch.empty(scales, dtype=torch.float16, device="cuda"))
    int32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    small, rows = tl.kv4_cache(1, 512, 1, dim), 300
    table = int32([0])
    # (each group of its own size, so that another's step shows)
    size = torch.tensor([1.0, 0.25, 4.0, 0.0625], device="cuda")[:dim // 32].repeat_interleave(32).half()
    for at_end in (False, True):
        gen = torch.Generator(device="cuda").manual_seed(dim)
        k, v = (torch.randn(rows, 1, dim, dtype=torch.float16, device="cuda", generator=gen) * size for _ in range(2))
        got = []
        for cache, length in ((big, page if at_end else rows), (small, 512 if at_end else rows)):
            batch = (int32(0, rows), int32(length), table)
            tl.kv4_append(k, v, *cache, *batch)
            ko, vo = torch.zeros_like(k), torch.zeros_like(v)
            tl.kv4_read(ko, vo, *cache, *batch)
            results = [ko, vo]
            for n in (1, 2, 7, 100):
                q = torch.randn(n, 4, dim, dtype=torch.float16, device="cuda", generator=torch.Generator(device="cuda").manual_seed(n))
                o = torch.full_like(q, 7.0)
                tl.attention_kv4(q, o, *cache, int32(0, n), int32(length), table, n, length, window=100)
                results.append(o)
            got.append(results)
        for a, b in zip(*got):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))
        k_read, v_read = got[1][:2]
        assert ((v_read - v).abs() <= 0.6 * size).all() and ((k_read - k).abs() <= 0.6 * size).all()
