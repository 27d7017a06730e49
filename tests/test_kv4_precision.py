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
