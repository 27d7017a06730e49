"""Rotary positions, the 4-bit paged key/value cache and attention over it: refusals on the CPU, values on the GPU against
the plain forms in 64 bits (tests/kv4_plain.py)."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import ternary_llm_amd as tl
from tests import kv4_plain as plain
from ternary_llm_amd import ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HALF_STEP = 2.0 ** -11   # of fp16, relative
TINY = 2.0 ** -25        # half a step of its subnormals


# ------------------------------------------------------------------------------------------------------------- refusals
def _rotary(q=0x10000, k=0x80000, q_out=0x20000, k_out=0x90000, qs=512, ks=256, qos=512, kos=256, pos=0x1000, n=4, h=8, kv=4, dim=64,
            rd=64, layout=1, scaling=0, length=8192, theta=10000.0, factor=2.0, low=1.0, high=4.0, mag=1.0, config=True):
    c = ops._RotaryConfig(rd, layout, scaling, length, theta, factor, low, high, mag)
    return tl.lib().tllm_rotary_f16(q, k, q_out, k_out, qs, ks, qos, kos, pos, n, h, kv, dim, C.byref(c) if config else None, None)


def test_rotary_refusals():
    assert _rotary(q=None) == -1 and _rotary(q_out=None) == -1 and _rotary(pos=None) == -1 and _rotary(config=False) == -1
    assert _rotary(k=None) == -1 and _rotary(k_out=None) == -1
    assert _rotary(n=0) == -2 and _rotary(h=0) == -2 and _rotary(kv=-1) == -2 and _rotary(rd=63) == -2 and _rotary(rd=66) == -2
    assert _rotary(rd=0) == -2 and _rotary(layout=2) == -2 and _rotary(scaling=5) == -2 and _rotary(scaling=-1) == -2
    assert _rotary(theta=0.0) == -2 and _rotary(theta=float("nan")) == -2 and _rotary(mag=float("inf")) == -2
    for s in (1, 2, 3, 4):
        assert _rotary(scaling=s, factor=0.0) == -2 and _rotary(scaling=s, factor=float("nan")) == -2
    for s in (3, 4):
        assert _rotary(scaling=s, low=4.0) == -2 and _rotary(scaling=s, low=0.0) == -2 and _rotary(scaling=s, length=0) == -2
    assert _rotary(scaling=4, theta=1.0) == -2 and _rotary(scaling=2, rd=2) == -2
    assert _rotary(qs=511) == -2 and _rotary(kos=255) == -2
    assert _rotary(n=1 << 24) == -4 and _rotary(h=1025, qs=1025 * 64, qos=1025 * 64) == -4
    assert _rotary(q=0x10001) == -7 and _rotary(k_out=0x90001) == -7 and _rotary(pos=0x1002) == -7
    assert _rotary(q_out=0x10002) == -5 and _rotary(k_out=0x20010) == -5 and _rotary(q_out=0x80000) == -5
    assert _rotary(q_out=0x10000, qos=520) == -5          # in place with another stride
    assert _rotary(pos=0x20010) == -5
    # rows of q, k and v in one buffer: k_out on q's part is refused, parts side by side are not an overlap (checked on the GPU)
    assert _rotary(q=0x10000, k=0x10000 + 1024, qs=1024, ks=1024, q_out=0x10000, qos=1024, k_out=0x10000 + 512, kos=1024) == -5


def _kv4(pages=4, page=16, heads=2, dim=64, batch=2, n=3, width=2, **at):
    p = dict(kc=0x100000, ks=0x200000, vc=0x300000, vs=0x400000, starts=0x10, lengths=0x40, table=0x80)
    p.update(at)
    return (ops._Kv4Cache(p["kc"], p["ks"], p["vc"], p["vs"], pages, page, heads, dim),
            ops._Kv4Batch(p["starts"], p["lengths"], p["table"], batch, n, width))


def _rows_call(name, k=0x500000, v=0x600000, k_stride=128, v_stride=128, **kw):
    c, b = _kv4(**kw)
    return getattr(tl.lib(), name)(k, v, k_stride, v_stride, c, b, None)


@pytest.mark.parametrize("name", ["tllm_kv4_append_f16", "tllm_kv4_read_f16"])
def test_cache_row_refusals(name):
    call = lambda **kw: _rows_call(name, **kw)  # noqa: E731
    f = getattr(tl.lib(), name)
    c, b = _kv4()
    assert f(0x500000, 0x600000, 128, 128, None, b, None) == -1 and f(0x500000, 0x600000, 128, 128, c, None, None) == -1
    for field in ("kc", "ks", "vc", "vs", "starts", "lengths", "table"):
        assert call(**{field: None}) == -1, field
        assert call(**{field: 0x700002}) == -7, field
    assert call(k=None) == -1 and call(v=None) == -1 and call(k=0x500008) == -7 and call(k_stride=132) == -7 and call(v_stride=120) == -2
    assert call(pages=0) == -2 and call(page=8) == -2 and call(page=48) == -2 and call(heads=0) == -2 and call(dim=96) == -2
    assert call(batch=0) == -2 and call(n=0) == -2 and call(width=0) == -2
    assert call(pages=1 << 30) == -4 and call(heads=2000, k_stride=1 << 20, v_stride=1 << 20) == -4 and call(batch=1 << 16) == -4
    assert call(n=1 << 24) == -4 and call(width=1 << 27) == -4
    assert call(k=0x100000) == -5 and call(v=0x400000 - 16) == -5
    if "append" in name:
        assert call(vc=0x100000) == -5 and call(table=0x200000) == -5
    else:
        assert call(v=0x500000) == -5 and call(k=0) != 0 and call(lengths=0x500040) == -5


def _attend_call(q=0x500000, out=0x600000, qs=256, os_=256, heads=4, mq=3, ml=32, scale=0.125, window=0, ws=0x800000, wsb=1 << 40, **kw):
    kv = kw.pop("kv_heads", 2)
    c, b = _kv4(heads=kv, **kw)
    return tl.lib().tllm_attention_kv4_f16(q, out, qs, os_, c, b, heads, mq, ml, scale, window, ws, wsb, None)


def test_attention_refusals():
    assert _attend_call(q=None) == -1 and _attend_call(out=None) == -1 and _attend_call(table=None) == -1
    assert _attend_call(heads=3) == -2 and _attend_call(heads=0) == -2 and _attend_call(mq=0) == -2 and _attend_call(ml=0) == -2
    assert _attend_call(window=-1) == -2 and _attend_call(scale=float("inf")) == -2 and _attend_call(scale=float("nan")) == -2
    assert _attend_call(heads=4098, qs=1 << 20, os_=1 << 20) == -4 and _attend_call(scale=2e12) == -2
    assert _attend_call(heads=4096, qs=1 << 20, os_=1 << 20, n=1 << 20, mq=1 << 16) == -4
    assert _attend_call(qs=248) == -2 and _attend_call(qs=260) == -7 and _attend_call(out=0x600008) == -7 and _attend_call(dim=32) == -2
    assert _attend_call(out=0x500100) == -5 and _attend_call(out=0x100000) == -5 and _attend_call(lengths=0x600040) == -5
    c, b = _kv4()
    size = tl.lib().tllm_attention_kv4_workspace_bytes
    assert size(c, b, 4, 3, 32) >= 0 and size(c, b, 3, 3, 32) == -2 and size(None, b, 4, 3, 32) == -1

    # one row over a long context is shared out: a workspace is asked for and checked
    long = dict(pages=2048, page=64, batch=1, n=1, width=2048, kc=0x10000000, ks=0x20000000, vc=0x30000000, vs=0x40000000)
    need = size(*_kv4(**long), 4, 1, 131072)
    assert need > 0
    assert _attend_call(mq=1, ml=131072, ws=None, **long) == -1
    assert _attend_call(mq=1, ml=131072, wsb=need - 1, **long) == -10 and _attend_call(mq=1, ml=131072, wsb=-1, **long) == -10
    assert _attend_call(mq=1, ml=131072, ws=0x800004, **long) == -7
    assert _attend_call(mq=1, ml=131072, ws=0x10000010, **long) == -5 and _attend_call(mq=1, ml=131072, ws=0x500010, **long) == -5
    assert _attend_call(mq=1, ml=131072, ws=0x600000 - 16, **long) == -5


def test_python_refusals():
    import torch
    q = torch.zeros(3, 4, 64, dtype=torch.float16)
    pos = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="layout"):
        tl.rotary(q, None, q, None, pos, 64, 1e4, layout="other")
    with pytest.raises(ValueError, match="scaling"):
        tl.rotary(q, None, q, None, pos, 64, 1e4, scaling="other")
    with pytest.raises(ValueError, match="int32"):
        tl.rotary(q, None, q, None, pos.long(), 64, 1e4)
    with pytest.raises(ValueError, match="fp16"):
        tl.rotary(q.float(), None, q, None, pos, 64, 1e4)
    with pytest.raises(ValueError, match="together"):
        tl.rotary(q, q, q, None, pos, 64, 1e4)
    with pytest.raises(ValueError, match="next to each other"):
        tl.rotary(q.transpose(1, 2).contiguous().transpose(1, 2), None, q, None, pos, 64, 1e4)
    with pytest.raises(ValueError, match="one GPU"):
        tl.rotary(q, None, q, None, pos, 64, 1e4)
    cache = tl.kv4_cache(4, 16, 4, 64, device="cpu")
    batch = (torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="one GPU"):
        tl.kv4_append(q, q, *cache, *batch)
    with pytest.raises(ValueError, match="one GPU"):
        tl.attention_kv4(q, q, *cache, *batch, 3, 32)
    with pytest.raises(ValueError, match="scales"):
        tl.kv4_read(q, q, cache[0], cache[1].float(), cache[2], cache[3], *batch)
    with pytest.raises(ValueError, match="codes"):
        tl.kv4_read(q, q, cache[0], cache[1], cache[0], cache[3], *batch)
    with pytest.raises(ValueError, match="query_starts"):
        tl.kv4_read(q, q, *cache, batch[1], batch[1], batch[2])
    with pytest.raises(ValueError, match="heads"):
        tl.kv4_read(q[:, :2], q[:, :2], *cache, *batch)
    with pytest.raises(ValueError, match="power of two"):
        tl.kv4_cache(4, 24, 4, 64, device="cpu")


def test_cpp_shim_compiles(tmp_path):
    """The C++ names over the C entry points, with the call refused (a NULL) so that nothing is launched."""
    src = tmp_path / "calls.cpp"
    src.write_text("""
#include "ternary_kernels.hpp"
int main() {
    ternary::error_handler() = nullptr;
    tllm_kv4_cache c{};
    tllm_kv4_batch b{};
    tllm_rotary_config r{};
    int bad = 0;
    auto refused = [&] { bad += ternary::last_error() == TLLM_ERR_NULL_POINTER; ternary::last_error() = 0; };
    ternary::rotary_forward(nullptr, nullptr, nullptr, nullptr, 0, 0, 0, 0, nullptr, 1, 1, 1, 64, r); refused();
    ternary::kv4_append(nullptr, nullptr, 0, 0, c, b); refused();
    ternary::kv4_read(nullptr, nullptr, 0, 0, c, b); refused();
    ternary::attention_kv4_forward(nullptr, nullptr, 0, 0, c, b, 1, 1, 1, 1.0f, 0, nullptr, 0); refused();
    return bad == 4 ? 0 : 1;
}
""")
    exe = tmp_path / "calls"
    libdir = os.path.dirname(tl.lib_path())
    subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I", "/opt/rocm/include", "-I", os.path.join(ROOT, "include"), str(src),
                    "-L", libdir, "-ltllm_ternary", f"-Wl,-rpath,{libdir}", "-o", str(exe)], check=True, capture_output=True, text=True)
    assert subprocess.run([str(exe)]).returncode == 0


def test_plain_layout_is_one_to_one():
    """Every dim of a k row has a nibble of its own, and putting a row and taking it back gives the values it stands for."""
    for dim in (64, 128):
        places = {plain.k_word_of(d, dim) for d in range(dim)}
        assert len(places) == dim and {w for w, _ in places} == set(range(dim // 8))
    rng = np.random.default_rng(1)
    c = plain.Cache(2, 16, 2, 128, rng)
    x = rng.standard_normal((2, 128)).astype(np.float16)
    c.put(1, 5, 1, x[0], x[1])
    for which, row in (("k", x[0]), ("v", x[1])):
        code, step, low = plain.quantise(row)
        want = np.repeat(low.astype(np.float64), 32) + np.repeat(step.astype(np.float64), 32) * code
        np.testing.assert_array_equal(c.rows(which, 1, np.array([5]), 1)[0], want)
        assert np.abs(want - row).max() <= step.max() * 0.51


# ------------------------------------------------------------------------------------------------------------------ GPU
@pytest.fixture(scope="module")
def torch_():
    import torch
    assert torch.cuda.is_available(), "these tests need the MI355X"
    tl.lib()
    return torch


def up(torch, a):
    a = np.ascontiguousarray(a)
    return torch.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a.view(np.float16) if a.dtype == np.uint16 else a).cuda()


def upload(torch, cache):
    return tuple(up(torch, a) for a in cache.arrays())


def rotary_bound(x, want, n, half, magnitude):
    """One rounding to fp16, and on the pair: the angle's fraction of a turn in fp32 (2 pi 2^-26), two units of the sine
    and cosine, their product with the magnitude, three roundings of the rotation: below 2^-21 of |x0| + |x1|."""
    mags = np.zeros_like(x)
    first, second = (slice(0, n // 2), slice(n // 2, n)) if half else (slice(0, n, 2), slice(1, n, 2))
    mags[..., first] = mags[..., second] = np.abs(x[..., first]) + np.abs(x[..., second])
    return HALF_STEP * np.abs(want) + TINY + 2.0 ** -21 * abs(magnitude) * mags


@pytest.mark.gpu
@pytest.mark.parametrize("rows,heads,kv,dim,rd,half,scaling,strided,inplace", [
    (1, 32, 8, 128, 128, True, "banded", False, False),
    (1, 1, 1, 2, 2, False, "none", False, False),
    (7, 4, 2, 64, 32, True, "linear", True, False),
    (7, 4, 2, 64, 32, False, "ntk", True, True),
    (33, 3, 1, 80, 20, False, "yarn", False, True),       # pieces of 16 bytes do not fit: one pair at a time
    (33, 3, 1, 80, 24, True, "none", False, False),
    (513, 12, 12, 128, 64, True, "yarn", True, True),
    (1500, 8, 1, 128, 128, False, "banded", False, False),
    (2, 5, 3, 1024, 1024, True, "none", False, False),     # the largest head
    (600, 2, 2, 16, 8, False, "linear", False, False),     # four pairs a head: many tokens share a workgroup
])
def test_rotary_values(torch_, rows, heads, kv, dim, rd, half, scaling, strided, inplace):
    torch = torch_
    rng = np.random.default_rng(rows * 31 + dim + rd)
    pos = rng.integers(-5, 1 << 20, rows).astype(np.int32)
    pos[0] = 0
    how = dict(layout="half" if half else "interleaved", scaling=scaling)
    magnitude, high = 1.0, 4.0
    if scaling != "none":
        how["factor"] = 4.0
    if scaling == "yarn":
        how["magnitude"], high = 1.25, 32.0
        magnitude = 1.25
    buf = rng.standard_normal((rows, heads + 2 * kv, dim)).astype(np.float16)
    whole = up(torch, buf)
    if strided:
        q, k = whole[:, :heads], whole[:, heads:heads + kv]
    else:
        q, k = whole[:, :heads].contiguous(), whole[:, heads:heads + kv].contiguous()
    qo, ko = (q, k) if inplace else (torch.full((rows, heads, dim), 7.0, dtype=torch.float16, device="cuda"),
                                     torch.full((rows, kv, dim), 7.0, dtype=torch.float16, device="cuda"))
    tl.rotary(q, k, qo, ko, up(torch, pos), rd, 500000.0, **how)
    torch.cuda.synchronize()
    w = plain.rates(rd, 500000.0, scaling, 4.0, 8192, 1.0, high)
    for got, x in ((qo, buf[:, :heads]), (ko, buf[:, heads:heads + kv])):
        x = x.astype(np.float64)
        want = plain.turn(x, pos, rd, w, half, magnitude)
        err = np.abs(got.cpu().numpy().astype(np.float64) - want)
        assert (err <= rotary_bound(x, want, rd, half, magnitude)).all(), err.max()
        np.testing.assert_array_equal(got.cpu().numpy()[..., rd:], x[..., rd:])
    if strided:  # the v part of the rows, and q and k where the outputs are elsewhere
        np.testing.assert_array_equal(whole[:, heads + kv:].cpu().numpy(), buf[:, heads + kv:])
        if not inplace:
            np.testing.assert_array_equal(whole.cpu().numpy(), buf)


@pytest.mark.gpu
def test_rotary_without_k_and_beside_rope(torch_):
    """Interleaved, unscaled, rising positions: what tllm_rope_f16 gives, within two roundings."""
    torch = torch_
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(40, 8, 128, dtype=torch.float16, device="cuda", generator=g)
    y, old = torch.empty_like(x), x.clone()
    tl.rotary(x, None, y, None, torch.arange(100, 140, dtype=torch.int32, device="cuda"), 128, 10000.0)
    tl.rope(old, old.clone(), 1, 40, 8, 8, 128, 100, 10000.0)
    assert ((y.double() - old.double()).abs() <= 2 * HALF_STEP * old.double().abs() + 2.0 ** -20 * 16).all()


def batch_of(rng, lengths, rows, page, heads, dim, extra_pages=3, fill=True, holes=()):
    """A cache image with the sequences' pages in random order (garbage in every slot that holds nothing), and its batch."""
    need = [-(-max(n, 0) // page) for n in lengths]
    cache = plain.Cache(sum(need) + extra_pages, page, heads, dim, rng)
    order = rng.permutation(cache.n)
    width = max(need + [1]) + 1
    table = np.full((len(lengths), width), -1, np.int32)
    used = 0
    for b, n in enumerate(need):
        table[b, :n] = order[used:used + n]
        used += n
    for b, j in holes:
        table[b, j] = cache.n + 7 if b % 2 else -3
    if fill:
        size = np.exp(0.4 * rng.standard_normal((2, heads, dim)))
        for b, n in enumerate(lengths):
            for j in range(need[b]):
                if not 0 <= table[b, j] < cache.n:
                    continue
                for t in range(j * page, min(n, (j + 1) * page)):
                    x = (rng.standard_normal((2, heads, dim)) * size).astype(np.float16)
                    for h in range(heads):
                        cache.put(table[b, j], t - j * page, h, x[0, h], x[1, h])
    starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    return cache, starts, np.array(lengths, np.int32), table


SPECIAL = np.array([0.0, -0.0, 65504.0, -65504.0, 6e-8, -6e-8, 1.0, np.inf, -np.inf, np.nan], np.float16)


def rows_for_quantiser(rng, n, heads, dim):
    x = (rng.standard_normal((n, heads, dim)) * np.exp(2 * rng.standard_normal((n, heads, 1)))).astype(np.float16)
    flat = x.reshape(-1, 32)
    for i in range(0, len(flat), 7):  # groups of special values, constant groups, halves between codes, tiny ones
        kind = (i // 7) % 6
        if kind == 0:
            flat[i] = rng.choice(SPECIAL, 32)
        elif kind == 1:
            flat[i] = flat[i, 0]
        elif kind == 2:
            flat[i] = rng.integers(0, 31, 32) * 0.5   # steps of 1 from 0 to 15, values on halves
            flat[i, :2] = 0, 15
        elif kind == 3:
            flat[i] = (rng.integers(-9, 9, 32) * 2.0 ** -24).astype(np.float16)
        elif kind == 4:
            flat[i] = rng.choice(SPECIAL[:7], 32)
        else:
            flat[i] = (rng.integers(-31, 31, 32) * 0.03125 + rng.choice([0, 2.0 ** -20], 32)).astype(np.float16)
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,rows,page,heads,dim,strided,holes", [
    ([1], [1], 16, 1, 64, False, ()),
    ([5, 17, 40], [1, 1, 1], 16, 2, 128, False, ()),
    ([0, 33, 70, 3, 16], [0, 33, 7, 5, 1], 32, 3, 64, True, ()),           # none, whole, some, more rows than positions
    ([130, 77], [130, 60], 64, 2, 128, True, ((1, 0),)),                    # a page that is missing
    ([50] * 70, [1] * 70, 16, 1, 128, False, ((3, 3), (64, 3))),            # more sequences than a wave has lanes
    ([1000], [999], 256, 1, 64, False, ()),
])
def test_append_and_read(torch_, lengths, rows, page, heads, dim, strided, holes):
    torch = torch_
    rng = np.random.default_rng(sum(lengths) + dim + page)
    cache, starts, lens, table = batch_of(rng, lengths, rows, page, heads, dim, fill=False, holes=holes)
    behind = 3
    n = int(starts[-1]) + behind
    x = rows_for_quantiser(rng, 2 * n, heads, dim).reshape(n, 2, heads, dim)
    whole = up(torch, x.view(np.uint16))
    k, v = (whole[:, 0], whole[:, 1]) if strided else (whole[:, 0].contiguous(), whole[:, 1].contiguous())
    dev = upload(torch, cache)
    batch = (up(torch, starts), up(torch, lens), up(torch, table))
    tl.kv4_append(k, v, *dev, *batch)
    torch.cuda.synchronize()
    placed = []
    for b in range(len(lengths)):
        for r in range(starts[b], starts[b + 1]):
            pos = int(lens[b]) - int(starts[b + 1]) + r
            if pos < 0 or pos >= table.shape[1] * page or not 0 <= table[b, pos // page] < cache.n:
                placed.append((r, None, None))
                continue
            placed.append((r, table[b, pos // page], pos % page))
            for h in range(heads):
                cache.put(table[b, pos // page], pos % page, h, x[r, 0, h], x[r, 1, h])
    for got, want, name in zip(dev, cache.arrays(), ("k_codes", "k_scales", "v_codes", "v_scales")):
        got = got.cpu().numpy()
        if want.dtype == np.uint16:  # (-0 and 0 as a minimum are the same; one NaN is as good as another)
            a, b = got, want.view(np.float16)
            assert ((a == b) | (np.isnan(a) & np.isnan(b))).all(), name
        else:
            np.testing.assert_array_equal(got.view(np.uint32), want, err_msg=name)
    ko, vo = (torch.full((n, heads, dim), 5.0, dtype=torch.float16, device="cuda") for _ in range(2))
    tl.kv4_read(ko, vo, *dev, *batch)
    torch.cuda.synchronize()
    ko, vo = ko.cpu().numpy(), vo.cpu().numpy()
    for r, page_, slot in placed:
        for h in range(heads):
            for which, got in (("k", ko[r, h]), ("v", vo[r, h])):
                if page_ is None:
                    assert (got == 0).all()
                    continue
                want = cache.rows(which, page_, np.array([slot]), h)[0]
                bad = np.isnan(want)
                assert (np.isnan(got) == bad).all()
                got, want = got[~bad].astype(np.float64), want[~bad].clip(-65504, 65504)
                assert (np.abs(got - want) <= (HALF_STEP + 2.0 ** -23) * np.abs(want) + TINY).all()
    assert (ko[-behind:] == 5).all() and (vo[-behind:] == 5).all()


def check_attention(got, want, size, reach, q, what=""):
    """One rounding of the result to fp16; and on sum p |v|: what rounding v, p and k to fp16 (half a step each) and fp32
    sums (2^-16, for up to 2^12 of them added in one accumulator in any order) can do. A score is off by at most (half a
    step + 2^-16) of scale sum |q k|, and p by twice that, relative."""
    seen = ~np.isnan(want)
    err = np.abs(got.astype(np.float64) - want)
    bound = HALF_STEP * np.abs(want) + 2 * TINY + size * (2 * HALF_STEP + 2.0 ** -16 + 2 * (HALF_STEP + 2.0 ** -16) * reach[..., None])
    assert np.isfinite(got[seen]).all(), what
    assert (err <= bound)[seen].all(), (what, float((err - bound)[seen].max()), float(err[seen].max()))


ATTENTION = [
    # lengths, rows, page, heads, kv, dim, window, holes
    ([1], [1], 16, 1, 1, 64, 0, ()),
    ([517], [1], 16, 8, 2, 64, 0, ()),
    ([0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65], [1] * 12, 16, 4, 2, 128, 0, ()),    # an empty one among them
    ([300, 40, 129], [1, 1, 1], 64, 12, 4, 128, 50, ()),
    ([100, 5, 77, 0], [5, 5, 1, 0], 32, 8, 2, 128, 0, ()),                              # drafts, none
    ([3, 90], [7, 4], 16, 6, 2, 64, 0, ()),                                             # rows before the first position
    ([200, 200], [1, 3], 16, 4, 1, 128, 0, ((0, 1), (0, 5), (1, 12), (1, 0))),           # pages missing
    ([64], [64], 16, 2, 1, 64, 0, ()),
    ([97], [97], 32, 5, 1, 128, 0, ()),                                                # a prompt, odd
    ([150, 33, 260], [150, 33, 90], 64, 4, 4, 64, 0, ()),                               # prompts, and one behind a cache
    ([190], [190], 16, 16, 1, 128, 20, ((0, 3),)),
    ([700], [40], 128, 8, 1, 128, 0, ()),
    ([260, 513, 1, 90], [130, 1, 1, 2], 16, 8, 2, 128, 0, ()),                          # prompts and single tokens together
    ([260, 513, 1, 90], [130, 1, 1, 2], 16, 3, 1, 64, 64, ()),
    ([1200], [1], 16, 32, 1, 64, 0, ()),                                               # 32 heads on one kv head
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", ATTENTION, ids=range(len(ATTENTION)))
def test_attention_values(torch_, case):
    torch = torch_
    lengths, rows, page, heads, kv, dim, window, holes = case
    rng = np.random.default_rng(sum(lengths) * 3 + heads + dim)
    cache, starts, lens, table = batch_of(rng, lengths, rows, page, kv, dim, holes=holes)
    behind = 2
    n = int(starts[-1]) + behind
    q = rng.standard_normal((n, heads, dim)).astype(np.float16)
    wide = torch.full((n, heads + 1, dim), 9.0, dtype=torch.float16, device="cuda")   # rows with a stride, for q and output
    wide[:, :heads] = up(torch, q)
    out = torch.full((n, heads + 3, dim), 7.0, dtype=torch.float16, device="cuda")
    dev = upload(torch, cache)
    batch = (up(torch, starts), up(torch, lens), up(torch, table))
    tl.attention_kv4(wide[:, :heads], out[:, 1:heads + 1], *dev, *batch, max(rows), max(max(lengths), 1), window=window)
    torch.cuda.synchronize()
    want, size, reach = plain.attend(cache, q, starts, lens, table, dim ** -0.5, window)
    got = out.cpu().numpy()
    check_attention(got[:, 1:heads + 1], want, size, reach, q)
    assert (got[:, 0] == 7).all() and (got[:, heads + 1:] == 7).all() and (got[n - behind:] == 7).all()
    empty = size.sum(-1) == 0
    assert (got[:, 1:heads + 1][:n - behind][empty[:n - behind]] == 0).all()
    # generous bounds and another scale of the launch: the same result within the same bound; twice: the same bits
    again = torch.full_like(out, 7.0)
    tl.attention_kv4(wide[:, :heads], again[:, 1:heads + 1], *dev, *batch, n, table.shape[1] * page, window=window)
    check_attention(again.cpu().numpy()[:, 1:heads + 1], want, size, reach, q)
    once = again.clone()
    tl.attention_kv4(wide[:, :heads], again[:, 1:heads + 1], *dev, *batch, n, table.shape[1] * page, window=window)
    assert torch.equal(once.view(torch.int16), again.view(torch.int16))
