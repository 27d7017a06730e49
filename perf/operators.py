"""Cases for the operators around attention: rotary positions, the 4-bit paged key/value cache (write, read back) and
attention over it, with their plain forms in torch and their values in 64 bits.

The cache. A row (one token, one kv head) is cut into groups of 32 dims; a group holds its minimum m and a step s in fp16
and one code c in 0..15 per value, which stands for m + s * c. s = fp16((max - min) / 15), c = (x - m) / s rounded to the
nearest whole number (ties to even) and kept in 0..15, 0 where s is 0.
  k_codes  int32 [pages, kv_heads, page, dim / 8]       dim d = p*64 + r*32 + q*8 + w*4 + b*2 + a is nibble 4a + 2b + r of
                                                        word q*(dim/32) + 2p + w  (p < dim/64, r,w,b,a < 2, q < 4)
  v_codes  int32 [pages, kv_heads, page/4, dim/8, 4]    dim d of token t is nibble d%8 of word [t/4][d/8][t%4]
  k_scales, v_scales  fp16 [pages, kv_heads, dim/32, page, 2]   (s, m) of each group and token
A batch is described by query_starts [batch + 1] (the rows of each sequence), lengths [batch] (its cached tokens, the rows
at hand being the last of them) and page_table [batch, width].
"""
import math
import random

import torch

own = False

GROUP = 32


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decoded token of an 8B model at the end of its context: pure latency
        {"name": "rotary_one_token", "kind": "rotary", "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "turned": 128,
         "layout": "half", "scaling": "banded", "factor": 8.0, "reach": 8192},
        # the rows of several prompts of a 70B model in one launch, positions far beyond the trained length, an odd count
        {"name": "rotary_prompts", "kind": "rotary", "tokens": 8191, "heads": 64, "kv_heads": 8, "dim": 128, "turned": 128,
         "layout": "interleaved", "scaling": "yarn", "factor": 16.0, "reach": 131072},
        # a decode step of 48 users: one new row each, written and read back
        {"name": "write_step", "kind": "write", "batch": 48, "kv_heads": 8, "dim": 128, "page": 16, "longest": 8192,
         "shortest": 100, "queries": 1, "mix": 1},
        # prompts of several users in one launch
        {"name": "write_prompts", "kind": "write", "batch": 5, "kv_heads": 8, "dim": 128, "page": 64, "longest": 16384,
         "shortest": 1500, "queries": 0, "mix": 2},
        # a short conversation of a 1B model handed over to an fp16 cache
        {"name": "read_conversation", "kind": "read", "batch": 1, "kv_heads": 8, "dim": 64, "page": 32, "longest": 777,
         "shortest": 777, "queries": 0, "mix": 3},
        # long sequences read back whole
        {"name": "read_long", "kind": "read", "batch": 4, "kv_heads": 8, "dim": 128, "page": 128, "longest": 32768,
         "shortest": 9000, "queries": 0, "mix": 4},
        # one decoded token of a 1B model, short context: latency
        {"name": "attend_one_token", "kind": "attend", "batch": 1, "heads": 32, "kv_heads": 8, "dim": 64, "page": 16,
         "longest": 517, "shortest": 517, "queries": 1, "window": 0, "mix": 5},
        # a decode step of 32 users with contexts of all lengths (8B shapes)
        {"name": "attend_step", "kind": "attend", "batch": 32, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "longest": 8192, "shortest": 200, "queries": 1, "window": 0, "mix": 6},
        # one user with a very long context (70B shapes): few rows, a long axis
        {"name": "attend_long", "kind": "attend", "batch": 1, "heads": 64, "kv_heads": 8, "dim": 128, "page": 128,
         "longest": 131072, "shortest": 131072, "queries": 1, "window": 0, "mix": 7},
        # drafts of five tokens checked for 16 users, sliding window
        {"name": "attend_drafts", "kind": "attend", "batch": 16, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32,
         "longest": 4100, "shortest": 900, "queries": 5, "window": 1024, "mix": 8},
        # a whole prompt from nothing
        {"name": "attend_prompt", "kind": "attend", "batch": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "longest": 4096, "shortest": 4096, "queries": 0, "window": 0, "mix": 9},
        # prompts taken in pieces: 512 rows each behind what is cached already, odd lengths
        {"name": "attend_pieces", "kind": "attend", "batch": 3, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "longest": 15001, "shortest": 5000, "queries": 512, "window": 0, "mix": 10},
    ]


def spread(rng, low, high):
    """A whole number between low and high, spread over their logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    kind = rng.choice(["rotary", "write", "read", "attend", "attend", "attend"])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 16])
    dim = rng.choice([64, 128, 128])
    mix = rng.randrange(1 << 20)
    if kind == "rotary":
        case = {"kind": kind, "tokens": spread(rng, 1, 8191), "heads": kv_heads * rng.choice([1, 2, 4, 8]), "kv_heads": kv_heads,
                "dim": dim, "turned": dim // rng.choice([1, 1, 2, 4]), "layout": rng.choice(["half", "interleaved"]),
                "scaling": rng.choice(["none", "linear", "ntk", "banded", "yarn"]), "factor": rng.choice([2.0, 4.0, 8.0, 16.0]),
                "reach": spread(rng, 2, 1000000)}
        case["tokens"] = max(1, min(case["tokens"], 8191 * 72 * 128 // ((case["heads"] + kv_heads) * dim)))
        return case
    page = rng.choice([16, 32, 64, 128, 256])
    if kind in ("write", "read"):
        case = {"kind": kind, "batch": spread(rng, 1, 64), "kv_heads": kv_heads, "dim": dim, "page": page,
                "longest": spread(rng, 1, 16384), "queries": rng.choice([0, 1, 7, 300]), "mix": mix}
        case["shortest"] = spread(rng, 1, case["longest"])
        case["longest"] = max(case["shortest"], min(case["longest"], (1 << 25) // (case["batch"] * kv_heads * dim)))
        case["shortest"] = min(case["shortest"], case["longest"])
        return case
    while True:
        case = {"kind": kind, "batch": spread(rng, 1, 64), "heads": kv_heads * rng.choice([1, 2, 4, 4, 8, 16]), "kv_heads": kv_heads, "dim": dim,
                "page": page, "longest": spread(rng, 1, 131072), "queries": rng.choice([1, 1, 1, 2, 6, 33, 257, 0]),
                "window": rng.choice([0, 0, 0, 100, 2048]), "mix": mix}
        case["shortest"] = spread(rng, 1, case["longest"])
        most = case["longest"] if case["queries"] == 0 else min(case["queries"], case["longest"])
        padded = case["batch"] * most * case["longest"] * case["heads"]
        if case["heads"] <= 64 and case["batch"] * case["longest"] * kv_heads * dim <= 1 << 27 and padded <= 1 << 29:
            return case


def sizes(case):
    """(cached tokens, rows) of every sequence of a case."""
    rng = random.Random(case["mix"])
    lengths = [case["longest"]] + [spread(rng, case["shortest"], case["longest"]) for _ in range(case["batch"] - 1)]
    return lengths, [n if case["queries"] == 0 else min(n, case["queries"]) for n in lengths]


# --------------------------------------------------------------------------------------------------------------- inputs
def places(case, device):
    """Where each dim's code lies: (k word, k shift, v word, v shift), int64 [dim]."""
    d = torch.arange(case["dim"], device=device)
    p, r, q, w, b, a = d // 64, d // 32 % 2, d // 8 % 4, d // 4 % 2, d // 2 % 2, d % 2
    return q * (case["dim"] // 32) + 2 * p + w, 4 * (4 * a + 2 * b + r), d // 8, 4 * (d % 8)


def quantise(x):
    """fp16 [..., dim] -> codes int32 [..., dim], (step, minimum) fp16 [..., dim / 32, 2]."""
    g = x.unflatten(-1, (-1, GROUP))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    step = ((high.double() - low.double()) / 15).half()
    # in 64 bits: a value half-way between two codes has to be seen as such
    code = torch.round((g.double() - low.double()) / torch.where(step == 0, torch.ones_like(step), step).double())
    code = torch.where(step == 0, torch.zeros_like(code), code.clamp(0, 15))
    return code.int().flatten(-2), torch.cat([step, low], -1)


def pack(codes, words, shift, count):
    """Codes int32 [..., dim] -> int32 words [..., count]; the nibbles of a word do not overlap, so their sum is their union."""
    out = torch.zeros(*codes.shape[:-1], count, dtype=torch.int64, device=codes.device)
    out.scatter_add_(-1, words.expand(codes.shape), codes.long() << shift)
    return torch.where(out >= 1 << 31, out - (1 << 32), out).int()


def store(state, k, v, seq, pos):
    """Quantises the rows k, v [n, kv_heads, dim] of the sequences `seq` and writes them at the positions `pos`."""
    kw, ks, vw, vs = state["places"]
    page = state["page_table"][seq, pos // state["page"]].long()
    slot = pos % state["page"]
    words = k.shape[-1] // 8
    kc, kd = quantise(k)
    vc, vd = quantise(v)
    state["k_codes"][page, :, slot] = pack(kc, kw, ks, words)
    state["v_codes"][page, :, slot // 4, :, slot % 4] = pack(vc, vw, vs, words)
    state["k_scales"][page, :, :, slot] = kd
    state["v_scales"][page, :, :, slot] = vd


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=gen, dtype=torch.float16)

    if case["kind"] == "rotary":
        # q, k and v lie next to each other in the rows of one projection, as q/k/v projections of one buffer leave them
        T, H, K, D = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        rows = normal(T, (H + 2 * K) * D)
        return {"case": case, "q": rows[:, :H * D].unflatten(-1, (H, D)), "k": rows[:, H * D:(H + K) * D].unflatten(-1, (K, D)),
                "positions": torch.randint(0, case["reach"], (T,), device=dev, generator=gen, dtype=torch.int32),
                "q_out": torch.empty(T, H, D, dtype=torch.float16, device=dev),
                "k_out": torch.empty(T, K, D, dtype=torch.float16, device=dev)}

    K, D, P = case["kv_heads"], case["dim"], case["page"]
    lengths, rows = sizes(case)
    B, width = len(lengths), -(-max(lengths) // P)
    pages = sum(-(-n // P) for n in lengths) + 3
    order = torch.randperm(pages, device=dev, generator=gen).int()
    table = torch.full((B, width), -1, dtype=torch.int32)
    used = 0
    host_order = order.cpu()
    for b, n in enumerate(lengths):
        need = -(-n // P)
        table[b, :need] = host_order[used:used + need]
        used += need
    starts = [0]
    for n in rows:
        starts.append(starts[-1] + n)
    state = {"case": case, "page": P, "places": places(case, dev), "max_query": max(rows), "max_length": max(lengths),
             "k_codes": torch.zeros(pages, K, P, D // 8, dtype=torch.int32, device=dev),
             "v_codes": torch.zeros(pages, K, P // 4, D // 8, 4, dtype=torch.int32, device=dev),
             "k_scales": torch.zeros(pages, K, D // GROUP, P, 2, dtype=torch.float16, device=dev),
             "v_scales": torch.zeros(pages, K, D // GROUP, P, 2, dtype=torch.float16, device=dev),
             "page_table": table.to(dev), "lengths": torch.tensor(lengths, dtype=torch.int32, device=dev),
             "query_starts": torch.tensor(starts, dtype=torch.int32, device=dev)}
    # keys have dims of their own size, as keys of trained models do; values are even
    size = torch.exp(0.5 * torch.randn(K, D, device=dev, generator=gen))
    size /= size.square().mean().sqrt()
    if case["kind"] == "write":
        state["k"], state["v"] = normal(starts[-1], K, D) * size.half(), normal(starts[-1], K, D)
        state["k_out"], state["v_out"] = torch.empty_like(state["k"]), torch.empty_like(state["v"])
        return state
    for b, n in enumerate(lengths):  # what is cached, a piece at a time
        for at in range(0, n, 16384):
            pos = torch.arange(at, min(n, at + 16384), device=dev)
            store(state, normal(len(pos), K, D) * size.half(), normal(len(pos), K, D), torch.full_like(pos, b), pos)
    if case["kind"] == "read":
        state["k_out"] = torch.empty(starts[-1], K, D, dtype=torch.float16, device=dev)
        state["v_out"] = torch.empty_like(state["k_out"])
    else:
        state["q"] = normal(starts[-1], case["heads"], D)
        state["out"] = torch.empty_like(state["q"])
    return state


# ----------------------------------------------------------------------------------------------------------- plain forms
def rotary_rates(case, device):
    """Radians per position of each pair, in 64 bits, and the magnitude of the turned pairs."""
    n, f, theta = case["turned"], case["factor"], 10000.0
    i = torch.arange(0, n, 2, dtype=torch.float64, device=device)
    rate = theta ** (-i / n)
    if case["scaling"] == "linear":
        return rate / f, 1.0
    if case["scaling"] == "ntk":
        return (theta * f ** (n / (n - 2))) ** (-i / n), 1.0
    if case["scaling"] == "banded":
        turns = 8192.0 * rate / (2 * math.pi)
        return rate * (1 / f + (1 - 1 / f) * ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)), 1.0
    if case["scaling"] == "yarn":
        low = max(0, math.floor(n * math.log(8192 / (2 * math.pi * 32)) / (2 * math.log(theta))))
        high = min(n - 1, math.ceil(n * math.log(8192 / (2 * math.pi * 1)) / (2 * math.log(theta))))
        ramp = ((i / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
        return rate * (1 - ramp + ramp / f), 0.1 * math.log(f) + 1
    return rate, 1.0


def plain_rotary(state):
    case = state["case"]
    n = case["turned"]
    rate, size = rotary_rates(case, state["q"].device)
    angle = state["positions"].double()[:, None, None] * rate
    c, s = (angle.cos() * size).float(), (angle.sin() * size).float()

    def turn(x):
        x = x.float()
        y = x.clone()
        if case["layout"] == "half":
            a, b = x[..., :n // 2], x[..., n // 2:n]
            y[..., :n // 2], y[..., n // 2:n] = a * c - b * s, a * s + b * c
        else:
            a, b = x[..., 0:n:2], x[..., 1:n:2]
            y[..., 0:n:2], y[..., 1:n:2] = a * c - b * s, a * s + b * c
        return y.half()

    return turn(state["q"]), turn(state["k"])


def row_places(state):
    """The sequence and the position of every row of the batch."""
    starts, lengths = state["query_starts"].long(), state["lengths"].long()
    row = torch.arange(state["k"].shape[0] if "k" in state else state["k_out"].shape[0], device=starts.device)
    seq = torch.searchsorted(starts, row, right=True) - 1
    return seq, lengths[seq] - starts[seq + 1] + row


def values(state, which, seq, pos):
    """What the cache holds for the sequences and positions given (any one shape), fp32 [..., kv_heads, dim]; 0 where a
    sequence has no page."""
    kw, ks, vw, vs = state["places"]
    page = state["page_table"][seq, pos // state["page"]].long()
    none = (page < 0)[..., None, None]
    page, slot = page.clamp(min=0), pos % state["page"]
    if which == "k":
        codes = state["k_codes"][page, :, slot][..., kw] >> ks
    else:
        codes = state["v_codes"][page, :, slot // 4, :, slot % 4][..., vw] >> vs
    pair = state[which + "_scales"][page, :, :, slot].float()
    found = (codes & 15).float().unflatten(-1, (-1, GROUP)) * pair[..., :1] + pair[..., 1:]
    return found.flatten(-2).masked_fill(none, 0)


def plain_attend(state):
    case, q = state["case"], state["q"]
    B, H, K, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    Q, L, dev = state["max_query"], state["max_length"], q.device
    starts, lengths = state["query_starts"].long(), state["lengths"].long()
    rows = starts[1:] - starts[:-1]
    i = torch.arange(Q, device=dev)
    real = i < rows[:, None]
    at = torch.where(real, starts[:-1, None] + i, 0)
    place = lengths[:, None] - rows[:, None] + i  # position of every row
    pos = torch.arange(L, device=dev).expand(B, L)
    seq = torch.arange(B, device=dev)[:, None].expand(B, L)
    keys, vals = values(state, "k", seq, pos), values(state, "v", seq, pos)  # [B, L, K, D]
    seen = (pos[:, None] <= place[..., None]) & real[..., None]
    if case["window"]:
        seen &= pos[:, None] > place[..., None] - case["window"]
    x = q[at].float().view(B, Q, K, H // K, D).permute(0, 2, 3, 1, 4).reshape(B, K, H // K * Q, D)
    score = (x @ keys.permute(0, 2, 3, 1)).view(B, K, H // K, Q, L) * (1 / math.sqrt(D))
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = p.view(B, K, H // K * Q, L) @ vals.permute(0, 2, 1, 3).contiguous()
    out = out.view(B, K, H // K, Q, D) / torch.where(total == 0, torch.ones_like(total), total)
    out = out.permute(0, 3, 1, 2, 4).reshape(B, Q, H, D)
    return out[real].half()


def run(state):
    """One pass: rotary (q and k turned), write (rows written, and read back as the values that the cache now stands for),
    read (whole sequences as fp16 rows), attend (a step's or a prompt's attention)."""
    case, kind = state["case"], state["case"]["kind"]
    if own:
        import ternary_llm_amd as tl

        if kind == "rotary":
            how = {"layout": case["layout"], "scaling": case["scaling"]}
            if case["scaling"] != "none":
                how["factor"] = case["factor"]
            if case["scaling"] == "yarn":
                how["magnitude"] = 0.1 * math.log(case["factor"]) + 1
            tl.rotary(state["q"], state["k"], state["q_out"], state["k_out"], state["positions"], case["turned"], 10000.0, **how)
            return state["q_out"], state["k_out"]
        cache = (state["k_codes"], state["k_scales"], state["v_codes"], state["v_scales"])
        batch = (state["query_starts"], state["lengths"], state["page_table"])
        if kind == "write":
            tl.kv4_append(state["k"], state["v"], *cache, *batch)
        if kind in ("write", "read"):
            tl.kv4_read(state["k_out"], state["v_out"], *cache, *batch)
            return state["k_out"], state["v_out"]
        tl.attention_kv4(state["q"], state["out"], *cache, *batch, state["max_query"], state["max_length"], window=case["window"])
        return state["out"]
    if kind == "rotary":
        return plain_rotary(state)
    if kind in ("write", "read"):
        seq, pos = row_places(state)
        if kind == "write":
            store(state, state["k"], state["v"], seq, pos)
        return values(state, "k", seq, pos).half(), values(state, "v", seq, pos).half()
    return plain_attend(state)


def work(case):
    if case["kind"] == "rotary":
        pairs = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["turned"] // 2
        return {"bytes": case["tokens"] * ((case["heads"] + case["kv_heads"]) * case["dim"] * 4 + 4), "flops": 6 * pairs}
    lengths, rows = sizes(case)
    K, D, P = case["kv_heads"], case["dim"], case["page"]
    about = 4 * (2 * len(lengths) + 1 + sum(-(-n // P) for n in lengths))
    held, full = 2 * K * (D // 2 + D // GROUP * 4), 2 * K * D * 2  # bytes of a token's rows in the cache, and in fp16
    if case["kind"] == "write":
        return {"bytes": sum(rows) * (2 * full + 2 * held) + about, "flops": sum(rows) * 2 * K * D * 6}
    if case["kind"] == "read":
        return {"bytes": sum(rows) * (full + held) + about, "flops": sum(rows) * 2 * K * D * 2}
    seen = pairs = 0
    for n, r in zip(lengths, rows):
        first, w = n - r, case["window"] or n + 1
        seen += n - max(0, first - w + 1)
        # row i sees min(first + i + 1, w) positions
        short = max(0, min(r, w - first))
        pairs += short * first + short * (short + 1) // 2 + (r - short) * w
    return {"bytes": seen * held + 2 * sum(rows) * case["heads"] * D * 2 + about, "flops": 4 * D * case["heads"] * pairs}


# ---------------------------------------------------------------------------------------------------- values in 64 bits
def pair_rate(case, i):
    """Radians per position of pair i, from the definition of each scaling."""
    n, f = case["turned"], case["factor"]
    rate = 10000.0 ** (-2.0 * i / n)
    turns = 8192.0 * rate / (2.0 * math.pi)  # full turns over the trained length
    if case["scaling"] == "linear":
        return rate / f
    if case["scaling"] == "ntk":
        return (10000.0 * f ** (n / (n - 2.0))) ** (-2.0 * i / n)
    if case["scaling"] == "banded":
        kept = min(1.0, max(0.0, (turns - 1.0) / 3.0))
        return kept * rate + (1.0 - kept) * rate / f
    if case["scaling"] == "yarn":
        index = lambda t: n * math.log(8192.0 / (t * 2.0 * math.pi)) / (2.0 * math.log(10000.0))  # of the pair that makes t turns
        first, last = max(math.floor(index(32.0)), 0), min(math.ceil(index(1.0)), n - 1)
        slow = min(1.0, max(0.0, (i - first) / max(last - first, 1e-3)))
        return (1.0 - slow) * rate + slow * rate / f
    return rate


def group_values(x):
    """The values that fp16 rows [n, heads, dim] have once they are held in 4 bits, from the definition, in 64 bits."""
    n, h, d = x.shape
    g = x.to(torch.float64).reshape(n, h, d // GROUP, GROUP)
    low = g.min(dim=3).values
    step = ((g.max(dim=3).values - low) / 15.0).to(torch.float16).to(torch.float64)
    code = torch.where(step[..., None] > 0, (g - low[..., None]) / step[..., None], 0.0).round().clamp(max=15.0)
    return (low[..., None] + code * step[..., None]).reshape(n, h, d)


def held_rows(state, which, b, count):
    """Sequence b's first `count` rows of the cache in 64 bits [count, kv_heads, dim], taken apart byte by byte."""
    D, P = state["case"]["dim"], state["page"]
    pages = state["page_table"][b, : -(-count // P)].long()
    words = state[which + "_codes"][pages]
    if which == "v":
        words = words.transpose(-1, -2).flatten(2, 3)  # [pages, kv_heads, page, dim / 8]
    octets = words.contiguous().view(torch.uint8)
    nibbles = torch.stack([octets % 16, octets // 16], -1).flatten(-2)  # [.., dim], nibble 0 of word 0 first
    if which == "k":
        n = nibbles.unflatten(-1, (4, D // 64, 2, 2, 2, 2))  # q p w a b r
        nibbles = n.permute(0, 1, 2, 4, 8, 3, 5, 7, 6).reshape(nibbles.shape)  # p r q w b a
    pair = state[which + "_scales"][pages].double().transpose(2, 3).repeat_interleave(GROUP, 3)  # [pages, heads, page, dim, 2]
    rows = pair[..., 1] + pair[..., 0] * nibbles.double()
    return rows.transpose(1, 2).flatten(0, 1)[:count]


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "rotary":
        size = 0.1 * math.log(case["factor"]) + 1 if case["scaling"] == "yarn" else 1.0
        rate = torch.tensor([pair_rate(case, i) for i in range(case["turned"] // 2)], dtype=torch.float64)
        turn = torch.polar(torch.full((case["tokens"], 1, len(rate)), size, dtype=torch.float64),
                           state["positions"].cpu().double()[:, None, None] * rate)
        out = []
        for x in (state["q"].cpu().double(), state["k"].cpu().double()):
            n, y = case["turned"], x.clone()
            first, second = (slice(0, n // 2), slice(n // 2, n)) if case["layout"] == "half" else (slice(0, n, 2), slice(1, n, 2))
            z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
            y[..., first], y[..., second] = z.real, z.imag
            out.append(y)
        return tuple(out)
    if case["kind"] == "write":
        return group_values(state["k"]), group_values(state["v"])
    lengths, rows = sizes(case)
    if case["kind"] == "read":
        return tuple(torch.cat([held_rows(state, w, b, n)[n - r:] for b, (n, r) in enumerate(zip(lengths, rows))]) for w in ("k", "v"))
    K, D, out, at = case["kv_heads"], case["dim"], [], 0
    G = case["heads"] // K
    for b, (n, r) in enumerate(zip(lengths, rows)):
        keys, vals = held_rows(state, "k", b, n), held_rows(state, "v", b, n)
        q = state["q"][at:at + r].double()
        at += r
        gap = torch.arange(n - r, n, device=q.device)[:, None] - torch.arange(n, device=q.device)
        hidden = (gap < 0) | (gap >= (case["window"] or n + 1))
        found = torch.empty_like(q)
        for h in range(case["heads"]):
            score = (q[:, h] @ keys[:, h // G].T) * D ** -0.5
            found[:, h] = torch.softmax(score.masked_fill(hidden, -math.inf), 1) @ vals[:, h // G]
        out.append(found)
    return torch.cat(out)
