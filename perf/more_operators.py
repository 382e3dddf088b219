"""What is measured of attention with a sliding window and of the pages of a cache.

Two families:

* `window`: attention in which a query sees the last `window` keys up to its own place and the first `sinks` keys of its sequence
  (`fmha_sail_plan(..., window_size, num_sink_tokens)` and `fmha_sail`): decode, drafted tokens, prompts, chunks behind a prefix;
* `pages`: copies of pages (`kv_pages_copy`), rows of the block table that share a parent's pages (`kv_pages_fork`), pages given back
  (`kv_pages_free`) and pages in use moved together (`kv_pages_compact`).

Heads are the shards of a 64-head layer that the repository's benchmark uses.  `q` and `kv` give the batch as texts of lengths
("8x1" is eight times 1).
"""
import math
import os
import random
import sys

import torch

own = False

D = PAGE = 128
HEADS = [(64, 8), (64, 4), (32, 4), (32, 2), (16, 2), (16, 1)]
# upper ends of what `draw` covers
MOST_SEEN = 128 * 8320 * 4              # (key, KV head) pairs of a decode step
MOST_PAIRS = 4096 * 4224 * 32           # (query, key, head) triples of a prompt
MOST_MOVED = 1 << 30                    # bytes of the caches of a pool


def listed():
    return [
        # The least there is: one token of one short conversation on a small shard.
        dict(name="window_decode_b1_kv4011", family="window", q="1", kv="4011", hq=16, hk=2, window=1024, sinks=4, qt="bf16", ct="bf16", layout="hnd"),
        # An ordinary decode batch at ragged lengths; some sequences are shorter than the window.
        dict(name="window_decode_ragged_b24", family="window", q="24x1", hq=64, hk=4, window=4096, sinks=64, qt="bf16", ct="bf16", layout="nhd",
             kv="9217,3000,15001,40960,128,6145,21777,7999,12345,30001,511,18432,26000,4097,10240,35555,2222,14336,8192,29000,1,16385,5000,11111"),
        # Many long conversations, most of whose pages were given back.
        dict(name="window_decode_b128_kv131072", family="window", q="128x1", kv="128x131072", hq=64, hk=4, window=8192, sinks=128, qt="bf16",
             ct="bf16", layout="hnd"),
        # Decode over an e4m3 cache with queries in bf16.
        dict(name="window_decode_b64_e4m3", family="window", q="64x1", kv="32x60001,32x7000", hq=64, hk=8, window=2048, sinks=4, qt="bf16",
             ct="e4m3", layout="hnd"),
        # Four tokens per sequence (verification of drafted tokens), queries and cache in e4m3.
        dict(name="window_decode_b32_q4_e4m3", family="window", q="32x4", hq=64, hk=4, window=1000, sinks=16, qt="e4m3", ct="e4m3", layout="hnd",
             kv="8192,1000,3333,16384,517,2048,12000,6001,4096,9999,131,7777,14001,5120,2500,11264,8191,1025,3000,15000,"
                "640,2047,13001,6144,4097,10240,257,7168,14336,5000,2600,11111"),
        # Ragged prompts, keys and values as the projections left them.
        dict(name="window_prompts_ragged", family="window", q="5000,777,4096,333", kv="5000,777,4096,333", hq=64, hk=8, window=1024, sinks=4,
             qt="bf16", ct="bf16", layout="ragged"),
        # A chunk of a prompt behind a cached prefix, in e4m3.
        dict(name="window_chunk_e4m3", family="window", q="4096", kv="36003", hq=32, hk=4, window=4096, sinks=128, qt="e4m3", ct="e4m3", layout="hnd"),
        # A handful of pages of one layer.
        dict(name="pages_copy_n5", family="pages", op="copy", pool=64, count=5, hk=8, layers=1, ct="bf16"),
        # Four samples of each of 16 prompts: three further rows share the pages of each.
        dict(name="pages_fork_16x3", family="pages", op="fork", pool=2048, rows=16, kids=3, longest=8192, width=65, hk=4, layers=4, ct="bf16"),
        # A scheduler gives back what finished, was rolled back or fell behind the window.
        dict(name="pages_free_b512", family="pages", op="free", pool=65536, rows=512, longest=32768, width=257, window=4096, sinks=4, sharing=True),
        # The same for a small batch without sharing: latency.
        dict(name="pages_free_b8", family="pages", op="free", pool=1024, rows=8, longest=8192, width=65, window=-1, sinks=0, sharing=False),
        # A pool with holes is closed up.
        dict(name="pages_compact_8192", family="pages", op="compact", pool=8192, rows=800, longest=8192, width=65, hk=2, layers=1, ct="bf16", sharing=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _text(v):
    return ",".join(str(x) for x in v)


def draw(rng):
    if rng.random() < 0.6:
        return _draw_window(rng)
    op = rng.choice(["copy", "fork", "free", "compact"])
    c = dict(family="pages", op=op)
    hk, layers, ct = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 4]), rng.choice(["bf16", "e4m3", "kv4"])
    most = MOST_MOVED // (2 * layers * _page_bytes(hk, ct))
    if op == "copy":
        pool = _log(rng, 8, most)
        return dict(c, pool=pool, count=_log(rng, 1, pool // 2), hk=hk, layers=layers, ct=ct)
    longest = _log(rng, 200, 16384)
    width = -(-longest // PAGE) + rng.randrange(1, 4)
    if op == "free":
        rows, sharing = _log(rng, 1, 512), rng.random() < 0.5
        return dict(c, pool=rows * width + 9, rows=rows, longest=longest, width=width, window=rng.choice([-1, 1, 100, 1024, 4096]),
                    sinks=rng.choice([0, 4, 128, 200]), sharing=sharing)
    if op == "fork":
        kids = rng.choice([1, 2, 3, 7])
        rows = _log(rng, 1, max(1, min(64, most // (width + kids))))
        return dict(c, pool=rows * (width + kids), rows=rows, kids=kids, longest=longest, width=width, hk=hk, layers=layers, ct=ct)
    rows = _log(rng, 1, max(1, min(256, most // (2 * width))))
    return dict(c, pool=2 * rows * width, rows=rows, longest=longest, width=width, hk=hk, layers=layers, ct=ct, sharing=rng.random() < 0.5)


def _draw_window(rng):
    hq, hk = rng.choice(HEADS)
    qt, ct = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("bf16", "e4m3"), ("e4m3", "e4m3")])
    c = dict(family="window", hq=hq, hk=hk, qt=qt, ct=ct, layout=rng.choice(["hnd", "hnd", "nhd"]))
    sinks = rng.choice([0, 1, 4, 64, 128, 200])
    if rng.random() < 0.4:                                      # prompts and chunks: queries and cache of one type
        c["ct"] = qt
        window = _log(rng, 64, 8192)
        q = [_log(rng, 130, 4096) for _ in range(rng.choice([1, 1, 2, 3]))]
        kv = [n + rng.choice([0, _log(rng, 1, 18000)]) for n in q]
        while sum(a * min(b, window + sinks) for a, b in zip(q, kv)) * hq > MOST_PAIRS:
            q = [max(130, int(n * 0.7)) for n in q]
            window = max(64, int(window * 0.9))
        if rng.random() < 0.5:
            c["layout"], kv = "ragged", [min(n, 20000) for n in kv]
        return dict(c, q=_text(q), kv=_text(kv), window=window, sinks=sinks)
    tokens = rng.choice([1, 1, 1, 2, 4])
    b = _log(rng, 1, 128)
    window = _log(rng, 64, max(64, min(16384, MOST_SEEN // (b * hk) - sinks - PAGE)))
    longest = _log(rng, 1500, 131072)
    kv = [max(tokens, int(longest * rng.uniform(0.05, 1.0))) for _ in range(b)]
    return dict(c, q="%dx%d" % (b, tokens), kv=_text(kv), window=window, sinks=sinks)


# ----------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------

def lengths(text):
    """"3x5,7" -> [5, 5, 5, 7]"""
    out = []
    for part in str(text).split(","):
        n, _, x = part.rpartition("x")
        out += [int(x)] * int(n or 1)
    return out


def _msa():
    """The framework, imported only where its calls are made."""
    path = os.path.join(os.getcwd(), "msa-for-sail_b200", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    import msa_for_sail
    return msa_for_sail


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _pages(n):
    return -(-n // PAGE)


_TYPES = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}


def _randn(g, shape, dtype):
    """Normal values, made piece by piece."""
    x = torch.empty(shape, dtype=dtype, device="cuda")
    flat = x.view(-1)
    for i in range(0, flat.numel(), 1 << 26):
        n = min(1 << 26, flat.numel() - i)
        flat[i:i + n] = torch.randn(n, device="cuda", generator=g).to(dtype)
    return x


def _spans(case):
    """For each sequence: sinks [0, s) and keys [lo, hi) that any of its queries sees."""
    out = []
    for n, keys in zip(lengths(case["q"]), lengths(case["kv"])):
        lo = max(0, keys - n - case["window"] + 1)
        out.append((min(case["sinks"], lo), lo, keys))
    return out


def _prepare_window(case, g):
    ql, kl = lengths(case["q"]), lengths(case["kv"])
    hq, hk = case["hq"], case["hk"]
    s = {"hk": hk, "ql": ql, "kl": kl, "window": case["window"], "sinks": case["sinks"], "layout": case["layout"], "spans": _spans(case)}
    s["q"] = _randn(g, (sum(ql), hq, D), _TYPES[case["qt"]])
    s["scales"] = {}
    if case["ct"] == "e4m3":                                    # what the cache was divided by
        s["scales"] = dict(k_scale=torch.rand(hk, device="cuda", generator=g) + 0.5, v_scale=torch.rand(hk, device="cuda", generator=g) + 0.5)
    s["table"], first = None, [sum(kl[:i]) for i in range(len(kl))]
    page_size = -1
    if case["layout"] == "ragged":
        s["k"], s["v"] = (_randn(g, (sum(kl), hk, D), _TYPES[case["ct"]]) for _ in range(2))
    else:
        page_size = PAGE
        # pages behind the window were given back: their entries are 0, as `paged_kv_tables` makes them of entries without a page
        held = [[i for i in range(_pages(keys)) if i * PAGE < sinks or (i + 1) * PAGE > lo] for (sinks, lo, _), keys in zip(s["spans"], kl)]
        P = sum(len(h) for h in held)
        order = torch.randperm(P, generator=g, device="cuda").tolist()
        first, table, at = [], [], 0
        for h, keys in zip(held, kl):
            first.append(len(table))
            row = [0] * _pages(keys)
            for i in h:
                row[i], at = order[at], at + 1
            table += row
        s["table"] = _i32(table)
        shape = (P, hk, PAGE, D) if case["layout"] == "hnd" else (P, PAGE, hk, D)
        s["k"], s["v"] = (_randn(g, shape, _TYPES[case["ct"]]) for _ in range(2))
        for at, keys in zip(first, kl):                         # nobody wrote behind the last key: what is there is no number
            if keys % PAGE:
                page = table[at + _pages(keys) - 1]
                for c in (s["k"], s["v"]):
                    rows = c[page, :, keys % PAGE:] if case["layout"] == "hnd" else c[page, keys % PAGE:]
                    rows.copy_(torch.full(rows.shape, math.nan, device="cuda").to(c.dtype))
    s["first"] = torch.tensor(first, device="cuda")
    s["out"] = torch.empty(sum(ql), hq, D, dtype=torch.bfloat16, device="cuda")
    if own:
        s["plan"] = _msa().fmha_sail_plan(torch.tensor(ql, dtype=torch.int32), torch.tensor(kl, dtype=torch.int32), hq, num_kv_heads=hk,
                                          page_size=page_size, use_fp8_kvcache=case["ct"] == "e4m3", window_size=case["window"],
                                          num_sink_tokens=case["sinks"])
    return s


def _page_bytes(hk, ct):
    return hk * PAGE * {"bf16": 2 * D, "e4m3": D, "kv4": 72}[ct]


def _caches(case, g):
    """Keys' and values' caches of each layer."""
    P, hk, ct = case["pool"], case["hk"], case["ct"]
    if ct == "kv4":
        return [torch.randint(0, 256, (P, hk, PAGE, 72), dtype=torch.uint8, device="cuda", generator=g) for _ in range(2 * case["layers"])]
    return [_randn(g, (P, hk, PAGE, D), _TYPES[ct]) for _ in range(2 * case["layers"])]


def _held(case, seed):
    """Tokens of each request."""
    rng = random.Random(seed)
    return [_log(rng, 1, case["longest"]) for _ in range(case["rows"])]


def _prepare_pages(case, g, seed):
    s = {"op": case["op"], "pool": case["pool"], "ct": case.get("ct")}
    if case["op"] == "copy":
        s["caches"] = _caches(case, g)
        order = torch.randperm(case["pool"], device="cuda", generator=g).to(torch.int32)
        n = case["count"]
        s["src"], s["dst"] = order[:n].contiguous(), order[n:2 * n].contiguous()
        if n > 4:                                               # an entry of a fixed-size list that is not used
            s["src"][n // 2] = -1
        return s
    rng = random.Random(seed)
    P, R, W = case["pool"], case["rows"], case["width"]
    lens = _held(case, seed)
    order = torch.randperm(P, device="cuda", generator=g).tolist()
    table, held, shares, at = [], [], [0] * P, 0
    for b, n in enumerate(lens):
        need, row = _pages(n), []
        if case.get("sharing") and b % 4 == 3:                  # a row that was forked from the one before it
            row = table[b - 1][:min(need, max(0, held[b - 1] - 1))]
            for p in row:
                shares[p] += 1
        fresh = need - len(row)
        row, at = row + order[at:at + fresh], at + fresh
        assert at <= P
        table.append(row + [-1] * (W - need))
        held.append(need)
    kids = case.get("kids", 0) * R
    B = R + kids
    table += [[-1] * W for _ in range(kids)]
    held += [0] * kids
    free = order[at:]
    now = list(lens) + [0] * kids
    if case["op"] == "free":                                    # a third finished, some had drafted tokens rejected
        now = [0 if rng.random() < 0.33 else max(0, n - rng.choice([0, 0, 0, 3, 150])) for n in lens]
    # all that the pass changes stands in one block, so that each pass starts from the same tables
    parts = {"table": [x for row in table for x in row], "held": held, "kv_lens": now, "free": free + [-1] * (P - len(free)), "num_free": [len(free)],
             "shares": shares}
    s["start"] = _i32([x for v in parts.values() for x in v])
    s["meta"] = torch.empty_like(s["start"])
    s.update(zip(parts, s["meta"].split([len(v) for v in parts.values()])))
    s["table"] = s["table"].view(B, W)
    if case["op"] == "free" and not case["sharing"]:
        s["shares"] = None
    s["window"], s["sinks"] = case.get("window", -1), case.get("sinks", 0)
    if case["op"] == "fork":
        s["parents"] = _i32([i for i in range(R) for _ in range(case["kids"])])
        s["children"] = _i32(list(range(R, B)))
    if case["op"] == "compact" and not case["sharing"]:
        s["shares"] = None
    s["caches"] = _caches(case, g) if case["op"] != "free" else []
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = _prepare_window(case, g) if case["family"] == "window" else _prepare_pages(case, g, seed)
    s["family"] = case["family"]
    return s


# ----------------------------------------------------------------------------------------------
# plain forms
# ----------------------------------------------------------------------------------------------

def _rows(s, cache, b, at):
    """fp32 keys or values at places `at` of sequences `b` (one tensor shape): [..., KV heads, 128]."""
    first, bits = s["first"][b], _bits(cache)
    if s["layout"] == "ragged":
        x = bits[first + at]
    else:
        page = s["table"][first + at // PAGE].long()
        x = bits[page, :, at % PAGE] if s["layout"] == "hnd" else bits[page, at % PAGE]
    return x.view(cache.dtype).float()


def _attend(s, q, k, v, see):
    """q [N, hk, rows, D], k and v [N, hk, keys, D], see [N, rows, keys] -> [N, hk, rows, D]; a query that sees nothing gets zeros."""
    x = (q @ k.transpose(-1, -2) * D ** -0.5).masked_fill(~see[:, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == -math.inf, 0, m))
    total = e.sum(-1, keepdim=True)
    return (e @ v) / torch.where(total == 0, 1, total)


def _plain_window(s):
    hk, W, S = s["hk"], s["window"], s["sinks"]
    q = s["q"].float()
    if s["scales"]:
        q = (q.unflatten(1, (hk, -1)) * s["scales"]["k_scale"][:, None, None]).flatten(1, 2)
    g = q.shape[1] // hk
    ql, kl = s["ql"], s["kl"]
    n = ql[0]
    if n <= 8 and min(ql) == max(ql):                           # decode: all sequences at once
        B = len(ql)
        b = torch.arange(B, device="cuda")[:, None]
        kv = torch.tensor(kl, device="cuda")[:, None]
        lo = (kv - n - W + 1).clamp_min(0)
        most = max(hi - a for _, a, hi in s["spans"])
        sink = torch.arange(S, device="cuda")[None].expand(B, S)
        at = torch.cat([sink, lo + torch.arange(most, device="cuda")], 1)
        there = torch.cat([sink < lo, at[:, S:] < kv], 1)
        at = torch.where(there, at, kv - 1)
        k, v = (_rows(s, c, b, at).transpose(1, 2) for c in (s["k"], s["v"]))
        pos = kv - n + torch.arange(n, device="cuda")[None]     # [B, n]
        see = there[:, None] & (at[:, None] <= pos[..., None]) & ((at[:, None] > pos[..., None] - W) | (at[:, None] < S))
        x = q.view(B, n, hk, g, D).permute(0, 2, 1, 3, 4).flatten(2, 3)
        o = _attend(s, x, k, v, see.repeat_interleave(g, 1))
        out = o.unflatten(2, (n, g)).permute(0, 2, 1, 3, 4).reshape(B * n, hk * g, D)
    else:
        out = torch.empty_like(q)
        tok = 0
        for i, (n, keys) in enumerate(zip(ql, kl)):
            for r0 in range(0, n, 512):
                r1 = min(n, r0 + 512)
                first, last = keys - n + r0, keys - n + r1
                lo = max(0, first - W + 1)
                at = torch.cat([torch.arange(min(S, lo), device="cuda"), torch.arange(lo, last, device="cuda")])
                b = torch.full_like(at, i)
                k, v = (_rows(s, c, b, at).transpose(0, 1)[None] for c in (s["k"], s["v"]))
                pos = torch.arange(first, last, device="cuda")[:, None]
                see = (at[None] <= pos) & ((at[None] > pos - W) | (at[None] < S))
                x = q[tok + r0:tok + r1].view(r1 - r0, hk, g, D).permute(1, 0, 2, 3).flatten(1, 2)[None]
                o = _attend(s, x, k, v, see.repeat_interleave(g, 0)[None])[0]
                out[tok + r0:tok + r1] = o.unflatten(1, (r1 - r0, g)).permute(1, 0, 2, 3).flatten(1, 2)
            tok += n
    if s["scales"]:
        out = (out.unflatten(1, (hk, g)) * s["scales"]["v_scale"][:, None, None]).flatten(1, 2)
    return {"out": out.to(torch.bfloat16)}


def _bits(c):
    return c.view(torch.uint8) if c.dtype == torch.float8_e4m3fn else c


def _plain_copy(s):
    real = (s["src"] >= 0) & (s["dst"] >= 0)
    src, dst = s["src"][real].long(), s["dst"][real].long()
    for c in s["caches"]:
        _bits(c)[dst] = _bits(c)[src]
    return {"caches": s["caches"]}


def _plain_fork(s):
    parents, children = s["parents"].long(), s["children"].long()
    table, held, free = s["table"], s["held"], s["free"]
    lens = s["kv_lens"][parents]
    full = lens // PAGE
    part = lens % PAGE
    rank = (part > 0).cumsum(0) - 1
    new = free[(s["num_free"] - 1 - rank).clamp_min(0).long()]
    col = torch.arange(table.shape[1], device="cuda")[None]
    src = table[parents, full.clamp_max(table.shape[1] - 1).long()]
    table[children] = torch.where(col < full[:, None], table[parents], torch.where((col == full[:, None]) & (part > 0)[:, None], new[:, None], -1))
    shared = table[parents][col < full[:, None]].long()
    s["shares"].index_add_(0, shared, torch.ones_like(shared, dtype=torch.int32))
    held[children] = full + (part > 0).int()
    s["kv_lens"][children] = lens
    s["num_free"] -= (part > 0).sum().int()
    own_page = part > 0
    src, new, part = src[own_page].long(), new[own_page].long(), part[own_page]
    used = (torch.arange(PAGE, device="cuda")[None] < part[:, None]).nonzero()
    a, b, t = src[used[:, 0]], new[used[:, 0]], used[:, 1]
    for c in s["caches"]:
        if s["ct"] == "kv4":                                    # codes of a page's tokens, then their scales
            f = c.flatten(2)
            codes, scales = f[..., :PAGE * 64].unflatten(-1, (PAGE, 64)), f[..., PAGE * 64:].unflatten(-1, (PAGE, 8))
            codes[b, :, t] = codes[a, :, t]
            scales[b, :, t] = scales[a, :, t]
        else:
            _bits(c)[b, :, t] = _bits(c)[a, :, t]
    return {"table": table, "held": held, "kv_lens": s["kv_lens"], "num_free": s["num_free"], "shares": s["shares"], "caches": s["caches"]}


def _plain_free(s):
    table, held, free = s["table"], s["held"], s["free"]
    kv = s["kv_lens"].clamp_min(0)
    keep = torch.minimum((kv + PAGE - 1) // PAGE, held)[:, None]
    col = torch.arange(table.shape[1], device="cuda")[None]
    out = (col >= keep) & (col < held[:, None])
    if s["window"] > 0:
        out |= (col >= -(-s["sinks"] // PAGE)) & (col < ((kv - s["window"] + 1).clamp_min(0) // PAGE)[:, None]) & (col < keep)
    out &= table >= 0
    page = torch.where(out, table, s["pool"]).flatten().long()
    count = torch.zeros(s["pool"] + 1, dtype=torch.int32, device="cuda").index_add_(0, page, torch.ones_like(page, dtype=torch.int32))
    shares = s["shares"] if s["shares"] is not None else torch.zeros(s["pool"], dtype=torch.int32, device="cuda")
    gone = torch.cat([count[:-1] > shares, count.new_zeros(1, dtype=torch.bool)])
    order = torch.arange(page.numel(), device="cuda")
    first = torch.full((s["pool"] + 1,), page.numel(), device="cuda").scatter_reduce_(0, page, order, "amin")
    push = gone[page] & (first[page] == order)
    place = torch.where(push, s["num_free"] + push.cumsum(0) - 1, s["pool"])
    longer = torch.cat([free, free.new_zeros(1)])
    longer[place] = torch.where(push, page, 0).to(torch.int32)
    free.copy_(longer[:-1])
    if s["shares"] is not None:
        s["shares"].copy_(torch.where(gone[:-1], 0, shares - count[:-1]))
    s["num_free"] += push.sum().int()
    table[out] = -1
    held.copy_(keep[:, 0])
    res = {"table": table, "held": held, "num_free": s["num_free"], "free": free}
    return res if s["shares"] is None else {**res, "shares": s["shares"]}


def _plain_compact(s):
    table, held, free = s["table"], s["held"], s["free"]
    P = s["pool"]
    live = torch.zeros(P, dtype=torch.bool, device="cuda")
    mine = (torch.arange(table.shape[1], device="cuda")[None] < held[:, None]) & (table >= 0)
    live[table[mine].long()] = True
    managed = live.clone()
    managed[free[torch.arange(P, device="cuda") < s["num_free"]].long()] = True
    low = managed & (managed.cumsum(0) <= live.sum())           # where the pages in use go
    src, dst = (live & ~low).nonzero()[:, 0], (low & ~live).nonzero()[:, 0]
    to = torch.arange(P, dtype=torch.int32, device="cuda")
    to[src] = dst.to(torch.int32)
    table[mine] = to[table[mine].long()]
    for c in s["caches"]:
        _bits(c)[dst] = _bits(c)[src]
    if s["shares"] is not None:
        s["shares"][dst] = s["shares"][src]
        s["shares"][src] = 0
    rest = (managed & ~low).nonzero()[:, 0].flip(0).to(torch.int32)      # the lowest on top
    free[:rest.shape[0]] = rest
    s["num_free"].fill_(rest.shape[0])
    res = {"table": table, "num_free": s["num_free"], "free": free, "caches": s["caches"]}
    return res if s["shares"] is None else {**res, "shares": s["shares"]}


# ----------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------

def _own_window(msa, s):
    msa.fmha_sail(s["q"], s["k"], s["v"], s["plan"], kv_indices=s["table"], out=s["out"], **s["scales"])
    return {"out": s["out"]}


def _own_pages(msa, s):
    if s["op"] == "copy":
        msa.kv_pages_copy(s["caches"], s["src"], s["dst"])
        return {"caches": s["caches"]}
    if s["op"] == "fork":
        msa.kv_pages_fork(s["table"], s["held"], s["kv_lens"], s["parents"], s["children"], s["free"], s["num_free"], s["shares"], s["caches"])
        return {k: s[k] for k in ("table", "held", "kv_lens", "num_free", "shares", "caches")}
    if s["op"] == "free":
        msa.kv_pages_free(s["table"], s["held"], s["kv_lens"], s["free"], s["num_free"], s["shares"], window_size=s["window"],
                          num_sink_tokens=s["sinks"])
        res = {"table": s["table"], "held": s["held"], "num_free": s["num_free"], "free": s["free"]}
    else:
        msa.kv_pages_compact(s["table"], s["held"], s["free"], s["num_free"], s["caches"], s["shares"])
        res = {"table": s["table"], "num_free": s["num_free"], "free": s["free"], "caches": s["caches"]}
    return res if s["shares"] is None else {**res, "shares": s["shares"]}


_PLAIN = {"copy": _plain_copy, "fork": _plain_fork, "free": _plain_free, "compact": _plain_compact}


def run(state):
    if state["family"] == "window":
        return _own_window(_msa(), state) if own else _plain_window(state)
    if "start" in state:
        state["meta"].copy_(state["start"])
    return _own_pages(_msa(), state) if own else _PLAIN[state["op"]](state)


# ----------------------------------------------------------------------------------------------
# the definition in 64 bits
# ----------------------------------------------------------------------------------------------

def _exact_window(case, s):
    W, S, hk = case["window"], case["sinks"], case["hk"]
    if sum(n * (a + hi - lo) for n, (a, lo, hi) in zip(s["ql"], s["spans"])) * case["hq"] > 1e10:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    q = out.new_tensor(D).rsqrt() * s["q"].double().unflatten(1, (hk, -1))
    scale = {c: s["scales"][c + "_scale"].double() if s["scales"] else out.new_ones(hk) for c in "kv"}
    for h in range(hk):
        rows = [{"hnd": c[:, h], "nhd": c[:, :, h], "ragged": c[:, h]}[case["layout"]].reshape(-1, D) for c in (s["k"], s["v"])]
        tok = 0
        for i, (n, keys, (a, lo, hi)) in enumerate(zip(s["ql"], s["kl"], s["spans"])):
            j = torch.cat([torch.arange(a), torch.arange(lo, hi)]).cuda()
            at = int(s["first"][i]) + j
            if case["layout"] != "ragged":
                at = s["table"][int(s["first"][i]) + j // PAGE].long() * PAGE + j % PAGE
            k, v = (_bits(c)[at].view(c.dtype).double() for c in rows)
            k, v = k * scale["k"][h], v * scale["v"][h]
            for r0 in range(0, n, 512):
                x = q[tok + r0:tok + min(n, r0 + 512), h] @ k.T        # [rows, group, keys]
                behind = (keys - n + r0 + torch.arange(x.shape[0], device="cuda"))[:, None] - j[None]
                x[((behind < 0) | ((behind >= W) & (j[None] >= S)))[:, None].expand_as(x)] = -math.inf
                group = x.shape[1]
                out[tok + r0:tok + r0 + x.shape[0], h * group:(h + 1) * group] = torch.softmax(x, 2) @ v
            tok += n
    return {"out": out}


def _exact_pages(case, s):
    """Where each page's values end up, found by walking the tables one entry after the other."""
    if case["op"] == "free" or case["ct"] == "kv4":
        return None
    moves = []                                                  # (from, to, tokens)
    if case["op"] == "copy":
        moves = [(a, b, PAGE) for a, b in zip(s["src"].tolist(), s["dst"].tolist()) if a >= 0]
    else:
        s["meta"].copy_(s["start"])
        table, held, kv = s["table"].tolist(), s["held"].tolist(), s["kv_lens"].tolist()
        stack = s["free"].tolist()[:int(s["num_free"])]
        if case["op"] == "fork":
            for p in s["parents"].tolist():
                if kv[p] % PAGE:
                    moves.append((table[p][kv[p] // PAGE], stack.pop(), kv[p] % PAGE))
        else:
            used = sorted({p for row, n in zip(table, held) for p in row[:n] if p >= 0})
            places = sorted(set(used) | set(stack))[:len(used)]
            moves = [(a, b, PAGE) for a, b in zip([p for p in used if p > places[-1]], sorted(set(places) - set(used)))]
    caches = []
    for c in s["caches"]:
        d = c.double()
        for a, b, n in moves:
            d[b, :, :n] = c[a, :, :n].double()
        caches.append(d)
    rest = {"copy": [], "fork": ["table", "held", "kv_lens", "num_free", "shares"], "compact": ["table", "num_free", "free"]}[case["op"]]
    if case["op"] == "compact" and s["shares"] is not None:
        rest.append("shares")
    return {**{k: None for k in rest}, "caches": caches}


def exact(case, seed):
    s = prepare(case, seed)
    return (_exact_window if case["family"] == "window" else _exact_pages)(case, s)


# ----------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------

def work(case):
    if case["family"] == "window":
        ql, kl, W, S = lengths(case["q"]), lengths(case["kv"]), case["window"], case["sinks"]
        size = {"bf16": 2, "e4m3": 1}
        seen = sum(a + hi - lo for a, lo, hi in _spans(case))
        pairs = 0
        for n, keys in zip(ql, kl):
            for r in range(n):
                lo = max(0, keys - n + r + 1 - W)
                pairs += keys - n + r + 1 - lo + min(S, lo)
        return {"bytes": seen * case["hk"] * 2 * D * size[case["ct"]] + sum(ql) * case["hq"] * D * (size[case["qt"]] + 2),
                "flops": pairs * case["hq"] * 4 * D}
    if case["op"] == "copy":
        return {"bytes": 2 * 2 * case["layers"] * (case["count"] - (case["count"] > 4)) * _page_bytes(case["hk"], case["ct"]), "flops": 0}
    tables = 8 * case["rows"] * (case["width"] + 2)
    if case["op"] == "free":
        return {"bytes": tables, "flops": 0}
    token = 2 * case["layers"] * _page_bytes(case["hk"], case["ct"]) / PAGE
    if case["op"] == "fork":
        # a last page is half full on average
        return {"bytes": int(case["rows"] * case["kids"] * (token * PAGE / 2 * 2 + 8 * _pages(case["longest"]) / 4)), "flops": 0}
    # on average: pages in use by the lengths' distribution, spread evenly; those above the line move
    mean = (case["longest"] - 1) / math.log(case["longest"]) / PAGE + 0.5
    used = min(1.0, mean * case["rows"] * (0.75 if case["sharing"] else 1.0) / case["pool"])
    return {"bytes": int(tables + 2 * token * PAGE * case["pool"] * used * (1 - used)), "flops": 0}


if __name__ == "__main__":
    for seed in range(12):
        print(draw(random.Random(seed)))
