"""What is measured of the operators around the attention path of a serving step.

Three families:

* `tables`: the page table, the slots and the positions of a step, built on the GPU from the requests' lengths, pages for new
  tokens taken from a stack of free ones (`paged_kv_tables`);
* `rope`: the norm of every query and key head, the rotation, and the write of keys and values into the paged cache, in bf16,
  e4m3 or 4 bits (`qk_norm_rope`; 4-bit rows are read back with `kv4_read`);
* `kv4`: attention over a cache held in 4 bits (`fmha_sail`), dense or over selected pages, decode or a prompt's chunk.

A 4-bit cache is uint8 [pages, KV heads, 128, 72]: the 9 216 bytes of one page and head are 128 rows of 64 bytes (two e2m1 codes a
byte, the even element in the low half), then 128 rows of eight e4m3 scales, one for each 16 elements.

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
MOST_ROPE = 32768 * 72                  # (token, head) rows of a norm and rotation
MOST_KEYS = 1048576 * 8                 # (key, KV head) pairs of a cache
MOST_PAIRS = 2048 * 20011 * 32          # (query, key, head) triples of a prompt's chunk
MOST_PICKED = 65536                     # (token, KV head, selected page) triples


def listed():
    return [
        # A decode step of a few requests: one launch, where latency is everything.
        dict(name="tables_decode_b8", family="tables", seed_lens=3, batch=8, longest=8192, tokens=1, width=128),
        # A full scheduler: two thousand requests at ragged lengths, drafted tokens for each.
        dict(name="tables_b2048", family="tables", seed_lens=5, batch=2048, longest=32768, tokens=3, width=257),
        # Decode: one token each of 32 requests, appended to a 4-bit cache; half of the head dimension is rotated.
        dict(name="rope_decode_b32_kv4", family="rope", tokens=32, hq=64, hk=4, rotary=64, style="half", axes=1, cache="kv4", weight="dim"),
        # A short prompt of odd length on a small shard, e4m3 queries and cache, neighbouring elements as pairs, a weight per head.
        dict(name="rope_prompt_t777_e4m3", family="rope", tokens=777, hq=16, hk=2, rotary=128, style="pairs", axes=1, cache="e4m3", weight="head"),
        # Tokens of a video prompt: three position axes, no cache yet (ragged prefill takes q and k as they are).
        dict(name="rope_video_t8192", family="rope", tokens=8192, hq=64, hk=8, rotary=128, style="half", axes=3, cache="none", weight="dim"),
        # A long prompt's chunk into a 4-bit cache.
        dict(name="rope_prompt_t32768_kv4", family="rope", tokens=32768, hq=64, hk=4, rotary=64, style="half", axes=1, cache="kv4", weight="dim"),
        # The least there is: one short sequence on a small shard.
        dict(name="kv4_decode_b1_kv4011", family="kv4", q="1", kv="4011", hq=16, hk=2, topk=0, heads_scale=False),
        # Sparse decode at long context: 16 selected pages of 1 024.
        dict(name="kv4_sparse_b32_kv131072", family="kv4", q="32x1", kv="32x131072", hq=64, hk=8, topk=16, heads_scale=True),
        # An ordinary decode batch at ragged lengths.
        dict(name="kv4_decode_ragged_b24", family="kv4", q="24x1", hq=64, hk=4, topk=0, heads_scale=True,
             kv="9217,3000,15001,40960,128,6145,21777,7999,12345,30001,511,18432,26000,4097,10240,35555,2222,14336,8192,29000,1,16385,5000,11111"),
        # Four tokens per sequence (verification of drafted tokens): 64 rows share a KV head.
        dict(name="kv4_decode_b32_q4", family="kv4", q="32x4", hq=64, hk=4, topk=0, heads_scale=False,
             kv="8192,1000,3333,16384,517,2048,12000,6001,4096,9999,131,7777,14001,5120,2500,11264,8191,1025,3000,15000,"
                "640,2047,13001,6144,4097,10240,257,7168,14336,5000,2600,11111"),
        # One sequence of a million tokens.
        dict(name="kv4_decode_kv1048576", family="kv4", q="1", kv="1048576", hq=64, hk=8, topk=0, heads_scale=False),
        # A chunk of a prompt behind a cached prefix.
        dict(name="kv4_prefill_chunk", family="kv4", q="2048", kv="20011", hq=32, hk=4, topk=0, heads_scale=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _text(v):
    return ",".join(str(x) for x in v)


def draw(rng):
    family = rng.choice(["tables", "rope", "rope", "kv4", "kv4", "kv4"])
    if family == "tables":
        longest = _log(rng, 200, 32768)
        return dict(family="tables", seed_lens=rng.randrange(1 << 20), batch=_log(rng, 1, 2048), longest=longest,
                    tokens=rng.choice([1, 1, 2, 5]), width=-(-longest // PAGE) + rng.randrange(4))
    hq, hk = rng.choice(HEADS)
    if family == "rope":
        tokens = min(_log(rng, 1, 32768), MOST_ROPE // (hq + 2 * hk))
        return dict(family="rope", tokens=tokens, hq=hq, hk=hk, rotary=rng.choice([32, 64, 96, 128]), style=rng.choice(["half", "half", "pairs"]),
                    axes=rng.choice([1, 1, 2, 3]), cache=rng.choice(["none", "bf16", "e4m3", "kv4", "kv4"]),
                    weight=rng.choice(["dim", "head", "none"]))
    c = dict(family="kv4", hq=hq, hk=hk, heads_scale=rng.random() < 0.5, topk=0)
    kind = rng.choice(["decode", "decode", "sparse", "chunk"])
    if kind == "chunk":
        q = [_log(rng, 130, 2048) for _ in range(rng.choice([1, 1, 2, 3]))]
        kv = [n + _log(rng, 1, 18000) for n in q]
        while len(q) * max(q) * max(kv) * hq > MOST_PAIRS:
            q = [max(130, int(n * 0.7)) for n in q]
            kv = [max(n, int(m * 0.7)) for n, m in zip(q, kv)]
        c.update(q=_text(q), kv=_text(kv))
        return c
    tokens = rng.choice([1, 1, 1, 2, 4, 8])
    if kind == "sparse":
        c["topk"] = rng.choice([4, 8, 16, 16, 32])
        b = _log(rng, 1, max(1, min(64, MOST_PICKED // (tokens * hk * c["topk"]))))
    else:
        b = _log(rng, 1, 64)
    most = min(131072 if b > 1 else 1048576, MOST_KEYS // (b * hk))
    longest = _log(rng, min(1500, most), most)
    kv = [max(tokens, int(longest * rng.uniform(0.1, 1.0))) for _ in range(b)]
    c.update(q="%dx%d" % (b, tokens), kv=_text(kv))
    return c


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


def _table_lens(case):
    """(new tokens, keys with them) per request; every eighth request of a larger batch idles this step."""
    rng = random.Random(case["seed_lens"])
    kv = [_log(rng, case["tokens"], case["longest"]) for _ in range(case["batch"])]
    ql = [0 if case["batch"] > 8 and i % 8 == 5 else min(case["tokens"], n) for i, n in enumerate(kv)]
    if case["batch"] > 64:                                      # some prompts' chunks among the decodes
        ql = [min(n, 200) if i % 64 == 9 else t for i, (t, n) in enumerate(zip(ql, kv))]
    return ql, kv


def _pages(kv):
    return [-(-n // PAGE) for n in kv]


def _prepare_tables(case, g):
    ql, kv = _table_lens(case)
    need = _pages(kv)
    held = _pages([n - t for t, n in zip(ql, kv)])              # pages of what was there before this step
    new = sum(need) - sum(held)
    pool = sum(need) + 37
    order = torch.randperm(pool, device="cuda", generator=g).to(torch.int32)
    table = torch.full((case["batch"], case["width"]), -1, dtype=torch.int32, device="cuda")
    cols = torch.arange(case["width"], device="cuda")
    mine = cols[None] < _i32(held)[:, None]
    table[mine] = order[:sum(held)]
    s = {"ql": _i32(ql), "kl": _i32(kv), "table": table, "held": _i32(held), "free": order[sum(held):].clone(),
         "num_free": _i32([pool - sum(held)]), "total_q": sum(ql) + 11, "pages": sum(need) + 5}
    assert new <= pool - sum(held)
    return s


def _sections(case):
    """Frequency pairs of each axis."""
    half = case["rotary"] // 2
    if case["axes"] == 1:
        return [half]
    first = half // 4
    rest = (half - first) // (case["axes"] - 1)
    return [half - rest * (case["axes"] - 1)] + [rest] * (case["axes"] - 1)


def _inv_freq(case):
    half = case["rotary"] // 2
    return torch.tensor([5e6 ** (-i / half) for i in range(half)], dtype=torch.float64)


def _prepare_rope(case, g):
    T, hq, hk = case["tokens"], case["hq"], case["hk"]
    heads = hq + 2 * hk
    x = torch.empty(T, heads, D, dtype=torch.bfloat16, device="cuda")       # one projection's output, q, k and v side by side
    step = max(1, (1 << 26) // (heads * D))
    for i in range(0, T, step):
        x[i:i + step] = torch.randn(min(step, T - i), heads, D, device="cuda", generator=g)
    x *= torch.rand(heads, 1, device="cuda", generator=g) * 2 + 0.2
    s = {"q": x[:, :hq], "k": x[:, hq:hq + hk], "v": x[:, hq + hk:], "cache": case["cache"], "style": case["style"], "rotary": case["rotary"]}
    s["w_q"] = s["w_k"] = None
    if case["weight"] != "none":
        shape = (D,) if case["weight"] == "dim" else (0, D)
        s["w_q"] = torch.rand(*(n or hq for n in shape), device="cuda", generator=g) + 0.5
        s["w_k"] = torch.rand(*(n or hk for n in shape), device="cuda", generator=g) + 0.5
    start = torch.randint(0, 900000, (case["axes"], 1), device="cuda", generator=g)
    span = torch.randint(0, 64, (case["axes"], T), device="cuda", generator=g)
    span[0] = torch.arange(T, device="cuda")
    s["pos"] = (start + span).to(torch.int32)
    s["sections"] = _sections(case)
    s["inv_freq"] = _inv_freq(case)
    s["turn"] = s["inv_freq"].cuda()
    s["axis"] = torch.repeat_interleave(torch.arange(case["axes"]), torch.tensor(s["sections"])).cuda()
    s["lut"] = _lut()
    s["slots"] = None
    if case["cache"] != "none":
        P = -(-T // PAGE) + 2
        free = torch.randperm(P, device="cuda", generator=g)
        t = torch.arange(T, device="cuda")
        s["slots"] = (free[t // PAGE] * PAGE + t % PAGE).to(torch.int32)
        if T > 4:                                               # padding rows of a captured step have no slot
            s["slots"][-2:] = -1
        if case["cache"] == "kv4":
            s["kc"], s["vc"] = (torch.zeros(P, hk, PAGE, 72, dtype=torch.uint8, device="cuda") for _ in range(2))
        else:
            dt = torch.bfloat16 if case["cache"] == "bf16" else torch.float8_e4m3fn
            s["kc"], s["vc"] = (torch.zeros(P, hk, PAGE, D, device="cuda").to(dt) for _ in range(2))
        low = case["cache"] == "e4m3"
        s["k_scale"] = torch.full((hk,), 0.03125 if low else 0.5, device="cuda")
        s["v_scale"] = torch.full((hk,), 0.0625 if low else 0.25, device="cuda")
        if case["cache"] == "bf16":
            s["k_scale"] = s["v_scale"] = None
    if own:
        s["rope"] = _msa().rope_plan(case["rotary"], inv_freq=s["inv_freq"], sections=s["sections"], interleaved=case["style"] == "pairs")
    return s


def _random_kv4(g, P, hk):
    """Codes and scales of values with an rms of about one."""
    c = torch.randint(0, 256, (P, hk, PAGE * 72), device="cuda", generator=g, dtype=torch.uint8)
    step = max(1, (1 << 25) // (hk * PAGE * 8))
    for i in range(0, P, step):
        n = min(step, P - i)
        sc = torch.rand(n, hk, PAGE * 8, device="cuda", generator=g) * 0.4 + 0.15
        c[i:i + n, :, PAGE * 64:] = sc.to(torch.float8_e4m3fn).view(torch.uint8)
    return c.view(P, hk, PAGE, 72)


def _pad_index(ql):
    """Token number of (sequence, i), and whether there is one."""
    start = torch.tensor([sum(ql[:i]) for i in range(len(ql))], device="cuda")
    i = torch.arange(max(ql), device="cuda")
    ok = i[None] < torch.tensor(ql, device="cuda")[:, None]
    return torch.where(ok, start[:, None] + i[None], 0), ok


def _prepare_kv4(case, g):
    ql, kl = lengths(case["q"]), lengths(case["kv"])
    hq, hk, T, topk = case["hq"], case["hk"], sum(ql), case["topk"]
    need = _pages(kl)
    P = sum(need)
    s = {"hq": hq, "hk": hk, "topk": topk, "ql": ql, "kl": kl, "P": P}
    s["q"] = torch.randn(T, hq, D, device="cuda", generator=g, dtype=torch.bfloat16)
    s["k"], s["v"] = _random_kv4(g, P, hk), _random_kv4(g, P, hk)
    s["table"] = torch.randperm(P, device="cuda", generator=g).to(torch.int32)
    ends = [sum(need[:i + 1]) - 1 for i in range(len(need))]
    for i, n in zip(ends, kl):                                  # nobody wrote behind the last key: what is there is no number
        if n % PAGE:
            for c in (s["k"], s["v"]):
                c.view(P, hk, PAGE * 72)[s["table"][i].long(), :, PAGE * 64 + 8 * (n % PAGE):] = 0x7F
    s["scales"] = {}
    if case["heads_scale"]:
        s["scales"] = dict(k_scale=torch.rand(hk, device="cuda", generator=g) + 0.5, v_scale=torch.rand(hk, device="cuda", generator=g) + 0.5)
    s["lut"] = _lut()
    start = [sum(need[:i]) for i in range(len(need))]
    if topk:
        tok_b = torch.repeat_interleave(torch.arange(len(ql)), torch.tensor(ql))
        seen = torch.tensor([kl[b] - ql[b] + i + 1 for b in range(len(ql)) for i in range(ql[b])])
        tok_b, seen = tok_b.cuda(), seen.cuda()
        vis = -(-seen // PAGE)
        score = torch.rand(T, hk, max(max(need), topk), device="cuda", generator=g)
        score[torch.arange(score.shape[2], device="cuda")[None, None].expand_as(score) >= vis[:, None, None]] = -1
        val, idx = score.topk(topk, dim=2)
        idx = torch.where(val < 0, 1 << 30, idx).sort(dim=2).values
        s["blocks"] = torch.where(idx == 1 << 30, -1, idx).to(torch.int32)
        s["seen"], s["start"] = seen, torch.tensor(start, device="cuda")[tok_b]
    else:
        s["tok"], s["ok"] = _pad_index(ql)
        col = torch.arange(max(need), device="cuda")
        at = torch.tensor(start, device="cuda")[:, None] + col[None]
        s["pages"] = s["table"].long()[torch.where(col[None] < torch.tensor(need, device="cuda")[:, None], at, 0)]
        s["len_q"], s["len_k"] = torch.tensor(ql, device="cuda"), torch.tensor(kl, device="cuda")
    s["out"] = torch.empty(T, hq, D, dtype=torch.bfloat16, device="cuda")
    s["lse"] = torch.empty(T, hq, device="cuda")
    if own:
        s["plan"] = _msa().fmha_sail_plan(torch.tensor(ql, dtype=torch.int32), torch.tensor(kl, dtype=torch.int32), hq, num_kv_heads=hk,
                                          page_size=PAGE, kv_block_num=topk if topk else -1, use_kv4_cache=True)
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"tables": _prepare_tables, "rope": _prepare_rope, "kv4": _prepare_kv4}[case["family"]](case, g)
    s["family"] = case["family"]
    return s


# ----------------------------------------------------------------------------------------------
# plain forms
# ----------------------------------------------------------------------------------------------

def _lut():
    m = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    return torch.tensor(m + [-x for x in m], device="cuda")


def _plain_tables(s):
    kl, ql, held = s["kl"].long(), s["ql"].long(), s["held"].long()
    B, W = s["table"].shape
    need = (kl + PAGE - 1) // PAGE
    ptr = torch.cat([need.new_zeros(1), need.cumsum(0)])
    new = (need - held).clamp_min(0)
    first_new = new.cumsum(0) - new
    col = torch.arange(W, device=kl.device)[None]
    fresh = (col >= held[:, None]) & (col < need[:, None])
    rank = first_new[:, None] + col - held[:, None]
    pop = (s["num_free"].long() - 1 - rank).clamp(0, s["free"].numel() - 1)
    table = torch.where(fresh, s["free"][pop], s["table"])
    flat = torch.full((s["pages"],), -1, dtype=torch.int32, device=kl.device)
    live = col < need[:, None]
    flat[(ptr[:-1, None] + col)[live]] = table[live]
    q0 = torch.cat([ql.new_zeros(1), ql.cumsum(0)])
    t = torch.arange(s["total_q"], device=kl.device)
    b = torch.searchsorted(q0[1:], t, right=True).clamp_max(B - 1)
    real = t < q0[-1]
    pos = torch.where(real, kl[b] - ql[b] + t - q0[b], 0)
    slot = table.long()[b, pos // PAGE] * PAGE + pos % PAGE
    return {"kv_indices": flat, "kv_page_indptr": ptr.to(torch.int32), "slot_map": torch.where(real, slot, -1).to(torch.int32),
            "positions": pos.to(torch.int32), "block_table": table, "num_held": torch.maximum(held, need).to(torch.int32),
            "num_free": (s["num_free"] - new.sum()).to(torch.int32)}


def _plain_norm_rope(s, x, w, dt):
    """x in `dt`: normed over the head, then rotated.  Angles are taken in 64 bits: positions are far."""
    x = x.to(dt)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    if w is not None:
        y = y * w.to(dt)
    t = s["pos"].double()[s["axis"]].T * s["turn"]              # [T, pairs]
    c, n = torch.cos(t).to(dt)[:, None], torch.sin(t).to(dt)[:, None]
    R = s["rotary"]
    if s["style"] == "half":
        a, b = y[..., :R // 2], y[..., R // 2:R]
        turned = torch.cat([a * c - b * n, b * c + a * n], -1)
    else:
        a, b = y[..., 0:R:2], y[..., 1:R:2]
        turned = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    return torch.cat([turned, y[..., R:]], -1)


def _to_e4m3(x, scale):
    return (x.float() / scale).clamp(-448, 448).to(torch.float8_e4m3fn)


def _quantise(x, scale):
    """bf16 [T, H, 128] -> codes [T, H, 128] and scales [T, H, 8], as bytes."""
    y = (x.float() / scale[:, None]).unflatten(-1, (8, 16))
    sc = (y.abs().amax(-1, keepdim=True) / 6).clamp(2.0 ** -9, 448).to(torch.float8_e4m3fn)
    r = y / sc.float()
    m = r.abs()
    code = ((m > 0.25).int() + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5)) | (torch.signbit(r).int() << 3)
    return code.flatten(-2), sc.view(torch.uint8)[..., 0]


def _parts(c):
    """Codes [P, H, 128, 64] and scales [P, H, 128, 8] of a cache, as views."""
    f = c.flatten(2)
    return f[..., :PAGE * 64].unflatten(-1, (PAGE, 64)), f[..., PAGE * 64:].unflatten(-1, (PAGE, 8))


def _values(code_bytes, scale_bytes, lut):
    """[..., 64] and [..., 8] bytes -> fp32 [..., 128]."""
    code = torch.stack([code_bytes & 15, code_bytes >> 4], -1).flatten(-2)
    v = lut[code.int()].unflatten(-1, (8, 16)) * scale_bytes.view(torch.float8_e4m3fn).float()[..., None]
    return v.flatten(-2)


def _plain_append_kv4(s, x, cache, scale):
    codes, scales = _quantise(x, scale)
    real = s["slots"] >= 0
    at = s["slots"][real].long()
    c, f = _parts(cache)
    c[at // PAGE, :, at % PAGE] = (codes[..., 0::2] | codes[..., 1::2] << 4).to(torch.uint8)[real]
    f[at // PAGE, :, at % PAGE] = scales[real]
    got = torch.zeros(x.shape, dtype=torch.bfloat16, device=x.device)
    got[real] = _values(c[at // PAGE, :, at % PAGE], f[at // PAGE, :, at % PAGE], s["lut"]).to(torch.bfloat16)
    return got


def _plain_rope(s):
    q = _plain_norm_rope(s, s["q"], s["w_q"], torch.float32)
    # keys in 64 bits: which code a key next to a border gets may not depend on the order of a sum
    k = _plain_norm_rope(s, s["k"], s["w_k"], torch.float64).to(torch.bfloat16)
    if s["cache"] == "e4m3":
        q = _to_e4m3(q.to(torch.bfloat16), 1.0)
    else:
        q = q.to(torch.bfloat16)
    if s["cache"] == "none":
        return {"q": q, "k": k}
    if s["cache"] == "kv4":
        return {"q": q, "k_rows": _plain_append_kv4(s, k, s["kc"], s["k_scale"]), "v_rows": _plain_append_kv4(s, s["v"], s["vc"], s["v_scale"])}
    v = s["v"]
    if s["cache"] == "e4m3":
        k, v = _to_e4m3(k, s["k_scale"][:, None]), _to_e4m3(v, s["v_scale"][:, None])
    real = s["slots"] >= 0
    at = s["slots"][real].long()
    s["kc"].view(_bits(k))[at // PAGE, :, at % PAGE] = k.view(_bits(k))[real]
    s["vc"].view(_bits(v))[at // PAGE, :, at % PAGE] = v.view(_bits(v))[real]
    return {"q": q, "k_cache": s["kc"], "v_cache": s["vc"]}


def _bits(x):
    return torch.uint8 if x.dtype == torch.float8_e4m3fn else torch.int16


def _gathered(s, cache, pages):
    """fp32 values of pages [..., n] for every head: [..., heads, n * 128, 128]."""
    c, f = _parts(cache)
    v = _values(c[pages], f[pages], s["lut"])                   # [..., n, heads, 128, 128]
    return v.movedim(-3, -4).flatten(-3, -2)


def _softmax(x, mask, v, v_scale):
    x = x.masked_fill(~mask, -math.inf)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == -math.inf, 0, m))
    total = e.sum(-1, keepdim=True)
    o = (e @ v) * v_scale / torch.where(total == 0, 1, total)
    return o, (m + torch.log(total))[..., 0]


def _plain_kv4(s):
    hq, hk = s["hq"], s["hk"]
    g = hq // hk
    one = torch.ones(hk, device="cuda")
    ks, vs = s["scales"].get("k_scale", one), s["scales"].get("v_scale", one)
    T = s["q"].shape[0]
    if s["topk"]:
        blocks = s["blocks"].long()                             # [T, hk, topk]
        phys = s["table"].long()[torch.where(blocks >= 0, s["start"][:, None, None] + blocks, 0)]
        head = torch.arange(hk, device="cuda")[None, :, None]
        kc, kf = _parts(s["k"])
        vc, vf = _parts(s["v"])
        k = _values(kc[phys, head], kf[phys, head], s["lut"]).flatten(2, 3)
        v = _values(vc[phys, head], vf[phys, head], s["lut"]).flatten(2, 3)
        key = (blocks[..., None] * PAGE + torch.arange(PAGE, device="cuda")).flatten(2)
        mask = (blocks >= 0).repeat_interleave(PAGE, 2) & (key < s["seen"][:, None, None])
        v = v.masked_fill(~mask[..., None], 0)
        x = s["q"].float().view(T, hk, g, D) @ k.transpose(-1, -2) * (ks[:, None, None] * D ** -0.5)
        o, lse = _softmax(x, mask[:, :, None], v, vs[:, None, None])
        return {"out": o.flatten(1, 2).to(torch.bfloat16), "lse": lse.flatten(1, 2)}
    k, v = _gathered(s, s["k"], s["pages"]), _gathered(s, s["v"], s["pages"])      # [B, hk, keys, D]
    key = torch.arange(k.shape[2], device="cuda")
    v = v.masked_fill((key[None] >= s["len_k"][:, None])[:, None, :, None], 0)
    n = s["tok"].shape[1]
    q = s["q"].float()[s["tok"]].view(-1, n, hk, g, D).permute(0, 2, 3, 1, 4).flatten(2, 3)      # [B, hk, g * n, D]
    x = q @ k.transpose(-1, -2) * (ks[:, None, None] * D ** -0.5)
    last = torch.arange(n, device="cuda")[None] + (s["len_k"] - s["len_q"])[:, None]             # [B, n]
    last = torch.minimum(last, s["len_k"][:, None] - 1).repeat(1, g)
    o, lse = _softmax(x, (key[None, None] <= last[..., None])[:, None], v, vs[:, None, None])
    o = o.unflatten(2, (g, n)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    lse = lse.unflatten(2, (g, n)).permute(0, 3, 1, 2).flatten(2, 3)
    return {"out": o[s["ok"]].to(torch.bfloat16), "lse": lse[s["ok"]]}


# ----------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------

def _own_tables(msa, s):
    t = msa.paged_kv_tables(s["ql"], s["kl"], s["table"], s["held"], s["free"], s["num_free"], max_total_q=s["total_q"],
                            max_total_pages=s["pages"])
    return {**{k: t[k] for k in ("kv_indices", "kv_page_indptr", "slot_map", "positions", "num_held", "num_free")}, "block_table": s["table"]}


def _own_rope(msa, s):
    if s["cache"] == "none":
        q, k = msa.qk_norm_rope(s["q"], s["k"], s["pos"], s["rope"], q_weight=s["w_q"], k_weight=s["w_k"])
        return {"q": q, "k": k}
    q_out = torch.empty(s["q"].shape, dtype=torch.float8_e4m3fn, device="cuda") if s["cache"] == "e4m3" else None
    q, _ = msa.qk_norm_rope(s["q"], s["k"], s["pos"], s["rope"], v=s["v"], q_weight=s["w_q"], k_weight=s["w_k"], q_out=q_out,
                            k_cache=s["kc"], v_cache=s["vc"], slot_map=s["slots"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    if s["cache"] == "kv4":
        return {"q": q, "k_rows": msa.kv4_read(s["kc"], s["slots"]), "v_rows": msa.kv4_read(s["vc"], s["slots"])}
    return {"q": q, "k_cache": s["kc"], "v_cache": s["vc"]}


def _own_kv4(msa, s):
    more = dict(kv_block_indexes=s["blocks"]) if s["topk"] else {}
    msa.fmha_sail(s["q"], s["k"], s["v"], s["plan"], kv_indices=s["table"], out=s["out"], lse=s["lse"], **more, **s["scales"])
    return {"out": s["out"], "lse": s["lse"]}


def run(state):
    if own:
        return {"tables": _own_tables, "rope": _own_rope, "kv4": _own_kv4}[state["family"]](_msa(), state)
    return {"tables": _plain_tables, "rope": _plain_rope, "kv4": _plain_kv4}[state["family"]](state)


# ----------------------------------------------------------------------------------------------
# the definition in 64 bits
# ----------------------------------------------------------------------------------------------

_STEPS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_rotated(case, s, x, w):
    z = x.double()
    z = z / torch.sqrt(z.pow(2).sum(-1) / D + 1e-6)[..., None]
    if w is not None:
        z = z * w.double()
    half = case["rotary"] // 2
    out = z.clone()
    pair = 0
    for axis, count in enumerate(s["sections"]):
        for _ in range(count):
            i, j = (pair, pair + half) if case["style"] == "half" else (2 * pair, 2 * pair + 1)
            t = (s["pos"][axis].double() * float(s["inv_freq"][pair]))[:, None]
            out[..., i] = z[..., i] * t.cos() - z[..., j] * t.sin()
            out[..., j] = z[..., i] * t.sin() + z[..., j] * t.cos()
            pair += 1
    return out


def _exact_held(x, scale):
    """What 4 bits hold of bf16 x: each value goes to the nearest step, ties to the even code."""
    y = (x.double() / scale.double()[:, None]).reshape(*x.shape[:2], 8, 16)
    f = (y.abs().amax(-1) / 6).clamp(2.0 ** -9, 448.0).float().to(torch.float8_e4m3fn).double()[..., None]
    m = y.abs() / f
    best = torch.zeros_like(m)
    for code in range(1, 8):
        edge = (_STEPS[code] + _STEPS[code - 1]) / 2
        best = torch.where((m > edge) | ((m == edge) if code % 2 == 0 else (m > edge)), _STEPS[code], best)
    return (best * f * torch.where(y < 0, -1.0, 1.0)).reshape(x.shape)


def _exact_rope(case, s):
    k = _exact_rotated(case, s, s["k"], s["w_k"])
    q = _exact_rotated(case, s, s["q"], s["w_q"])
    if case["cache"] == "none":
        return {"q": q, "k": k}
    k = k.to(torch.bfloat16)                                    # a cache takes keys that were rounded to bf16
    real = (s["slots"] >= 0)[:, None, None]
    if case["cache"] == "kv4":
        return {"q": q, "k_rows": torch.where(real, _exact_held(k, s["k_scale"]), 0.0), "v_rows": torch.where(real, _exact_held(s["v"], s["v_scale"]), 0.0)}
    rows = {}
    for name, x, scale in (("k", k, s["k_scale"]), ("v", s["v"], s["v_scale"])):
        c = torch.zeros(s["kc"].shape, dtype=torch.float64, device="cuda")
        at = s["slots"][s["slots"] >= 0].long()
        y = x.double() if scale is None else x.double() / scale.double()[:, None]
        c[at // PAGE, :, at % PAGE] = y[s["slots"] >= 0]
        rows[name + "_cache"] = c
    return {"q": q, **rows}


def _exact_pages(c, pages, head):
    """fp64 [keys, 128] of the listed pages of one head."""
    raw = c.view(c.shape[0], c.shape[1], -1)[pages, head]
    b = raw[:, :PAGE * 64].reshape(-1, 64).long()
    f = raw[:, PAGE * 64:].reshape(-1, 8).view(torch.float8_e4m3fn).double()
    n = torch.empty(b.shape[0], D, dtype=torch.long, device=b.device)
    n[:, 0::2], n[:, 1::2] = b % 16, b // 16
    step = torch.tensor(_STEPS, dtype=torch.float64, device=b.device)[n % 8]
    return torch.where(n >= 8, -step, step) * f.repeat_interleave(16, 1)


def _exact_kv4(case, s):
    hq, hk, ql, kl = s["hq"], s["hk"], s["ql"], s["kl"]
    if s["topk"] and sum(ql) * hk > 1024 or hq * sum(a * b for a, b in zip(ql, kl)) > MOST_PAIRS:
        return None
    g = hq // hk
    out = torch.zeros(sum(ql), hq, D, dtype=torch.float64, device="cuda")
    lse = torch.full((sum(ql), hq), -math.inf, dtype=torch.float64, device="cuda")
    tok = page0 = 0
    for n, keys in zip(ql, kl):
        table = s["table"][page0:page0 + -(-keys // PAGE)].long()
        for h in range(hk):
            ks = float(s["scales"]["k_scale"][h]) if s["scales"] else 1.0
            vs = float(s["scales"]["v_scale"][h]) if s["scales"] else 1.0
            rows = [(tok, tok + n, None)] if not s["topk"] else [(t, t + 1, s["blocks"][t, h]) for t in range(tok, tok + n)]
            for a, b, picked in rows:
                pages = torch.arange(len(table), device="cuda") if picked is None else picked[picked >= 0].long()
                at = (pages[:, None] * PAGE + torch.arange(PAGE, device="cuda")).reshape(-1)
                k, v = _exact_pages(s["k"], table[pages], h)[at < keys], _exact_pages(s["v"], table[pages], h)[at < keys]
                at = at[at < keys]
                pos = torch.arange(keys - n + a - tok, keys - n + b - tok, device="cuda")
                for j in range(h * g, h * g + g):
                    x = s["q"][a:b, j].double() @ k.T * (ks / math.sqrt(D))
                    x = torch.where(at[None] <= pos[:, None], x, -math.inf)
                    total = torch.logsumexp(x, 1)
                    lse[a:b, j] = total
                    out[a:b, j] = torch.where(torch.isinf(total)[:, None], 0.0, torch.exp(x - total[:, None])) @ v * vs
        tok, page0 = tok + n, page0 + len(table)
    return {"out": out, "lse": lse}


def exact(case, seed):
    if case["family"] == "tables":
        return None
    s = prepare(case, seed)
    return (_exact_rope if case["family"] == "rope" else _exact_kv4)(case, s)


# ----------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------

def work(case):
    if case["family"] == "tables":
        ql, kv = _table_lens(case)
        pages = sum(_pages(kv))
        new = pages - sum(_pages([n - t for t, n in zip(ql, kv)]))
        return {"bytes": 4 * (5 * len(kv) + 2 * pages + 2 * new + 2 * sum(ql)), "flops": 0}
    hq, hk = case["hq"], case["hk"]
    if case["family"] == "rope":
        T = case["tokens"]
        row = {"none": 2 * D, "bf16": 2 * D, "e4m3": D, "kv4": 72}[case["cache"]]
        read = 2 * D * (hq + hk * (1 if case["cache"] == "none" else 2))
        wrote = D * hq * (1 if case["cache"] == "e4m3" else 2) + row * hk * (1 if case["cache"] == "none" else 2)
        back = 2 * hk * (row + 2 * D) if case["cache"] == "kv4" else 0
        return {"bytes": T * (read + wrote + back + 4 * case["axes"]), "flops": T * (hq + hk) * 10 * D}
    ql, kl = lengths(case["q"]), lengths(case["kv"])
    topk = case["topk"]
    rows = sum(ql) * hq * (4 * D + 4)
    if topk:                                                    # pages that a sequence's tokens can select, each once
        keys = sum(min(k, q * topk * PAGE) for q, k in zip(ql, kl))
        pairs = sum(min(k - q + 1 + i, topk * PAGE) for q, k in zip(ql, kl) for i in range(q))
        return {"bytes": keys * hk * 144 + rows, "flops": pairs * hq * 4 * D}
    return {"bytes": sum(kl) * hk * 144 + rows, "flops": sum(q * k - q * (q - 1) / 2 for q, k in zip(ql, kl)) * hq * 4 * D}


if __name__ == "__main__":
    for seed in range(12):
        print(draw(random.Random(seed)))
