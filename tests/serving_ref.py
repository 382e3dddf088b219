"""Plain 64-bit forms of the operators around the attention call, for their tests."""
import math

import torch

PAGE, D = 128, 128
STEPS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


# ---- 4-bit cache ----

def kv4_values(cache):
    """uint8 [P, H, 128, 72] -> fp64 [P, H, 128, 128] (a scale per head is not in it)."""
    P, H = cache.shape[:2]
    raw = cache.reshape(P, H, PAGE * 72).cpu()
    codes = raw[:, :, :PAGE * 64].reshape(P, H, PAGE, 64).long()
    scales = raw[:, :, PAGE * 64:].contiguous().view(torch.float8_e4m3fn).double().reshape(P, H, PAGE, 8)
    n = torch.stack([codes & 15, codes >> 4], -1).reshape(P, H, PAGE, D)
    v = STEPS[n & 7] * torch.where(n >= 8, -1.0, 1.0)
    return v * scales.repeat_interleave(16, -1)


def kv4_encode(x, scale):
    """bf16-valued [T, H, 128] and fp32 scale [H] -> code bytes [T, H, 64], scale bytes [T, H, 8].  Divisions in 32 bits, as documented;
    the nearest code by exact comparison, ties to the even one."""
    y = (x.float() / scale.float()[:, None]).reshape(*x.shape[:2], 8, 16)
    s = (y.abs().amax(-1, keepdim=True) / 6)
    s = torch.where(s < 2.0 ** -9, torch.full_like(s, 2.0 ** -9), s).clamp(max=448).to(torch.float8_e4m3fn)
    q = (y / s.float()).double()
    m = q.abs()
    code = torch.zeros(m.shape, dtype=torch.long)
    for c in range(1, 8):
        edge = float(STEPS[c] + STEPS[c - 1]) / 2
        code = torch.where((m > edge) | ((m == edge) & (c % 2 == 0)), torch.tensor(c), code)
    code = (code | (torch.signbit(q).long() << 3)).reshape(*x.shape[:2], D)
    return (code[..., 0::2] | code[..., 1::2] << 4).to(torch.uint8), s.view(torch.uint8)[..., 0]


def kv4_parts(cache):
    """Code bytes [P, H, 128, 64] and scale bytes [P, H, 128, 8] of a cache."""
    P, H = cache.shape[:2]
    raw = cache.cpu().reshape(P, H, PAGE * 72)
    return raw[:, :, :PAGE * 64].reshape(P, H, PAGE, 64), raw[:, :, PAGE * 64:].reshape(P, H, PAGE, 8)


def random_kv4(g, P, H, scale=0.4):
    """Codes and scales of values with an rms of about one."""
    c = torch.randint(0, 256, (P, H, PAGE * 72), generator=g, dtype=torch.uint8)
    c[:, :, PAGE * 64:] = (torch.rand(P, H, PAGE * 8, generator=g) * scale + 0.1).to(torch.float8_e4m3fn).view(torch.uint8)
    return c.view(P, H, PAGE, 72)


# ---- attention ----

def attention(q, k, v, table, indptr, qo_lens, kv_lens, offsets, sm_scale=D ** -0.5, blocks=None, k_scale=None, v_scale=None):
    """fp64 over fp64 page values k, v [P, H, 128, 128].  Returns (out, lse, spread, error of a score) per (token, head): spread is
    sum p |v|, the error 2^-16 sum |q k| of the largest such sum (128 products summed in 32 bits)."""
    T, hq, _ = q.shape
    hk = k.shape[1]
    g = hq // hk
    out = torch.zeros(T, hq, D, dtype=torch.float64)
    spread = torch.zeros(T, hq, D, dtype=torch.float64)
    lse = torch.full((T, hq), -math.inf, dtype=torch.float64)
    score_err = torch.zeros(T, hq, dtype=torch.float64)
    qd = q.double().cpu()
    t = 0
    for b, (n, keys) in enumerate(zip(qo_lens, kv_lens)):
        pages = table[indptr[b]:indptr[b + 1]].long().cpu()
        for i in range(n):
            for h in range(hk):
                if blocks is None:
                    at = torch.arange(keys)
                else:
                    sel = blocks[t, h].long().cpu()
                    sel = sel[(sel >= 0) & (sel < len(pages))]
                    at = (sel[:, None] * PAGE + torch.arange(PAGE)).reshape(-1)
                at = at[(at < keys) & (at <= i + offsets[b])]
                if not len(at):
                    continue
                ks, vs = (1.0 if s is None else float(s[h]) for s in (k_scale, v_scale))
                kk, vv = k[pages[at // PAGE], h, at % PAGE] * ks, v[pages[at // PAGE], h, at % PAGE] * vs
                rows = slice(h * g, h * g + g)
                x = qd[t, rows] @ kk.T * sm_scale
                lse[t, rows] = torch.logsumexp(x, 1)
                p = torch.exp(x - lse[t, rows, None])
                out[t, rows], spread[t, rows] = p @ vv, p @ vv.abs()
                score_err[t, rows] = (qd[t, rows].abs() @ kk.abs().T).amax(1) * abs(sm_scale) * 2.0 ** -16
            t += 1
    return out, lse, spread, score_err


def check_attention(o, lse, ref, p_rounding, what):
    """bf16 results: half a step of the result, the rounding of P and the errors of the scores (twice: in P and in its sum) on sum p |v|."""
    out, want, spread, err = ref
    o, nan = o.double().cpu(), torch.isnan(out)
    assert torch.equal(torch.isnan(o), nan), what
    tol = 2.0 ** -8 * out.abs() + (p_rounding + 2 * err[..., None] + 2.0 ** -18) * spread + 1e-30
    bad = ((o - out).abs() > tol) & ~nan
    assert not bad.any(), f"{what}: {((o - out).abs() / tol)[bad].max():.3g} of the tolerance"
    if lse is not None:
        lse = lse.double().cpu()
        none = torch.isinf(want)
        assert torch.equal(torch.isinf(lse) & (lse < 0), none), what
        tol = err + 2.0 ** -15 + 2.0 ** -21 * want.abs()
        assert ((lse - want).abs() <= tol)[~none & ~torch.isnan(want)].all(), f"{what}: lse off by {(lse - want).abs()[~none].max():.3g}"


# ---- norm and rotation ----

def norm_rope(x, positions, inv_freq, sections, interleaved, weight=None, eps=1e-6, norm=True):
    """fp64 of x [T, H, 128]; also the sum of the magnitudes that each result is made of."""
    z = x.double().cpu()
    if norm:
        z = z / torch.sqrt(z.square().mean(-1, keepdim=True) + eps)
        if weight is not None:
            z = z * weight.double().cpu()
    out, size = z.clone(), z.abs()
    half = len(inv_freq)
    pair = 0
    for axis, count in enumerate(sections):
        for _ in range(count):
            i, j = (2 * pair, 2 * pair + 1) if interleaved else (pair, pair + half)
            t = (positions[axis].double().cpu() * float(inv_freq[pair]))[:, None]
            out[..., i] = z[..., i] * t.cos() - z[..., j] * t.sin()
            out[..., j] = z[..., j] * t.cos() + z[..., i] * t.sin()
            size[..., i] = size[..., j] = z[..., i].abs() + z[..., j].abs()
            pair += 1
    return out, size


# ---- page tables ----

def page_tables(qo_lens, kv_lens, table, held, free, num_free, max_q, max_pages, page_size):
    """Lists in, lists out; changes `table`."""
    width = len(table[0]) if table else 0
    flat, indptr, slots, pos, new_held, missing = [], [0], [], [], [], 0
    stack = list(free[:num_free]) if free is not None else []
    left = len(stack)
    for b, (n, keys) in enumerate(zip(qo_lens, kv_lens)):
        need = -(-keys // page_size)
        have = need if held is None else min(held[b], width)
        got = 0
        for p in range(have, min(need, width)):
            if left > 0:
                left -= 1
                table[b][p] = stack[left]
                got += 1
            else:
                table[b][p] = -1
                missing += 1
        missing += max(0, need - width)
        new_held.append(max(0 if held is None else held[b], have + got))
        real = [table[b][p] if p < width else -1 for p in range(need)]
        flat += [max(p, 0) for p in real]
        indptr.append(indptr[-1] + need)
        for i in range(n):
            at = keys - n + i
            page = real[at // page_size] if at >= 0 else -1
            slots.append(page * page_size + at % page_size if page >= 0 else -1)
            pos.append(max(at, 0))
    missing += max(0, len(flat) - max_pages) + max(0, len(slots) - max_q)
    flat = (flat + [-1] * max_pages)[:max_pages]
    return (flat, indptr, (slots + [-1] * max_q)[:max_q], (pos + [0] * max_q)[:max_q], new_held, left, missing)
