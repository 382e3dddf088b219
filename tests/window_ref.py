"""Attention with a window and sink tokens in 64 bits, from its definition, and how far a kernel may be from it."""
import math

import torch


def attention(q, ks, vs, places, window, sinks, scale, k_head=None, v_head=None):
    """q [T, Hq, 128]; ks / vs: keys and values of each sequence, [n, Hk, 128]; places: of each sequence's queries, int64 tensors.
    Returns O, the weights' mean of |v| (what a relative error of the weights is multiplied by), the LSE and the largest scale * sum |q k| of a row,
    all fp64 on the CPU."""
    q = q.double().cpu()
    T, hq = q.shape[0], q.shape[1]
    out, mean, dots = (torch.zeros(T, hq, n, dtype=torch.float64) for n in (128, 128, 1))
    lse = torch.full((T, hq), -math.inf, dtype=torch.float64)
    tok = 0
    for k, v, place in zip(ks, vs, places):
        n, keys, hk = len(place), k.shape[0], k.shape[1]
        if n and keys:
            g = hq // hk
            k, v = k.double().cpu(), v.double().cpu()
            if k_head is not None:
                k = k * k_head.double().cpu()[:, None]
            if v_head is not None:
                v = v * v_head.double().cpu()[:, None]
            j = torch.arange(keys)
            see = (j[None] <= place[:, None]) & ((j[None] > place[:, None] - window) | (j[None] < sinks))
            some = see.any(1)
            used = see.any(0)                               # keys that nobody sees may hold anything
            k, v, see = k[used], v[used], see[:, used]
            for h in range(hk):
                x = torch.einsum("tgd,jd->tgj", q[tok:tok + n, h * g:(h + 1) * g], k[:, h]) * scale
                big = torch.einsum("tgd,jd->tgj", q[tok:tok + n, h * g:(h + 1) * g].abs(), k[:, h].abs()) * abs(scale)
                x = x.masked_fill(~see[:, None], -math.inf)
                m = torch.logsumexp(x, 2)
                w = torch.where(some[:, None, None], torch.exp(x - torch.where(m == -math.inf, 0.0, m)[..., None]), 0.0)
                at = (slice(tok, tok + n), slice(h * g, (h + 1) * g))
                out[at], mean[at], lse[at] = w @ v[:, h], w @ v[:, h].abs(), m
                if k.shape[0]:
                    dots[at] = big.masked_fill(~see[:, None], 0).amax(2, keepdim=True)
        tok += n
    return out, mean, lse, dots


def check(out, lse, want, p_step, q_step=0.0, what=""):
    """|error| <= (relative error of a weight) * mean |v| + of their sum * |O| + half a step of the output.

    p_step: half a step of the type that the products take weights in (bf16 2^-8; the generic kernel on e4m3 caches takes f16, 2^-11; pairs of e4m3 values 2^-8).
    q_step: half a step of what queries are rounded to (0: not rounded); a score is off by at most that times scale * sum |q k|, a weight by the
    exponential of it.  2^-12 on top: exponentials (7.5e-5), 32-bit sums of products."""
    o, mean, ref_lse, dots = want
    err = (out.double().cpu() - o).abs()
    x_err = q_step * dots
    w_err = torch.expm1(x_err) + p_step + 2 ** -12
    tol = w_err * (mean + o.abs()) + 2 ** -8 * o.abs() + 1e-6
    assert torch.isfinite(out).all(), f"{what}: not finite"
    assert (err <= tol).all(), f"{what}: {(err / tol).max():.3f} of the tolerance, at {torch.nonzero(err > tol)[:4].tolist()}"
    if lse is not None:
        got = lse.double().cpu()
        assert torch.equal(got == -math.inf, ref_lse == -math.inf), f"{what}: rows that see nothing"
        fin = ref_lse != -math.inf
        worst = ((got - ref_lse).abs() - x_err[..., 0] - p_step - 2 ** -10 - 2 ** -20 * ref_lse.abs().masked_fill(~fin, 0))[fin]
        assert worst.numel() == 0 or worst.max() <= 0, f"{what}: lse off by {worst.max() + p_step:.2g}"
