"""Windowed attention whose rows have one key, or a few, far above all others: what thousands of small weights have together is not lost.

Weights over an e4m3 cache are pairs of e4m3 values: each is within 2^-8 of itself, and all that its small values lose is at most 1.5 * 2^-8 of a row's sum."""
import math

import pytest
import torch

import window_ref as ref
from test_window_gpu import BF, E4, SCALE, kernels  # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(v, device=DEV):
    return torch.tensor(v, dtype=torch.int32, device=device)


class Peaks:
    """Element 0 of every query is 16, so a key with `a` there has 1.414 a nats more than one with 0; a and 16 are exact in every type."""

    def __init__(self, tokens, kl, hq, hk, types, peaks, paged=True, noise=0.03, v=None, seed=3):
        """peaks: {place of a key, from the end if negative: a}"""
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.tokens, self.kl, self.hq, self.hk = tokens, kl, hq, hk
        self.q = torch.randn(tokens * len(kl), hq, 128, device=DEV, generator=g)
        self.q[..., 0] = 16
        self.q = self.q.to(types[0])
        self.ks, self.vs = [], []
        for n in kl:
            k = torch.randn(n, hk, 128, device=DEV, generator=g) * noise
            k[..., 0] = 0
            for at, a in peaks.items():
                k[at, :, 0] = a
            self.ks.append(k.to(types[1]))
            v_ = 1 + 0.25 * torch.rand(n, hk, 128, device=DEV, generator=g) if v is None else v(n, hk, g)
            self.vs.append(v_.to(types[1]))
        self.table, self.page_size = None, -1
        if not paged:
            self.k, self.v = torch.cat(self.ks), torch.cat(self.vs)
            return
        self.page_size = 128
        need = [-(-n // 128) for n in kl]
        order = torch.randperm(sum(need), generator=torch.Generator().manual_seed(seed))
        self.k, self.v = (torch.zeros(sum(need), hk, 128, 128, device=DEV).to(types[1]) for _ in range(2))
        self.table, at = order.int().to(DEV), 0
        for k, v_, n in zip(self.ks, self.vs, kl):
            for i in range(-(-n // 128)):
                rows = slice(128 * i, min(n, 128 * (i + 1)))
                for c, x in ((self.k, k), (self.v, v_)):
                    c[int(order[at])].transpose(0, 1)[:rows.stop - rows.start] = x[rows]
                at += 1

    def check(self, window, sinks, scale=SCALE, **kw):
        import msa_for_sail as msa
        from msa_for_sail import api
        ql = [self.tokens] * len(self.kl)
        plan = msa.fmha_sail_plan(_i32(ql, "cpu"), _i32(self.kl, "cpu"), self.hq, num_kv_heads=self.hk, page_size=self.page_size, window_size=window,
                                  num_sink_tokens=sinks, **kw)
        lse = torch.empty(self.q.shape[:2], device=DEV)
        out, _ = msa.fmha_sail(self.q, self.k, self.v, plan, kv_indices=self.table, lse=lse, sm_scale=scale)
        assert api.last_status() == 0
        places = [torch.arange(self.tokens) + n - self.tokens for n in self.kl]
        o, mean, want_lse, dots = ref.attention(self.q, self.ks, self.vs, places, window, sinks, scale)
        # element 0 is exact in pairs of e4m3 values too: the other elements' products are what queries' rounding is multiplied by
        rest = self.q.double().cpu()
        rest[..., 0] = 0
        _, _, _, dots = ref.attention(rest, self.ks, self.vs, places, window, sinks, scale)
        x_err = (2 ** -8 if self.q.dtype != self.k.dtype else 0.0) * dots
        most = max(float(v.double().abs().max()) for v in self.vs)
        err = (out.double().cpu() - o).abs()
        # each weight, the row's sum of what small ones lose, the result's last bit
        lost = 1.5 * 2 ** -8 if self.k.dtype == E4 else 0.0
        tol = (torch.expm1(x_err) + 2 ** -8 + 2 ** -12) * mean + lost * most + 2 ** -8 * o.abs() + 1e-6
        assert torch.isfinite(out).all()
        assert (err <= tol).all(), f"{(err / tol).max():.2f} of the tolerance, {(err / o.abs()).max():.4f} relative"
        worst = (lse.double().cpu() - want_lse).abs() - x_err[..., 0] - 2 ** -8 - 2 ** -10 - 2 ** -20 * want_lse.abs()
        assert worst.max() <= 0
        return out


TYPES = [(BF, E4), (E4, E4)]
# one row of a KV head to 128, in items that clusters share and in more of them, prompts
SHAPES = [(1, 2, 8, 2), (1, 39, 16, 2), (1, 2, 16, 1), (1, 39, 32, 2), (3, 2, 16, 2), (4, 12, 16, 2), (7, 1, 16, 1), (130, 1, 4, 2), (300, 1, 2, 1)]


@pytest.mark.parametrize("tokens,batch,hq,hk", SHAPES)
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("window,a", [(4096, 6.5), (4096, 7), (8192, 10)])
def test_a_sink(kernels, tokens, batch, hq, hk, types, window, a):  # noqa: F811
    kl = [9000 + 61 * i if i < 1 else 4200 + i for i in range(batch)]
    Peaks(tokens, kl, hq, hk, types, {0: a}, paged=window == 4096).check(window, 4)


@pytest.mark.parametrize("tokens,batch,hq,hk", SHAPES)
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("peaks", [{-1: 7}, {0: 4.5, -1000: 9, -1: 14}, {-700: 60}, {-3000: 60, -2000: 120}, {-2600: 26, -2500: 20, -2400: 14, -1000: 7}], ids=str)
def test_peaks_anywhere(kernels, tokens, batch, hq, hk, types, peaks):  # noqa: F811
    kl = [3200 + 61 * i for i in range(batch)]
    Peaks(tokens, kl, hq, hk, types, peaks, paged=tokens != 3).check(4096, 4)


@pytest.mark.parametrize("tokens,batch,hq,hk", SHAPES)
@pytest.mark.parametrize("types", [(E4, E4), (BF, BF)])                    # (the bound for rounded queries says nothing here)
@pytest.mark.parametrize("noise,splits", [(1.0, -1), (2.0, 3), (4.0, -1)])
def test_scores_of_any_spread(tokens, batch, hq, hk, types, noise, splits):
    """Scores with a standard deviation of one to four nats: maxima that rise and fall from tile to tile."""
    kl = [1500 + 61 * i for i in range(batch)]
    Peaks(tokens, kl, hq, hk, types, {0: 3}, noise=noise, v=lambda n, h, g: torch.randn(n, h, 128, device=DEV, generator=g)).check(1000, 4, num_kv_splits=splits)


@pytest.mark.parametrize("tokens,batch,hq,hk", SHAPES)
@pytest.mark.parametrize("types", [*TYPES, (BF, BF)])
def test_a_sink_that_holds_no_value(tokens, batch, hq, hk, types):
    """Values of the heavy key are 0, as they often are: the result is the tail's."""
    def v(n, h, g):
        x = 1 + 0.25 * torch.rand(n, h, 128, device=DEV, generator=g)
        x[0] = 0
        return x
    Peaks(tokens, [5000] * batch, hq, hk, types, {0: 7}, v=v).check(4096, 1)
