"""msa_lse_merge_many against the merge in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _run(po, pl, spr=None, out_dtype=torch.float32, scale=1.0, pad=0, lse=True):
    from msa_for_sail import _lib
    S, T, H, _ = po.shape
    out = torch.full((T, H, 128 + pad), 7.0, dtype=out_dtype, device="cuda")
    l = torch.full((T, H), 7.0, device="cuda") if lse else None
    rc = _lib.lib.msa_lse_merge_many(po.data_ptr(), pl.data_ptr(), None if spr is None else spr.data_ptr(), out.data_ptr(),
                                     _lib.MSA_DT_F32 if out_dtype == torch.float32 else _lib.MSA_DT_BF16, None if l is None else l.data_ptr(),
                                     S, T, H, out.stride(0), out.stride(1), scale, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    assert (out[..., 128:] == 7.0).all()
    return out[..., :128], l


def _want(po, pl, spr, scale):
    S = po.shape[0]
    pl, po = pl.double(), po.double()
    if spr is not None:
        pl = torch.where(torch.arange(S, device="cuda")[:, None, None] < spr[None, :, None], pl, -torch.inf)
    w = torch.exp(pl - pl.amax(0).clamp(min=-1e300))
    po = torch.where(w[..., None] > 0, po, 0.0)
    sw = w.sum(0)
    out = torch.where(sw[..., None] > 0, (w[..., None] * po).sum(0) / sw[..., None], 0.0) * scale
    spread = torch.where(sw[..., None] > 0, (w[..., None] * po.abs()).sum(0) / sw[..., None], 0.0) * scale
    return out, spread, torch.logsumexp(pl, 0)


@pytest.mark.parametrize("S", [1, 2, 5, 31, 32, 33, 128, 129, 300])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_against_64_bits(S, out_dtype):
    g = torch.Generator("cuda").manual_seed(S)
    T, H = 3, 5
    po = torch.randn(S, T, H, 128, device="cuda", generator=g)
    pl = 3 * torch.randn(S, T, H, device="cuda", generator=g)
    empty = torch.rand(S, T, H, device="cuda", generator=g) < 0.3
    pl[empty] = -torch.inf
    po[empty] = torch.nan                                       # the partial of an empty split is not looked at
    pl[:, 1, 2] = -torch.inf                                    # a row without a key
    spr = torch.tensor([S, max(1, S // 2), 1], dtype=torch.int32, device="cuda")
    for limit in (None, spr):
        out, lse = _run(po, pl, limit, out_dtype, 0.5, pad=8)
        want, spread, wl = _want(po, pl, limit, 0.5)
        # a weight: exponent of a difference of at most 30 (2^-24 of it, twice), the function's 2 ulp + 2^-21 of the argument; sums of S + 4
        step = 2.0 ** -8 if out_dtype == torch.bfloat16 else 2.0 ** -24
        tol = step * want.abs() + (2 * (30 * 2.0 ** -23 + 2.0 ** -21) + (S + 8) * 2.0 ** -24) * spread + 1e-30
        assert ((out.double() - want).abs() <= tol).all()
        got = lse.double()
        assert torch.equal(torch.isinf(got), torch.isinf(wl)) and (out[1, 2] == 0).all()
        ok = ~torch.isinf(wl)
        assert ((got - wl).abs()[ok] <= 2.0 ** -17 + 2.0 ** -22 * wl.abs()[ok]).all()


@pytest.mark.parametrize("S,T,H", [(1, 1100, 1), (3, 300, 7), (17, 600, 2), (33, 1025, 1), (100, 20, 64)])
def test_many_rows(S, T, H):
    g = torch.Generator("cuda").manual_seed(S)
    po, pl = torch.randn(S, T, H, 128, device="cuda", generator=g), 3 * torch.randn(S, T, H, device="cuda", generator=g)
    empty = torch.rand(S, T, H, device="cuda", generator=g) < 0.3
    pl[empty], po[empty] = -torch.inf, torch.nan
    pl[:, 1] = -torch.inf
    spr = torch.randint(1, S + 1, (T,), device="cuda", generator=g, dtype=torch.int32)
    spr[3] = 0                                                  # a padded row
    for limit in (None, spr):
        out, lse = _run(po, pl, limit)
        want, spread, wl = _want(po, pl, limit, 1.0)
        tol = 2.0 ** -24 * want.abs() + (2 * (30 * 2.0 ** -23 + 2.0 ** -21) + (S + 8) * 2.0 ** -24) * spread + 1e-30
        assert ((out.double() - want).abs() <= tol).all()
        ok = ~torch.isinf(wl)
        assert torch.equal(torch.isinf(lse), ~ok) and (out[1] == 0).all()
        assert ((lse.double() - wl).abs()[ok] <= 2.0 ** -17 + 2.0 ** -22 * wl.abs()[ok]).all()


def test_not_a_number_and_large_differences():
    po = torch.ones(40, 1, 3, 128, device="cuda")
    pl = torch.zeros(40, 1, 3, device="cuda")
    pl[7, 0, 1] = torch.nan
    pl[9, 0, 2] = 1e30
    po[9, 0, 2] = 5.0
    out, lse = _run(po, pl)
    assert (out[0, 0] == 1).all() and torch.isnan(out[0, 1]).all() and torch.isnan(lse[0, 1]) and (out[0, 2] == 5).all()
    assert float(lse[0, 2]) == pytest.approx(1e30)
    out, lse = _run(po[5:15].contiguous(), pl[5:15].contiguous())    # few splits: the other kernel
    assert (out[0, 0] == 1).all() and torch.isnan(out[0, 1]).all() and torch.isnan(lse[0, 1]) and (out[0, 2] == 5).all()


def test_runs_are_repeatable_and_lse_is_optional():
    po, pl = torch.randn(129, 4, 16, 128, device="cuda"), torch.randn(129, 4, 16, device="cuda")
    first = _run(po, pl)[0]
    for _ in range(5):
        assert torch.equal(_run(po, pl, lse=False)[0], first)
