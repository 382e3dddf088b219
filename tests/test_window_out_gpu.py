"""Results of windowed attention written into views: the same ones are taken whether a plan cuts its items or not."""
import pytest
import torch

from test_window_gpu import BF, E4, Case

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("types", [(BF, BF), (E4, E4)])
def test_views(splits, types):
    import msa_for_sail as msa
    c = Case([1, 2, 1], [900, 700, 0], 8, 2, 300, 4, "hnd", 128, *types)
    plan = c.plan(num_kv_splits=splits)
    assert plan[3]["num_kv_splits"] == splits
    T, want = c.q.shape[0], None
    for dtype, lead, pad, taken in [(BF, 0, 0, True), (BF, 8, 8, True), (BF, 4, 4, False), (BF, 0, 4, False), (BF, 1, 7, False),
                                    (torch.float32, 0, 0, True), (torch.float32, 4, 4, True), (torch.float32, 2, 2, True), (torch.float32, 1, 0, True)]:
        wide = torch.full((T, 8, lead + 128 + pad), 5.0, dtype=dtype, device=DEV)
        out = wide[..., lead:lead + 128]
        if not taken:
            with pytest.raises(Exception):
                msa.fmha_sail(c.q, c.k, c.v, plan, kv_indices=c.table, out=out)
            torch.cuda.synchronize()
            assert (wide == 5).all()
            continue
        got, _ = msa.fmha_sail(c.q, c.k, c.v, plan, kv_indices=c.table, out=out)
        assert got is out and (wide[..., :lead] == 5).all() and (wide[..., lead + 128:] == 5).all()
        want = out.float() if want is None else want
        assert (out.float() - want).abs().max() <= 2 ** -8 * want.abs().max()
