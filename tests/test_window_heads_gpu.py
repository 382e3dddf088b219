"""A plan made without num_kv_heads takes the cache's, with a window as without one."""
import pytest
import torch

from test_window_gpu import BF, E4, Case, kernels  # noqa: F401

pytestmark = pytest.mark.gpu


def _i32(v):
    return torch.tensor(v, dtype=torch.int32)


@pytest.mark.parametrize("types", [(BF, BF), (BF, E4), (E4, E4)])
@pytest.mark.parametrize("tokens", [1, 4, 40, 200])
@pytest.mark.parametrize("splits", [-1, 2])
def test_heads_of_the_cache(kernels, types, tokens, splits):  # noqa: F811
    import msa_for_sail as msa
    c = Case([tokens] * 2, [700, 1100], 8, 2, 300, 4, "hnd", 128, *types)
    plan = msa.fmha_sail_plan(_i32(c.ql), _i32(c.kl), 8, page_size=128, window_size=300, num_sink_tokens=4, num_kv_splits=splits)
    c.check(plan=plan)
    all_heads = Case([tokens] * 2, [700, 1100], 8, 8, 300, 4, "hnd", 128, *types)
    all_heads.check(plan=plan)                                  # one plan, two caches
    three = Case([tokens] * 2, [700, 1100], 9, 3, 300, 4, "hnd", 128, *types)
    with pytest.raises(ValueError, match="head"):
        msa.fmha_sail(three.q, three.k, three.v, plan, kv_indices=three.table)
    given = msa.fmha_sail_plan(_i32(c.ql), _i32(c.kl), 8, num_kv_heads=8, page_size=128, window_size=300, num_sink_tokens=4)
    with pytest.raises(ValueError, match="head"):
        msa.fmha_sail(c.q, c.k, c.v, given, kv_indices=c.table)
