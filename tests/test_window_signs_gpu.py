"""Factors of the scores of any sign, one for each KV head, on every kernel that has windows."""
import pytest
import torch

from test_window_gpu import BF, E4, Case, kernels  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("types", [(BF, BF), (BF, E4), (E4, E4)])
@pytest.mark.parametrize("tokens,hq,hk", [(1, 12, 3), (1, 48, 3), (3, 48, 3), (7, 48, 3), (150, 6, 3), (300, 3, 3)])
@pytest.mark.parametrize("window,sinks", [(100, 4), (300, 40), (3000, 0), (1, 0)])
def test_a_factor_for_each_head(kernels, types, tokens, hq, hk, window, sinks):  # noqa: F811
    c = Case([tokens] * 2, [900, tokens + 5], hq, hk, window, sinks, "hnd", 128, *types)
    c.scales = dict(k_scale=torch.tensor([-1.25, 0.0, 0.75], device="cuda"), v_scale=torch.tensor([1.0, -2.0, 0.5], device="cuda"))
    c.check()
