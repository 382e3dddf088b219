"""Mean error of windowed attention over an e4m3 cache: queries in bf16 and weights as pairs of e4m3 values, on every kernel that makes them."""
import pytest
import torch

import window_pairs as wp
from test_window_gpu import BF, E4, Case, kernels  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("types", [(BF, E4), (E4, E4)])
@pytest.mark.parametrize("tokens,batch,hq,hk,layout,page", [(1, 3, 16, 2, "hnd", 128), (1, 3, 16, 1, "ragged", 0), (1, 80, 16, 1, "hnd", 128), (4, 3, 16, 2, "nhd", 64),
                                                            (2, 3, 32, 2, "hnd", 128), (4, 24, 32, 2, "hnd", 128), (8, 3, 32, 2, "nhd", 128), (150, 2, 4, 2, "hnd", 128),
                                                            (300, 1, 2, 1, "ragged", 0)])
@pytest.mark.parametrize("window,sinks", [(32, 0), (100, 4), (513, 200), (1000, 4), (2000, 64)])
def test_mean_error(kernels, types, tokens, batch, hq, hk, layout, page, window, sinks):  # noqa: F811
    import msa_for_sail as msa
    c = Case([tokens] * batch, [1500 + 61 * (i % 7) for i in range(batch)], hq, hk, window, sinks, layout, page, *types)
    out, _ = msa.fmha_sail(c.q, c.k, c.v, c.plan(), kv_indices=c.table)
    error = wp.rms(out.cpu(), c.want()[0])
    assert error < wp.RMS, error
