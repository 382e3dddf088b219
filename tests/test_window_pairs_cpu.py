"""The bound on the mean error of windowed attention over an e4m3 cache tells pairs of e4m3 values from single ones."""
import pytest
import torch

import window_pairs as wp
import window_ref as ref

SCALE = 128 ** -0.5


@pytest.mark.parametrize("window,sinks", [(32, 0), (100, 4), (128, 128), (300, 5), (513, 200), (1000, 4), (2000, 64)])
def test_the_bound_sees_both_second_values(window, sinks):
    g = torch.Generator().manual_seed(window)
    T, G, n = 4, 8, 2500
    q = torch.randn(T, G, 128, generator=g).bfloat16()
    k, v = (torch.randn(n, 1, 128, generator=g).to(torch.float8_e4m3fn) for _ in range(2))
    place = torch.arange(n - T, n)
    j = torch.arange(n)
    see = (j[None] <= place[:, None]) & ((j[None] > place[:, None] - window) | (j[None] < sinks))
    want = ref.attention(q, [k], [v], [place], window, sinks, SCALE)[0]
    error = lambda **kw: wp.rms(wp.model(q, k[:, 0], v[:, 0], see, SCALE, **kw), want)
    assert error() < wp.RMS
    assert error(second_q=False) > 2 * wp.RMS and error(second_p=False) > 2 * wp.RMS
