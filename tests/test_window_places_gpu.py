"""Windows of queries at the last places that fit 32 bits."""
import pytest
import torch

from test_window_gpu import BF, E4, Case, _device_plan, kernels  # noqa: F401

pytestmark = pytest.mark.gpu
LAST = 2 ** 31 - 1


@pytest.mark.parametrize("types", [(BF, BF), (E4, E4), (BF, E4)])
@pytest.mark.parametrize("tokens", [1, 3, 17, 130, 300])
@pytest.mark.parametrize("window,sinks", [(100, 40), (100, 20), (1, 0), (LAST, 40), (LAST - 200, 130), (LAST, LAST)])
def test_the_last_places(kernels, types, tokens, window, sinks):  # noqa: F811
    """A Q tile's rows behind the last token have places past 32 bits."""
    Case([tokens, tokens], [500, 500], 8, 2, window, sinks, "hnd", 128, *types, offsets=[LAST - tokens, 500 - tokens]).check()


@pytest.mark.parametrize("tokens", [1, 40, 300])
@pytest.mark.parametrize("past", [0, 1, 300])
def test_the_last_places_on_the_device(tokens, past):
    """An offset that leads past them is taken as the last one that does not."""
    offsets = [LAST - tokens, 200]
    c = Case([tokens] * 2, [500, 500], 8, 2, 100, 40, offsets=offsets)
    given = torch.tensor([min(LAST, offsets[0] + past), 200], dtype=torch.int32, device="cuda")
    c.check(plan=_device_plan(c, tokens, 2 * tokens, qo_offset=given))
