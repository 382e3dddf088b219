"""How far windowed attention over an e4m3 cache may be from 64 bits in the mean, and a model of the pairs of e4m3 values that it multiplies.

The bound, root of the mean square relative to that of the result: the result's rounding to bf16 is 2^-8 / sqrt(3) at most, of mantissas that are spread
evenly 0.72 of it: 0.0017.  The second value of a pair leaves 2^-8 x at most, in the mean 0.0007 x, of each weight and of each query's element, whose products'
errors are independent and make as much of a score of 1 nat: sqrt(0.0017^2 + 2 * 0.0007^2) = 0.002.  A single e4m3 value has 0.026."""
import torch

RMS = 0.003


def rms(got, want):
    return float((got.double() - want.double()).square().mean().sqrt() / want.double().square().mean().sqrt())


def _e4m3(x):
    return x.float().to(torch.float8_e4m3fn).double()


def _pair(x, second):
    hi = _e4m3(x)
    return hi + _e4m3(x - hi) if second else hi


def model(q, k, v, see, scale, second_q=True, second_p=True):
    """q [T, G, 128] bf16, k and v [n, 128] e4m3, see [T, n]: O of one KV head with queries and weights as pairs, or without the second value of either."""
    q, k, v = q.double(), k.double(), v.double()
    up = torch.exp2(7 - torch.floor(torch.log2(q.abs().amax(-1, keepdim=True))))
    x = torch.einsum("tgd,jd->tgj", _pair(q * up, second_q) / up, k) * scale
    x = x.masked_fill(~see[:, None], -torch.inf)
    w = torch.exp(x - x.amax(-1, keepdim=True)) * 32
    return ((_pair(w, second_p) @ v) / w.sum(-1, keepdim=True)).bfloat16()
