"""The activations of the feed-forward operators on the GPU where they are small, relative to themselves.  Against 64 bits, bounds
fixed from the arithmetic before the first run; u is 2^-24, half a step of fp32."""
import math

import pytest
import torch

from clpeak_amd import capi
from test_gpu_ffn import ACTS, E, act64, dv, tiled  # noqa: F401

pytestmark = pytest.mark.gpu


def tail_off(act, x):
    """Relative error of the fp32 activation of an exact argument, in u.  silu: 2^(-x log2 e) has an argument rounded twice
    (2 |x|), and with the sum, 1/x (an ulp, 2 u) and the product 8.  The tanh form of gelu: the same of 2 y, which is off by 7
    roundings itself.  The erf form: t = 1 / (1 + c |x|) is off by 3, twice as much of t P(t); its polynomial of eighth degree
    by 8; exp(-x^2 / 2) by 2 x^2 and an ulp; three products; 20 + 2 x^2."""
    if act == capi.GLU_SILU:
        return (8 + 2 * x.abs()) * E
    if act == capi.GLU_GELU_TANH:
        return (8 + 8 * (math.sqrt(8 / math.pi) * (x + 0.044715 * x ** 3)).abs()) * E
    if act == capi.GLU_GELU:
        return (20 + 2 * x * x) * E
    return torch.zeros_like(x)


@pytest.mark.parametrize("act", ACTS)
def test_activations_keep_their_bits_where_they_are_small(tiled, act):
    """fp32 outputs of the int8 gated projection.  G is a whole number n, |n| <= 16129, times 2^-10, 2^-9 or 2^-13, exactly,
    and U is 1: H is the activation, at arguments from 0 to 31 on both sides, and has to be right relative to itself."""
    dv = tiled
    K, F, steps = 128, 3, (2.0 ** -10, 2.0 ** -9, 2.0 ** -13)
    n = torch.arange(-16129, 16130, 7)
    q = torch.div(n, 127, rounding_mode="trunc")
    M = n.numel()
    a = torch.zeros(M, K, dtype=torch.int8)
    a[:, 0], a[:, 1], a[:, 2] = q.to(torch.int8), (n - 127 * q).to(torch.int8), 1
    bg, bu = torch.zeros(F, K, dtype=torch.int8), torch.zeros(F, K, dtype=torch.int8)
    bg[:, 0], bg[:, 1], bu[:, 2] = 127, 1, 1
    a, bg, bu = a.cuda(), bg.cuda(), bu.cuda()
    sa, su, sg = torch.ones(M, device="cuda"), torch.ones(F, device="cuda"), torch.tensor(steps, device="cuda")
    h = torch.empty(M, F, device="cuda")
    dv.glu_i8(act, a, K, bg, bu, K, sa, sg, su, capi.TYPE_F32, h, F, M, F, K)
    x = n.double().cuda()[:, None] * torch.tensor(steps, dtype=torch.float64, device="cuda")
    ref = act64(act, x)
    off = 2 * tail_off(act, x) * ref.abs() + E * ref.abs()
    bad = ((h.double() - ref).abs() > off) & (ref.abs() > 2.0 ** -100)      # (smaller: an exponential that small is 0 on the way)
    assert not bool(bad.any()), (int(bad.sum()), x[bad][:3].tolist(), h[bad][:3].tolist(), ref[bad][:3].tolist())
    assert bool((h[ref.abs() <= 2.0 ** -100].abs() <= 2.0 ** -99).all())
