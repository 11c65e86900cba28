"""Paths of the feed-forward operators that tests/test_gpu_ffn.py does not reach."""
import math

import pytest
import torch

from clpeak_amd import capi
from test_gpu_ffn import E, TYPES, dv, gen, operand, padded, quantized, untouched, within  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("keep", [True, False])
@pytest.mark.parametrize("type", [capi.TYPE_BF16, capi.TYPE_F16])
def test_glu_forward_many_rounds_of_rows_that_start_on_lines(dv, type, keep):
    """At least four rounds of 256x256 tiles over the CUs and outputs whose rows start on 64 bytes: stored past the caches,
    but for what lies at the odd end of a row."""
    T, F, D, ld, dt = 8200, 4131, 64, 4160, TYPES[type]
    g = gen(78)
    x, wg, wu = operand(g, T, D, D, dt), operand(g, F, D, D, dt, 0.25), operand(g, F, D, D, dt, 0.25)
    (hb, h), (gb, G), (ub, U) = (padded(T, F, ld, dt, -7.0) for _ in range(3))
    assert ((T + 255) // 256) * ((F + 127) // 128) >= 4 * dv.props.num_cus
    assert ld * 2 % 64 == 0 and all(v.data_ptr() % 64 == 0 for v in (h, G, U))
    dv.glu_forward(type, capi.GLU_RELU, x, D, wg, wu, D, h, ld, G if keep else None, U if keep else None, ld if keep else 0, T, F, D)
    G64, U64 = x.double() @ wg.double().T, x.double() @ wu.double().T
    sg, su = 2 * D * E * (x.double().abs() @ wg.double().abs().T), 2 * D * E * (x.double().abs() @ wu.double().abs().T)
    within(h, G64.clamp(min=0) * U64, sg * U64.abs() + G64.abs() * su + 4 * E * (G64 * U64).abs(), dt)
    assert untouched(hb, h, ld, -7.0)
    if keep:
        within(G, G64, sg, dt)
        within(U, U64, su, dt)
        assert untouched(gb, G, ld, -7.0) and untouched(ub, U, ld, -7.0)
    else:
        assert bool((gb == -7.0).all()) and bool((ub == -7.0).all())


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("M, K, k_pad", [(3, 65535, 65536), (2, 65536, 65536), (3, 65537, 65664), (2, 73729, 73729), (3, 130957, 131072)])
def test_quantize_rows_that_registers_do_not_hold(dv, type, M, K, k_pad):
    """Rows around and past 65536 elements, which are read twice; the largest value in the last, partial chunk, in the first
    or in between."""
    dt = TYPES[type]
    g = gen(K)
    ldx, ldq = K + 3, k_pad + 1
    _, x = padded(M, K, ldx, dt, math.nan)
    x.copy_(torch.randn(M, K, generator=g, device="cuda").to(dt))
    for m, at in enumerate((K - 1, 0, 40000)[:M]):
        x[m, at] = -9.0
    qb, q = padded(M, k_pad, ldq, torch.int8, 77)
    s = torch.full((M + 1,), -1.0, device="cuda")
    dv.quantize_i8(type, x, ldx, q, ldq, s, M, K, k_pad)
    rq, rs = quantized(x)
    assert torch.equal(q[:, :K].double(), rq) and torch.equal(s[:-1], rs) and s[-1] == -1
    assert bool((q[:, K:] == 0).all()) and untouched(qb, q, ldq, 77)
