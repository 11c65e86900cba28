"""Paths of the feed-forward operators that tests/test_gpu_ffn.py does not reach."""
import pytest
import torch

from clpeak_amd import capi
from test_gpu_ffn import E, TYPES, dv, gen, operand, padded, untouched, within  # noqa: F401

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
