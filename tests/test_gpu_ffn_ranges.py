"""fp16 gradients of the gated projection on the GPU from dH far from 1, against 64 bits; bounds fixed from the arithmetic
before the first run."""
import math

import pytest
import torch

from clpeak_amd import capi
from test_gpu_ffn import ACTS, E, UNIT, act64, act_off, dv, gen, grad64, grad_off, tiled, within  # noqa: F401

pytestmark = pytest.mark.gpu


def gradients_f16(dv, act, dh, x, wg, wu, G, U):
    """The call on contiguous operands, and the definition with how far dG and dU may be off: their rounding to fp16 (few
    values: twice) after a power of two that brings the largest of them, `top`, to 2^14 at least: below 2^-14 / 2^14 top the
    step is 2^-24 / 2^14 top, half of it 2^-39 top."""
    T, D = x.shape
    F = wg.shape[0]
    n = dv.glu_backward_workspace(T, F, D)
    ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")
    dx, dwg, dwu = (torch.empty(r, D, dtype=torch.float16, device="cuda") for r in (T, F, F))
    dv.glu_backward(capi.TYPE_F16, act, dh, F, x, D, wg, wu, D, G, U, F, dx, D, dwg, dwu, D, T, F, D, ws, n)
    G64, U64, d64 = G.double(), U.double(), dh.double()
    dG, dU = d64 * U64 * grad64(act, G64), d64 * act64(act, G64)
    top = max(float(v[torch.isfinite(v)].abs().max()) for v in (dG, dU))
    unit = UNIT[torch.float16] ** 2 if T * F <= 32768 else UNIT[torch.float16]
    oG = unit * dG.abs() + top * 2.0 ** -39 + (d64 * U64).abs() * (grad_off(act, G64) + 4 * E)
    oU = unit * dU.abs() + top * 2.0 ** -39 + d64.abs() * (act_off(act, G64) + 4 * E)
    w64g, w64u, x64 = wg.double(), wu.double(), x.double()
    got = (dx, dwg, dwu)
    ref = (dG @ w64g + dU @ w64u, dG.T @ x64, dU.T @ x64)
    off = ((oG + 4 * F * E * dG.abs()) @ w64g.abs() + (oU + 4 * F * E * dU.abs()) @ w64u.abs(),
           (oG + 2 * T * E * dG.abs()).T @ x64.abs(), (oU + 2 * T * E * dU.abs()).T @ x64.abs())
    return got, ref, off


F16_SIZES = [(1, 300, 128), (48, 992, 64), (300, 1000, 256), (2048, 200, 128), (4200, 300, 128), (513, 2100, 64)]


@pytest.mark.parametrize("size", [1e-7, 1e-6, 1e-5, 1e-3])
@pytest.mark.parametrize("T, F, D", F16_SIZES)
def test_fp16_gradients_of_a_small_loss(tiled, size, T, F, D):
    """dH as an unscaled mean over many tokens gives it.  X and the weights are large enough that the results are not lost
    in fp16 as well."""
    act = ACTS[(T + F) % 4]
    g = gen(T + F)
    h = lambda r, c, s: (torch.randn(r, c, generator=g, device="cuda") * s).half()  # noqa: E731
    dh, x, wg, wu, G, U = h(T, F, size), h(T, D, 64), h(F, D, 64), h(F, D, 64), h(T, F, 1.5), h(T, F, 1)
    got, ref, off = gradients_f16(tiled, act, dh, x, wg, wu, G, U)
    for a, b, o in zip(got, ref, off):
        within(a, b, o, torch.float16)


@pytest.mark.parametrize("T, F, D", F16_SIZES)
def test_fp16_gradients_of_a_large_loss(tiled, T, F, D):
    """dG and dU past 65504, results well within: small weights and activations."""
    act = ACTS[(T + F) % 4]
    g = gen(T + F + 1)
    h = lambda r, c, s: (torch.randn(r, c, generator=g, device="cuda") * s).half()  # noqa: E731
    dh, x, wg, wu, G, U = h(T, F, 8000), h(T, D, 2e-4), h(F, D, 2e-4), h(F, D, 2e-4), h(T, F, 1.5).abs() + 30, h(T, F, 40)
    got, ref, off = gradients_f16(tiled, act, dh, x, wg, wu, G, U)
    for a, b, o in zip(got, ref, off):
        within(a, b, o, torch.float16)
    assert float((dh.double() * U.double()).abs().max()) > 2 * 65504


@pytest.mark.parametrize("T, F, D", F16_SIZES[1:])
def test_fp16_gradients_of_rows_of_very_different_sizes(tiled, T, F, D):
    """Rows of dH from 1e-7 to 1e3 in one call: every value as near as the largest one allows."""
    act = ACTS[(T + F) % 4]
    g = gen(T + F + 2)
    h = lambda r, c, s: (torch.randn(r, c, generator=g, device="cuda") * s).half()  # noqa: E731
    rows = 10 ** (10 * torch.rand(T, 1, generator=g, device="cuda") - 7)
    dh, x, wg, wu, G, U = h(T, F, rows), h(T, D, 1 / 16), h(F, D, 1 / 16), h(F, D, 1 / 16), h(T, F, 1.5), h(T, F, 1)
    got, ref, off = gradients_f16(tiled, act, dh, x, wg, wu, G, U)
    for a, b, o in zip(got, ref, off):
        within(a, b, o, torch.float16)


@pytest.mark.parametrize("T, F, D", [(40, 70, 64), (300, 1000, 128)])
def test_fp16_gradients_where_dh_is_not_finite(tiled, T, F, D):
    """An infinity and a NaN in dH stay in their rows of dX and of the weights' gradients, and say nothing about the size of
    the others."""
    g = gen(T)
    h = lambda r, c, s: (torch.randn(r, c, generator=g, device="cuda") * s).half()  # noqa: E731
    dh, x, wg, wu, G, U = h(T, F, 1e-6), h(T, D, 64), h(F, D, 64), h(F, D, 64), h(T, F, 1.5), h(T, F, 1)
    dh[5, 3], dh[20, 60] = math.inf, math.nan
    got, ref, off = gradients_f16(tiled, capi.GLU_SILU, dh, x, wg, wu, G, U)
    for a, b, o, rows in zip(got, ref, off, ((5, 20), (3, 60), (3, 60))):
        rest = [r for r in range(a.shape[0]) if r not in rows]
        assert not bool(torch.isfinite(a[list(rows)]).any())
        within(a[rest], b[rest], o[rest], torch.float16)


def test_fp16_gradients_that_are_all_zero(tiled):
    T, F, D = 130, 300, 128
    z = lambda r, c, v: torch.full((r, c), v, dtype=torch.float16, device="cuda")  # noqa: E731
    got, _, _ = gradients_f16(tiled, capi.GLU_SILU, z(T, F, 0.0), z(T, D, 1.0), z(F, D, 1.0), z(F, D, 1.0), z(T, F, 1.0), z(T, F, 1.0))
    assert all(bool((a == 0).all()) for a in got)


@pytest.mark.parametrize("rows", [1, 700])
def test_bf16_gradients_of_factors_that_are_far_apart(tiled, rows):
    """dG = dH U act'(G) in range with dH or U at the end of theirs: no product of two of the three leaves it, or loses
    bits below it, on the way.  X is the identity, so dWg is dG turned (dU = dH act(G) is out of range in some of the rows, which
    shows in dWu).  silu' at -14 is two terms of 14 : 1 that are each (8 + 2 |x|) u off: 50 u with the products."""
    T, F, dt = 8 * rows, 64, torch.bfloat16
    D = -(-T // 64) * 64
    big, small, u = 1.9921875 * 2.0 ** 127, 1.5 * 2.0 ** -126, 2.0 ** -20
    case = torch.tensor([(big, 2.4, u), (u, 2.4, big), (-big, 2.4, -u), (small, -14.0, 2.0 ** 100), (2.0 ** 100, -14.0, small), (small, 2.4, 1.0),
                         (1.0, 2.4, -big / 2), (big, -14.0, 1.0)], dtype=torch.float64).repeat(rows, 1)
    dh, G, U = (case[:, k, None].expand(T, F).to(dt).contiguous().cuda() for k in range(3))
    x, dwg, dwu = torch.eye(T, D, dtype=dt, device="cuda"), *(torch.empty(F, D, dtype=dt, device="cuda") for _ in range(2))
    n = tiled.glu_backward_workspace(T, F, D)
    tiled.glu_backward(capi.TYPE_BF16, capi.GLU_SILU, dh, F, x, D, None, None, D, G, U, F, None, D, dwg, dwu, D, T, F, D, torch.empty(n, dtype=torch.uint8, device="cuda"), n)
    ref = dh.double() * U.double() * grad64(capi.GLU_SILU, G.double())
    assert float(ref.abs().max()) < 3.38e38
    # (of many values dG is rounded to bf16 first)
    within(dwg[:, :T].T, ref, (50 * E + (0 if T * F <= 32768 else UNIT[dt])) * ref.abs(), dt)


@pytest.mark.parametrize("at", [(0, 0), (4199, 1098), (0, 1098), (4199, 0), (2111, 700), (4100, 1050)])
def test_fp16_gradients_with_the_largest_value_anywhere(dv, at):
    """More tiles of dH than there are workgroups that look for its largest value, and one value 10^8 times the others, in the
    first and in the last of rows and columns that are no multiples of anything: missed, it would overflow."""
    T, F, D = 4200, 1099, 64
    g = gen(at[0] + at[1])
    h = lambda r, c, s: (torch.randn(r, c, generator=g, device="cuda") * s).half()  # noqa: E731
    dh, x, wg, wu, G, U = h(T, F, 1e-5), h(T, D, 1 / 16), h(F, D, 1 / 16), h(F, D, 1 / 16), h(T, F, 1.5), h(T, F, 1)
    dh[at], G[at], U[at] = 1000.0, 3.0, 1.0
    got, ref, off = gradients_f16(dv, capi.GLU_SILU, dh, x, wg, wu, G, U)
    for a, b, o in zip(got, ref, off):
        within(a, b, o, torch.float16)


@pytest.mark.parametrize("T, F", [(3, 384), (300, 384)])
def test_fp16_gradients_captured_and_replayed_on_dh_of_other_sizes(T, F):
    """The scaling is found anew on every replay: dH from 1e-6 to 1e4, infinities in between, each replay as the eager call."""
    D = 128
    st = torch.cuda.Stream()
    d = capi.Device(0, stream=st.cuda_stream)
    g = gen(61)
    h = lambda r, c, s: (torch.randn(r, c, generator=g, device="cuda") * s).half()  # noqa: E731
    x, wg, wu, G, U = h(T, D, 1e-3), h(F, D, 1e-3), h(F, D, 1e-3), h(T, F, 1.5), h(T, F, 1)
    dh = torch.zeros(T, F, dtype=torch.float16, device="cuda")
    outs = [torch.zeros(r, D, dtype=torch.float16, device="cuda") for r in (T, F, F)]
    n = d.glu_backward_workspace(T, F, D)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")

    def call():
        d.glu_backward(capi.TYPE_F16, capi.GLU_SILU, dh, F, x, D, wg, wu, D, G, U, F, outs[0], D, outs[1], outs[2], D, T, F, D, ws, n)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        call()
    for size in (1e4, 1e-6, 1.0, math.inf, 1e-3, 0.0, 100.0):
        dh.copy_(h(T, F, size if math.isfinite(size) else 1.0))
        if not math.isfinite(size):
            dh[1, 5] = size
        for o in outs:
            o.fill_(7.0)
        ws.fill_(0xFF)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        call()
        d.sync()
        assert all(torch.equal(a.view(torch.int16), o.view(torch.int16)) for a, o in zip(got, outs)), size
        assert bool(torch.isfinite(got[0]).all()) == math.isfinite(size) and not bool((got[0] == 7.0).any())
    del graph
    d.close()


def test_fp16_gradients_without_rows(tiled):
    F, D = 100, 128
    n = tiled.glu_backward_workspace(0, F, D)
    ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")
    dwg, dwu = (torch.full((F, D), 3.0, dtype=torch.float16, device="cuda") for _ in range(2))
    tiled.glu_backward(capi.TYPE_F16, capi.GLU_GELU, None, F, None, D, None, None, D, None, None, F, None, D, dwg, dwu, D, 0, F, D, ws, n)
    assert bool((dwg == 0).all()) and bool((dwu == 0).all())
