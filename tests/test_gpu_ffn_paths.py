"""Paths of the feed-forward operators that tests/test_gpu_ffn.py does not reach."""
import math

import pytest
import torch

from clpeak_amd import capi
from test_gpu_ffn import E, TYPES, dv, gen, i8_problem, operand, padded, quantized, tiled, untouched, within  # noqa: F401

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


def test_gemm_i8_scaled_scales_at_the_ends_of_their_range(tiled):
    """scale_a below 2^97 against any scale_b: the product with the largest sum stays in fp32's range, and with a scale_b as
    small as scale_a is large so does the result."""
    dv = tiled
    M, N, K = 40, 50, 256
    g, a, lda, (b,), ldb, sa, (sb,) = i8_problem(M, N, K, 10)
    a[1, :], b[1, :] = -128, -128
    sa[1], sb[1], sa[2], sb[2] = 2.0 ** 96, 2.0 ** -96, 2.0 ** -126, 2.0 ** 120
    c = torch.empty(M, N, device="cuda")
    dv.gemm_i8_scaled(a, lda, b, ldb, sa, sb, None, capi.TYPE_F32, c, N, M, N, K)
    prod = (a.double() @ b.double().T) * sa.double()[:, None] * sb.double()[None, :]
    for m, n in ((1, 1), (2, 2)):
        assert abs(float(c[m, n]) - float(prod[m, n])) <= 4 * E * abs(float(prod[m, n]))
    assert float(c[1, 1]) == 128 * 128 * K


@pytest.mark.parametrize("first", ["gradients", "product"])
def test_fp16_gradients_in_slices_and_the_fp8_product_on_one_handle(first):
    """Both kernels take the whole LDS of a CU, each by a permission of its own."""
    T, F, D, n = 8192, 512, 4096, 512
    d = capi.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    g = gen(5)
    dh, x, G, U = (operand(g, T, c, c, torch.float16) for c in (F, D, F, F))
    dw = torch.empty(2, F, D, dtype=torch.float16, device="cuda")
    a, b = (torch.randint(0, 8, (n, n), generator=g, device="cuda").float().to(torch.float8_e4m3fn) for _ in range(2))
    c = torch.empty(n, n, dtype=torch.bfloat16, device="cuda")
    size = d.glu_backward_workspace(T, F, D)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")

    def gradients():
        d.glu_backward(capi.TYPE_F16, capi.GLU_RELU, dh, F, x, D, None, None, D, G, U, F, None, D, dw[0], dw[1], D, T, F, D, ws, size)

    def product():
        d.gemm_tiling(capi.GEMM_TILING_256)
        d._check(d.lib.mi355_gemm_fp8_e4m3(d.h, a.data_ptr(), b.data_ptr(), c.data_ptr(), n, n, n, 1.0, 1.0))
        d.gemm_tiling(capi.GEMM_TILING_AUTO)

    for call in ((gradients, product) if first == "gradients" else (product, gradients)):
        call()
    ref = a.double() @ b.double().T
    within(c, ref, 2 * n * E * ref.abs(), torch.bfloat16)
    dU = dh.double() * G.double().clamp(min=0)
    within(dw[1], dU.T @ x.double(), (2.0 ** -11 + 2 * T * E) * (dU.abs().T @ x.double().abs()), torch.float16)
    torch.cuda.synchronize()
    d.close()
