"""The feed-forward operators on the GPU against plain evaluations in 64 bits.

Tolerances, fixed from the arithmetic before the first run.  u is the rounding of the output type, half a step of it
(2^-8 bf16, 2^-11 fp16, 2^-24 fp32), relative; fp16 also rounds to a multiple of 2^-24 near zero (t: half of that).
  sums     a sum of n products in fp32 is off by at most n 2^-23 sum |a||b| (n additions, each of which may truncate);
  sigmoid  2^x and 1/x are off by an ulp each and their arguments by 2^-24 relative: (8 + 2 |x|) 2^-24 relative;
  erf      absolute, 4 ulp of 1;
and what follows is first order in these (act' is at most 1.13, act at most |x|), with a factor of 2 over all."""
import math

import numpy as np
import pytest
import torch

from clpeak_amd import capi

pytestmark = pytest.mark.gpu

TYPES = {capi.TYPE_BF16: torch.bfloat16, capi.TYPE_F16: torch.float16, capi.TYPE_F32: torch.float32}
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
ACTS = [capi.GLU_SILU, capi.GLU_GELU, capi.GLU_GELU_TANH, capi.GLU_RELU]
E = 2.0 ** -24


@pytest.fixture(scope="module")
def dv():
    """A handle on torch's own stream: what the tests prepare with torch, the calls and the comparisons are in order."""
    d = capi.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    yield d
    torch.cuda.synchronize()
    d.close()


@pytest.fixture(params=["auto", "256", "128", "64", "256x128"])
def tiled(dv, request):
    """The library's own choice of kernel (one for few rows, four tilings) and each tiling pinned."""
    dv.gemm_tiling({"auto": capi.GEMM_TILING_AUTO, "256": capi.GEMM_TILING_256, "128": capi.GEMM_TILING_128, "64": capi.GEMM_TILING_64,
                     "256x128": capi.GEMM_TILING_256X128}[request.param])
    yield dv
    dv.gemm_tiling(capi.GEMM_TILING_AUTO)


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def act64(act, x):
    if act == capi.GLU_SILU:
        return x * torch.sigmoid(x)
    if act == capi.GLU_GELU:
        return x * 0.5 * torch.erfc(-x * math.sqrt(0.5))
    if act == capi.GLU_GELU_TANH:
        return x * torch.sigmoid(math.sqrt(8 / math.pi) * (x + 0.044715 * x ** 3))
    return x.clamp(min=0)


def grad64(act, x):
    if act == capi.GLU_SILU:
        p = torch.sigmoid(x)
        return p + x * p * (1 - p)
    if act == capi.GLU_GELU:
        return 0.5 * torch.erfc(-x * math.sqrt(0.5)) + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    if act == capi.GLU_GELU_TANH:
        c = math.sqrt(8 / math.pi)
        p = torch.sigmoid(c * (x + 0.044715 * x ** 3))
        return p + x * p * (1 - p) * c * (1 + 3 * 0.044715 * x * x)
    return (x > 0).double()


def act_off(act, x):
    """How far the fp32 activation of an exact argument may be off."""
    return x.abs() * ((16 + 4 * x.abs().clamp(max=40)) * E if act != capi.GLU_GELU else 8 * E)


def grad_off(act, x):
    return (1 + x.abs().clamp(max=20)) * ((16 + 8 * x.abs().clamp(max=20)) * E if act != capi.GLU_GELU else 16 * E)


def padded(rows, cols, ld, dtype, fill):
    """A rows x cols matrix with rows ld apart in a buffer that holds nothing but `fill`, with a spare row on both sides."""
    buf = torch.full(((rows + 2) * ld,), fill, dtype=dtype, device="cuda")
    return buf, buf[ld:ld + rows * ld].view(rows, ld)[:, :cols]


def untouched(buf, view, ld, fill):
    """Nothing but the view's elements was written."""
    rows, cols = view.shape
    whole = buf.view(rows + 2, ld)
    same = (lambda x: torch.isnan(x)) if isinstance(fill, float) and math.isnan(fill) else (lambda x: x == fill)
    return bool(same(whole[0]).all() and same(whole[-1]).all() and same(whole[1:-1, cols:]).all())


def operand(g, rows, cols, ld, dtype, scale=1.0):
    """An operand whose padding between the rows holds NaN (int8: 111), which no product may take up."""
    fill = 111 if dtype == torch.int8 else math.nan
    buf, v = padded(rows, cols, ld, dtype, fill)
    if dtype == torch.int8:
        v.copy_(torch.randint(-128, 128, (rows, cols), generator=g, device="cuda"))
    else:
        v.copy_((torch.randn(rows, cols, generator=g, device="cuda") * scale).to(dtype))
    return v


def within(got, ref, off, dtype):
    """|got - ref| <= 2 off + u |ref| + t, and what is not finite is not finite in the same way."""
    got = got.double()
    bad = (got - ref).abs() > 2 * off + UNIT[dtype] * ref.abs() + TINY[dtype]
    bad &= torch.isfinite(ref)
    bad |= torch.isfinite(ref) != torch.isfinite(got)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:3].tolist(), got[bad][:3].tolist(), ref[bad][:3].tolist())


# ---- the gated projection --------------------------------------------------------------------------------------------

SIZES = [  # T, F, D: one token, around the edges of 16-, 64-, 128- and 256-row tiles, more tiles than CUs, long and short sums
    (1, 1, 64), (1, 16, 64), (1, 257, 1024), (2, 17, 128), (15, 100, 192), (16, 128, 320), (17, 31, 64), (33, 64, 512), (63, 65, 448),
    (64, 130, 256), (65, 127, 640), (127, 129, 576), (128, 64, 704), (129, 191, 384), (255, 257, 128), (256, 128, 1088), (257, 383, 320),
    (300, 1000, 960), (511, 640, 64), (777, 129, 1024), (1025, 2050, 256),
]


@pytest.mark.parametrize("type", [capi.TYPE_BF16, capi.TYPE_F16])
@pytest.mark.parametrize("T, F, D", SIZES)
def test_glu_forward(tiled, type, T, F, D):
    dv = tiled
    dt, act = TYPES[type], ACTS[(T + F) % 4]
    g = gen(T * 7 + F)
    ldx, ldw, ldh, ldg = D + 8 * (T % 3), D + 8 * (F % 5), F + T % 4, F + F % 3
    x, wg, wu = operand(g, T, D, ldx, dt), operand(g, F, D, ldw, dt, 2 / math.sqrt(D)), operand(g, F, D, ldw, dt, 2 / math.sqrt(D))
    G64, U64 = x.double() @ wg.double().T, x.double() @ wu.double().T
    sg, su = D * 2 * E * (x.double().abs() @ wg.double().abs().T), D * 2 * E * (x.double().abs() @ wu.double().abs().T)
    H64 = act64(act, G64) * U64
    off = (1.13 * sg + act_off(act, G64)) * U64.abs() + G64.abs() * su + 4 * E * H64.abs()
    for keep in (True, False):
        hb, h = padded(T, F, ldh, dt, -7.0)
        gb, gk = padded(T, F, ldg, dt, -7.0)
        ub, uk = padded(T, F, ldg, dt, -7.0)
        dv.glu_forward(type, act, x, ldx, wg, wu, ldw, h, ldh, gk if keep else None, uk if keep else None, ldg if keep else 0, T, F, D)
        within(h, H64, off, dt)
        assert untouched(hb, h, ldh, -7.0)
        if keep:
            within(gk, G64, sg, dt)
            within(uk, U64, su, dt)
            assert untouched(gb, gk, ldg, -7.0) and untouched(ub, uk, ldg, -7.0)
            again, first = torch.empty(T, F, dtype=dt, device="cuda"), h.clone()
            dv.glu_forward(type, act, x, ldx, wg, wu, ldw, again, F, None, None, 0, T, F, D)
            assert torch.equal(again, first)     # the same bits on every call, kept sums or not
        else:
            assert bool((gb == -7.0).all())


def test_glu_forward_keeps_what_is_not_finite_in_its_row(tiled):
    """An infinity or NaN in a row of X shows in that row of H and nowhere else; one in a row of a weight in that column."""
    dv = tiled
    T, F, D = 70, 150, 128
    g = gen(3)
    x, wg, wu = (operand(g, n, D, D, torch.bfloat16, s) for n, s in ((T, 1.0), (F, 0.1), (F, 0.1)))
    h = torch.zeros(T, F, dtype=torch.bfloat16, device="cuda")
    x[5, 3], x[69, 100], wg[149, 0], wu[20, 127] = math.nan, math.inf, math.nan, -math.inf
    dv.glu_forward(capi.TYPE_BF16, capi.GLU_SILU, x, D, wg, wu, D, h, F, None, None, 0, T, F, D)
    odd = ~torch.isfinite(h)
    want = torch.zeros_like(odd)
    want[5], want[:, 149], want[:, 20] = True, True, True
    rows = [t for t in range(T) if t != 69]
    assert torch.equal(odd[rows], want[rows])
    assert bool(torch.isnan(h[5]).all()) and bool(torch.isnan(h[:, 149]).all())


@pytest.mark.parametrize("act", ACTS)
def test_glu_activations_over_the_whole_range(tiled, act):
    """G is one product of a value and 1 and U is 1, so H is the activation itself, at every bf16 value there is."""
    dv = tiled
    D = 64
    bits = torch.arange(0, 1 << 16, device="cuda", dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    vals = bits[torch.isfinite(bits)]
    T, F = vals.numel(), 1
    x = torch.zeros(T, D, dtype=torch.bfloat16, device="cuda")
    x[:, 0], x[:, 1] = vals, 1.0
    wg, wu = torch.zeros(F, D, dtype=torch.bfloat16, device="cuda"), torch.zeros(F, D, dtype=torch.bfloat16, device="cuda")
    wg[0, 0], wu[0, 1] = 1.0, 1.0
    h = torch.empty(T, F, dtype=torch.bfloat16, device="cuda")
    dv.glu_forward(capi.TYPE_BF16, act, x, D, wg, wu, D, h, F, None, None, 0, T, F, D)
    ref = act64(act, vals.double())[:, None]
    ok = (ref.abs() >= 2.0 ** -120) | (ref == 0)      # (a product that small may be flushed to zero on the way)
    within(torch.where(ok, h, 0), torch.where(ok, ref, 0.0), act_off(act, vals.double())[:, None], torch.bfloat16)
    # and its gradient: dX has dG in column 0 and dU in column 1
    G, U, dH = vals[:, None].contiguous(), torch.ones(T, 1, dtype=torch.bfloat16, device="cuda"), torch.ones(T, 1, dtype=torch.bfloat16, device="cuda")
    dx = torch.empty(T, D, dtype=torch.bfloat16, device="cuda")
    n = dv.glu_backward_workspace(T, F, D)
    dv.glu_backward(capi.TYPE_BF16, act, dH, F, x, D, wg, wu, D, G, U, F, dx, D, None, None, 0, T, F, D, torch.empty(n, dtype=torch.uint8, device="cuda"), n)
    v = vals.double()
    within(dx[:, 1], torch.where(ok[:, 0], ref[:, 0], dx[:, 1].double()), act_off(act, v) + 2.0 ** -120, torch.bfloat16)
    within(dx[:, 0], grad64(act, v.clamp(-1e9, 1e9)), grad_off(act, v), torch.bfloat16)
    assert bool((dx[:, 2:] == 0).all())


@pytest.mark.parametrize("type", [capi.TYPE_BF16, capi.TYPE_F16])
@pytest.mark.parametrize("T, F, D", SIZES)
def test_glu_backward(tiled, type, T, F, D):
    dv = tiled
    dt, act = TYPES[type], ACTS[(T + F + 1) % 4]
    g = gen(T * 11 + F)
    ldx, ldw, ldd, ldg, lddx, lddw = D + 8 * (T % 3), D + 8 * (F % 5), F + T % 4, F + F % 3, D + T % 3, D + F % 7
    x, wg, wu = operand(g, T, D, ldx, dt), operand(g, F, D, ldw, dt, 1 / math.sqrt(F)), operand(g, F, D, ldw, dt, 1 / math.sqrt(F))
    dh, G, U = operand(g, T, F, ldd, dt), operand(g, T, F, ldg, dt, 1.5), operand(g, T, F, ldg, dt)
    G64, U64, d64 = G.double(), U.double(), dh.double()
    dG, dU = d64 * U64 * grad64(act, G64), d64 * act64(act, G64)
    # rounded to the type before the products, on top of what the activations are off; few values as two of the type,
    # the second of which is what the first is off, at most a unit of the value, and off by a unit of that
    unit = UNIT[dt] ** 2 if T * F <= 32768 else UNIT[dt]
    oG = unit * dG.abs() + TINY[dt] + (d64 * U64).abs() * (grad_off(act, G64) + 4 * E)
    oU = unit * dU.abs() + TINY[dt] + d64.abs() * (act_off(act, G64) + 4 * E)
    w64g, w64u, x64 = wg.double(), wu.double(), x.double()
    n = dv.glu_backward_workspace(T, F, D)
    room = torch.full((n + 512,), 0xFF, dtype=torch.uint8, device="cuda")     # (0xffff is a NaN of both types)
    ws = room[256 - room.data_ptr() % 256 if room.data_ptr() % 256 else 0:]
    ref = {"dx": dG @ w64g + dU @ w64u, "dwg": dG.T @ x64, "dwu": dU.T @ x64}
    off = {"dx": (oG + 4 * F * E * dG.abs()) @ w64g.abs() + (oU + 4 * F * E * dU.abs()) @ w64u.abs(),
           "dwg": (oG + 2 * T * E * dG.abs()).T @ x64.abs(), "dwu": (oU + 2 * T * E * dU.abs()).T @ x64.abs()}
    first = None
    for parts in ("dx dw", "dx", "dw"):
        bx, dx = padded(T, D, lddx, dt, -7.0)
        bg, dwg = padded(F, D, lddw, dt, -7.0)
        bu, dwu = padded(F, D, lddw, dt, -7.0)
        has_x, has_w = "dx" in parts, "dw" in parts
        dv.glu_backward(type, act, dh, ldd, x if has_w else None, ldx, wg if has_x else None, wu if has_x else None, ldw, G, U, ldg,
                        dx if has_x else None, lddx, dwg if has_w else None, dwu if has_w else None, lddw, T, F, D, ws, n)
        if has_x:
            within(dx, ref["dx"], off["dx"], dt)
            assert untouched(bx, dx, lddx, -7.0)
        else:
            assert bool((bx == -7.0).all())
        if has_w:
            within(dwg, ref["dwg"], off["dwg"], dt)
            within(dwu, ref["dwu"], off["dwu"], dt)
            assert untouched(bg, dwg, lddw, -7.0) and untouched(bu, dwu, lddw, -7.0)
        else:
            assert bool((bg == -7.0).all()) and bool((bu == -7.0).all())
        if first is None:
            first = (dx.clone(), dwg.clone(), dwu.clone())
        else:   # the same bits, whichever parts are asked for
            assert (not has_x or torch.equal(dx, first[0])) and (not has_w or (torch.equal(dwg, first[1]) and torch.equal(dwu, first[2])))
    assert bool((room[ws.data_ptr() - room.data_ptr() + n:] == 0xFF).all())


@pytest.mark.parametrize("T, F, D", [(4200, 320, 4096), (600, 4096, 512), (2048, 2752, 1024), (130, 8192, 256), (3000, 70, 2048), (33, 2752, 1024), (100, 5000, 2048),
                                     (8192, 500, 512), (1, 8192, 512), (16, 4099, 1024), (32, 1000, 4096), (33, 992, 64), (33, 993, 64), (450, 70, 1024), (2000, 16, 8192),
                                     (256, 128, 256)])
def test_glu_backward_larger(tiled, T, F, D):
    """Sizes at which the products are cut along their sums, go round the CUs more than once, and have rows left over for a
    launch of their own."""
    test_glu_backward(tiled, capi.TYPE_BF16, T, F, D)


@pytest.mark.parametrize("T, F, D", [(4200, 1100, 128), (2176, 2100, 64), (513, 20000, 64)])
def test_glu_forward_larger(tiled, T, F, D):
    """More tiles than CUs, and rows left over for a launch of their own."""
    test_glu_forward(tiled, capi.TYPE_F16, T, F, D)


def test_glu_forward_many_rounds(dv):
    """More than four rounds of 256x256 tiles over the CUs, where the outputs are stored past the caches: an odd number of
    channels, both sums kept, whole outputs."""
    T, F, D, dt = 8200, 4131, 64, torch.bfloat16
    g = gen(77)
    x, wg, wu = operand(g, T, D, D, dt), operand(g, F, D, D, dt, 0.25), operand(g, F, D, D, dt, 0.25)
    (hb, h), (gb, G), (ub, U) = (padded(T, F, F + 2, dt, -7.0) for _ in range(3))
    assert ((T + 255) // 256) * ((F + 127) // 128) >= 4 * dv.props.num_cus
    dv.glu_forward(capi.TYPE_BF16, capi.GLU_RELU, x, D, wg, wu, D, h, F + 2, G, U, F + 2, T, F, D)
    G64, U64 = x.double() @ wg.double().T, x.double() @ wu.double().T
    sg, su = 2 * D * E * (x.double().abs() @ wg.double().abs().T), 2 * D * E * (x.double().abs() @ wu.double().abs().T)
    within(G, G64, sg, dt)
    within(U, U64, su, dt)
    within(h, G64.clamp(min=0) * U64, sg * U64.abs() + G64.abs() * su + 4 * E * (G64 * U64).abs(), dt)
    assert untouched(hb, h, F + 2, -7.0) and untouched(gb, G, F + 2, -7.0) and untouched(ub, U, F + 2, -7.0)


def test_nothing_is_summed_over_no_rows_on_any_tiling(tiled):
    test_glu_backward_without_rows_clears_the_weights_gradients(tiled)


def test_glu_backward_without_rows_clears_the_weights_gradients(dv):
    F, D = 100, 128
    n = dv.glu_backward_workspace(0, F, D)
    ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")
    dwg, dwu = (torch.full((F, D), 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    dv.glu_backward(capi.TYPE_BF16, capi.GLU_SILU, None, F, None, D, None, None, D, None, None, F, None, D, dwg, dwu, D, 0, F, D, ws, n)
    assert bool((dwg == 0).all()) and bool((dwu == 0).all())


def test_the_gradient_formula_against_differences():
    """The 64-bit formulas the kernels are held to, against central differences of the 64-bit forward pass."""
    g = torch.Generator().manual_seed(1)
    T, F, D = 5, 7, 6
    for act in ACTS:
        x, wg, wu, dh = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((T, D), (F, D), (F, D), (T, F)))
        f = lambda x, wg, wu: float((act64(act, x @ wg.T) * (x @ wu.T) * dh).sum())  # noqa: E731
        G, U = x @ wg.T, x @ wu.T
        dG, dU = dh * U * grad64(act, G), dh * act64(act, G)
        grads = (dG @ wg + dU @ wu, dG.T @ x, dU.T @ x)
        for k, (p, got) in enumerate(zip((x, wg, wu), grads)):
            for i, j in ((0, 0), (2, 3), (4, 5)):
                e = 1e-6
                args = [[a.clone() for a in (x, wg, wu)] for _ in range(2)]
                args[0][k][i, j] += e
                args[1][k][i, j] -= e
                assert abs((f(*args[0]) - f(*args[1])) / (2 * e) - float(got[i, j])) < 1e-6 * (1 + abs(float(got[i, j]))), (act, k, i, j)


# ---- int8 ------------------------------------------------------------------------------------------------------------

def quantized(x):
    """The definition, in 64 bits: 127 x / amax is exact enough there to fall on the right side of every border."""
    x = x.double()
    top = x.abs().amax(1)
    q = torch.where(top[:, None] > 0, x * 127 / top[:, None], torch.zeros_like(x)).round()
    return q, (top / 127).float()


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("M, K", [(1, 1), (3, 7), (5, 8), (9, 100), (2, 511), (7, 512), (4, 513), (6, 1024), (13, 2047), (3, 2048), (5, 2049), (3, 4096),
                                  (2, 4104), (3, 8191), (2, 8200), (2, 16384), (2, 16385), (1, 50001), (1030, 64)])
def test_quantize(dv, type, M, K):
    dt = TYPES[type]
    g = gen(M * 5 + K)
    ldx, k_pad = K + M % 5, -(-K // 128) * 128 + 128 * (M % 2)
    ldq = k_pad + M % 3
    xb, x = padded(M, K, ldx, dt, math.nan)
    x.copy_((torch.randn(M, K, generator=g, device="cuda") * torch.exp(3 * torch.randn(M, 1, generator=g, device="cuda"))).to(dt))
    if M > 4:
        x[1] = 0
        x[2] = torch.randint(-127, 128, (K,), generator=g, device="cuda").to(dt) * 0.5       # amax 63.5: about half of the quotients are ties
        x[2, K - 1] = 63.5
        x[3] *= 1e-30 if dt != torch.float16 else 1e-4
    for kp in (k_pad, K):
        qb, q = padded(M, kp, ldq, torch.int8, 77)
        s = torch.full((M + 2,), -1.0, device="cuda")
        dv.quantize_i8(type, x, ldx, q, ldq, s[1:], M, K, kp)
        rq, rs = quantized(x)
        assert torch.equal(q[:, :K].double(), rq)
        assert torch.equal(s[1:-1], rs) and s[0] == -1 and s[-1] == -1
        assert bool((q[:, K:] == 0).all()) and untouched(qb, q, ldq, 77)


@pytest.mark.parametrize("type", list(TYPES))
def test_quantize_decides_the_borders_exactly(dv, type):
    """Rows whose quotients lie on, just under and just over the borders between two whole numbers: for a largest
    magnitude `top`, the values of the type next to (k + 1/2) top / 127."""
    dt = TYPES[type]
    rows = []
    for top in (127.0, 1.0, 63.5, 3.96875, 100.0, 0.3, 17.25, 2.0 ** -14, 60000.0, 1e-3):
        top = torch.tensor(top, dtype=torch.float64).to(dt)
        mid = ((torch.arange(127, dtype=torch.float64) + 0.5) * top.double() / 127).to(dt)
        step = {2: torch.int16, 4: torch.int32}[mid.element_size()]
        near = [(mid.view(step) + d).view(dt) for d in (-2, -1, 0, 1, 2)]
        near = torch.cat(near + [-v for v in near])
        near = torch.where(near.abs() <= top, near, torch.zeros_like(near))
        rows.append(torch.cat((near, top[None])))
    x = torch.stack(rows).cuda()
    M, K = x.shape
    q, s = torch.empty(M, K, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    dv.quantize_i8(type, x, K, q, K, s, M, K, K)
    rq, rs = quantized(x)
    assert torch.equal(q.double(), rq) and torch.equal(s, rs)


def test_quantize_extremes(dv):
    """The smallest and largest values of fp32, and rows that are not finite."""
    tiny, huge = 2.0 ** -149, 3.4028234663852886e38
    x = torch.tensor([[tiny, 0, -tiny, tiny], [3 * tiny, 2 * tiny, tiny, -tiny], [huge, -huge, huge / 254, 1.0], [2.0 ** -126, 2.0 ** -130, -2.0 ** -133, 0],
                      [1, math.inf, 2, 3], [1, 2, math.nan, 3], [-math.inf, math.nan, 0, 0], [0, -0.0, 0, 0]], dtype=torch.float64).float().cuda()
    M, K = x.shape
    q, s = torch.full((M, 8), 9, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    dv.quantize_i8(capi.TYPE_F32, x, K, q, 8, s, M, K, 8)
    rq, rs = quantized(x)
    fine = torch.isfinite(x).all(1)
    assert torch.equal(q[fine, :K].double(), rq[fine]) and torch.equal(s[fine], rs[fine])
    assert bool(torch.isnan(s[~fine]).all()) and bool((q[~fine] == 0).all()) and bool((q[:, K:] == 0).all())


I8_SIZES = [  # M, N, K
    (1, 1, 128), (1, 16, 128), (1, 1000, 4096), (2, 33, 256), (16, 128, 384), (17, 200, 1152), (31, 64, 640), (33, 100, 128), (64, 65, 2048),
    (65, 129, 512), (100, 256, 4224), (128, 127, 256), (129, 640, 384), (200, 257, 16384), (255, 256, 128), (256, 512, 1280), (257, 129, 640),
    (511, 383, 896), (700, 1030, 256), (2100, 2300, 384),
]


def i8_problem(M, N, K, seed, ws=1):
    g = gen(seed)
    lda, ldb = K + 16 * (M % 4), K + 16 * (N % 3)
    a, b = operand(g, M, K, lda, torch.int8), [operand(g, N, K, ldb, torch.int8) for _ in range(ws)]
    a[0], b[0][0] = -128, -128          # the largest sum there is
    sa, sb = torch.rand(M, generator=g, device="cuda") * 0.02, [torch.rand(N, generator=g, device="cuda") * 0.02 / math.sqrt(K) for _ in range(ws)]
    return g, a, lda, b, ldb, sa, sb


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("M, N, K", I8_SIZES)
def test_gemm_i8_scaled(tiled, type, M, N, K):
    dv = tiled
    dt = TYPES[type]
    g, a, lda, (b,), ldb, sa, (sb,) = i8_problem(M, N, K, M + 3 * N + K)
    bias = torch.randn(N, generator=g, device="cuda")
    ldc = N + M % 3
    n = dv.gemm_i8_scaled_workspace(M, N, K)
    ws = torch.full((max(n, 16),), 0x7F, dtype=torch.uint8, device="cuda")
    prod = (a.double() @ b.double().T) * sa.double()[:, None] * sb.double()[None, :]
    for with_bias in (False, True):
        ref = prod + bias.double() if with_bias else prod
        off = 4 * E * (prod.abs() + ref.abs())
        outs = []
        for w, nb in ((None, 0), (ws, n)):
            cb, c = padded(M, N, ldc, dt, -7.0)
            dv.gemm_i8_scaled(a, lda, b, ldb, sa, sb, bias if with_bias else None, type, c, ldc, M, N, K, w, nb)
            within(c, ref, off, dt)
            assert untouched(cb, c, ldc, -7.0)
            outs.append(c)
        assert torch.equal(outs[0], outs[1])      # the sums are exact, however K is split


def test_gemm_i8_scaled_the_deepest_sum(tiled):
    """K = 130944 of (-128)^2: the sum is 2^31 - 2^21, and its rounding to fp32 the only one before the scales."""
    dv = tiled
    K, N = 130944, 5
    for M in (1, 70):
        a, b = (torch.full((r, K), -128, dtype=torch.int8, device="cuda") for r in (M, N))
        c = torch.empty(M, N, device="cuda")
        one = torch.ones(max(M, N), device="cuda")
        dv.gemm_i8_scaled(a, K, b, K, one, one, None, capi.TYPE_F32, c, N, M, N, K)
        assert bool((c == float(K * 16384)).all())


def test_gemm_i8_scaled_scales_that_are_extreme(tiled):
    """A zero scale gives zeros, a NaN its row or column; a large scale against a small one stays in range."""
    dv = tiled
    M, N, K = 40, 50, 256
    g, a, lda, (b,), ldb, sa, (sb,) = i8_problem(M, N, K, 9)
    sa[3], sa[4], sb[7], sa[5], sb[9] = 0.0, math.nan, math.nan, 1e-36, 1e36
    c = torch.empty(M, N, device="cuda")
    dv.gemm_i8_scaled(a, lda, b, ldb, sa, sb, None, capi.TYPE_F32, c, N, M, N, K)
    prod = (a.double() @ b.double().T) * sa.double()[:, None] * sb.double()[None, :]
    odd = torch.isnan(c)
    assert bool(odd[4].all()) and bool(odd[:, 7].all()) and int(odd.sum()) == M + N - 1
    assert bool((c[3][~odd[3]] == 0).all())
    fine = prod[5, 9]
    assert abs(float(c[5, 9]) - float(fine)) <= 8 * E * abs(float(fine))


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("M, F, K", I8_SIZES)
def test_glu_i8(tiled, type, M, F, K):
    dv = tiled
    dt, act = TYPES[type], ACTS[(M + F) % 4]
    g, a, lda, (bg, bu), ldb, sa, (sg, su) = i8_problem(M, F, K, M + 5 * F + K, ws=2)
    ldh = F + M % 3
    G = (a.double() @ bg.double().T) * sa.double()[:, None] * sg.double()[None, :]
    U = (a.double() @ bu.double().T) * sa.double()[:, None] * su.double()[None, :]
    ref = act64(act, G) * U
    off = (1.13 * 3 * E * G.abs() + act_off(act, G)) * U.abs() + 4 * E * (G * U).abs()
    hb, h = padded(M, F, ldh, dt, -7.0)
    dv.glu_i8(act, a, lda, bg, bu, ldb, sa, sg, su, type, h, ldh, M, F, K)
    within(h, ref, off, dt)
    assert untouched(hb, h, ldh, -7.0)
    again = torch.empty(M, F, dtype=dt, device="cuda")
    dv.glu_i8(act, a, lda, bg, bu, ldb, sa, sg, su, type, again, F, M, F, K)
    assert torch.equal(again, h)


# ---- together, on other streams, in graphs -----------------------------------------------------------------------------

def test_no_rows_is_a_call_that_writes_nothing(dv):
    e = torch.empty(0, device="cuda")
    dv.glu_forward(capi.TYPE_BF16, 0, e, 64, e, e, 64, e, 8, None, None, 0, 0, 8, 64)
    dv.quantize_i8(capi.TYPE_F32, e, 64, e, 128, e, 0, 64, 128)
    dv.gemm_i8_scaled(e, 128, e, 128, e, e, None, capi.TYPE_BF16, e, 8, 0, 8, 128)
    dv.glu_i8(0, e, 128, e, e, 128, e, e, e, capi.TYPE_BF16, e, 8, 0, 8, 128)


@pytest.mark.parametrize("T", [1, 19, 200, 600])
def test_an_8bit_feed_forward_layer(tiled, T):
    """Activations quantised for each token, the gated projection, its result quantised, the projection back: the layer
    as a server runs it, against the same steps in 64 bits on what each step was given, and as a whole against the
    unquantised layer (whose distance is that of the two 8-bit roundings, a percent or so)."""
    dv = tiled
    D, F = 500, 700
    g = gen(T)
    Dp, Fp = 512, 768
    x = torch.randn(T, D, generator=g, device="cuda").bfloat16()
    w = [torch.randn(F, D, generator=g, device="cuda") / math.sqrt(D), torch.randn(F, D, generator=g, device="cuda") / math.sqrt(D),
         torch.randn(D, F, generator=g, device="cuda") / math.sqrt(F)]

    def rows(m, kp, type=capi.TYPE_F32):
        q, s = torch.empty(m.shape[0], kp, dtype=torch.int8, device="cuda"), torch.empty(m.shape[0], device="cuda")
        dv.quantize_i8(type, m, m.shape[1], q, kp, s, m.shape[0], m.shape[1], kp)
        return q, s

    (qg, sg), (qu, su), (qd, sd) = rows(w[0], Dp), rows(w[1], Dp), rows(w[2], Fp)
    qx, sx = rows(x, Dp, capi.TYPE_BF16)
    h = torch.empty(T, F, dtype=torch.bfloat16, device="cuda")
    dv.glu_i8(capi.GLU_SILU, qx, Dp, qg, qu, Dp, sx, sg, su, capi.TYPE_BF16, h, F, T, F, Dp)
    qh, sh = rows(h, Fp, capi.TYPE_BF16)
    y = torch.empty(T, D, dtype=torch.bfloat16, device="cuda")
    n = dv.gemm_i8_scaled_workspace(T, D, Fp)
    dv.gemm_i8_scaled(qh, Fp, qd, Fp, sh, sd, None, capi.TYPE_BF16, y, D, T, D, Fp, torch.empty(n, dtype=torch.uint8, device="cuda") if n else None, n)

    # (the whole numbers are summed before they are scaled: exact, a sum that is 0 stays 0)
    times = lambda a, sa, b, sb: (a.double() @ b.double().T) * sa.double()[:, None] * sb.double()[None, :]  # noqa: E731
    assert torch.equal(qx[:, :D].double(), quantized(x)[0]) and torch.equal(qh[:, :F].double(), quantized(h)[0])
    G, U = times(qx, sx, qg, sg), times(qx, sx, qu, su)
    within(h, act64(capi.GLU_SILU, G) * U, (1.13 * 3 * E * G.abs() + act_off(capi.GLU_SILU, G)) * U.abs() + 4 * E * (G * U).abs(), torch.bfloat16)
    Y = times(qh, sh, qd, sd)
    within(y, Y, 8 * E * Y.abs(), torch.bfloat16)
    whole = (act64(capi.GLU_SILU, x.double() @ w[0].double().T) * (x.double() @ w[1].double().T)) @ w[2].double().T
    assert float((y.double() - whole).norm() / whole.norm()) < 0.05


def test_a_feed_forward_layer_and_its_gradients(dv):
    """The layer as it is trained: gated projection, projection back (this library's plain bf16 product), the gradient of
    the hidden values, the gated projection's gradients.  Every step against 64 bits on what it was given."""
    T, F, D = 256, 384, 128
    dt = torch.bfloat16
    g = gen(8)
    x, wg, wu = operand(g, T, D, D, dt), operand(g, F, D, D, dt, 1 / math.sqrt(D)), operand(g, F, D, D, dt, 1 / math.sqrt(D))
    wd = operand(g, D, F, F, dt, 1 / math.sqrt(F))
    dy = operand(g, T, D, D, dt)
    h, G, U = (torch.empty(T, F, dtype=dt, device="cuda") for _ in range(3))
    y = torch.empty(T, D, dtype=dt, device="cuda")
    dh = torch.empty(T, F, dtype=dt, device="cuda")
    dv.glu_forward(capi.TYPE_BF16, capi.GLU_SILU, x, D, wg, wu, D, h, F, G, U, F, T, F, D)
    dv._check(dv.lib.mi355_gemm_bf16(dv.h, h.data_ptr(), wd.data_ptr(), y.data_ptr(), T, D, F))
    wdt = wd.t().contiguous()
    dv._check(dv.lib.mi355_gemm_bf16(dv.h, dy.data_ptr(), wdt.data_ptr(), dh.data_ptr(), T, F, D))
    n = dv.glu_backward_workspace(T, F, D)
    dx, dwg, dwu = torch.empty(T, D, dtype=dt, device="cuda"), torch.empty(F, D, dtype=dt, device="cuda"), torch.empty(F, D, dtype=dt, device="cuda")
    dv.glu_backward(capi.TYPE_BF16, capi.GLU_SILU, dh, F, x, D, wg, wu, D, G, U, F, dx, D, dwg, dwu, D, T, F, D,
                    torch.empty(n, dtype=torch.uint8, device="cuda"), n)
    d = [v.double().requires_grad_() for v in (x, wg, wu)]
    H = act64(capi.GLU_SILU, d[0] @ d[1].T) * (d[0] @ d[2].T)
    Y = H @ wd.double().T
    Y.backward(dy.double())
    # roundings to bf16 along the way (h; dh, G, U, dG, dU), half a step each, over values of about that size: sums of
    # independent ones, 2^-8 times the root of their number in the norm at most
    assert float((y.double() - Y).norm() / Y.norm()) < math.sqrt(2) * 2.0 ** -8
    for got, ref in zip((dx, dwg, dwu), d):
        assert float((got.double() - ref.grad).norm() / ref.grad.norm()) < math.sqrt(6) * 2.0 ** -8


def test_two_streams_at_once():
    """Two handles on two streams, their calls in flight together, with a workspace each."""
    T, F, D = 384, 640, 512
    n = None
    streams, jobs = [torch.cuda.Stream() for _ in range(2)], []
    for k, st in enumerate(streams):
        g = gen(40 + k)
        x, wg, wu, dh = (operand(g, r, c, c, torch.bfloat16, s) for r, c, s in ((T, D, 1.0), (F, D, 0.05), (F, D, 0.05), (T, F, 1.0)))
        G, U = (x.float() @ wg.float().T).bfloat16(), (x.float() @ wu.float().T).bfloat16()
        d = capi.Device(0, stream=st.cuda_stream)
        n = d.glu_backward_workspace(T, F, D)
        out = [torch.zeros(T, D, dtype=torch.bfloat16, device="cuda")] + [torch.zeros(F, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        jobs.append((d, (dh, F, x, D, wg, wu, D, G, U, F), out, torch.empty(n, dtype=torch.uint8, device="cuda")))
    torch.cuda.synchronize()

    def go(k):
        d, a, o, ws = jobs[k]
        d.glu_backward(capi.TYPE_BF16, capi.GLU_SILU, *a, o[0], D, o[1], o[2], D, T, F, D, ws, n)

    want = []
    for k in range(2):
        go(k)
        torch.cuda.synchronize()
        want.append([o.clone() for o in jobs[k][2]])
    for _ in range(5):
        for k in range(2):
            go(k)
            go(k)
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(o, w) for o, w in zip(jobs[k][2], want[k]))
        jobs[k][0].close()


@pytest.mark.parametrize("T", [1, 40, 300])
def test_captured_and_replayed(T):
    """All five operators on a fresh handle in one graph, replayed on changed inputs with eager work in between: every
    replay gives the eager calls' bits."""
    F, D = 384, 512
    st = torch.cuda.Stream()
    d = capi.Device(0, stream=st.cuda_stream)
    g = gen(60)
    x = torch.empty(T, D, dtype=torch.bfloat16, device="cuda")
    wg, wu = operand(g, F, D, D, torch.bfloat16, 0.05), operand(g, F, D, D, torch.bfloat16, 0.05)
    qw, sw = torch.randint(-127, 128, (2, F, D), generator=g, device="cuda").to(torch.int8), torch.rand(2, F, generator=g, device="cuda") * 1e-3
    new = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    h, G, U, dx, dwg, dwu = new(T, F), new(T, F), new(T, F), new(T, D), new(F, D), new(F, D)
    q, s, h8, c = new(T, D, dtype=torch.int8), new(T, dtype=torch.float32), new(T, F), new(T, F)
    n, m = d.glu_backward_workspace(T, F, D), d.gemm_i8_scaled_workspace(T, F, D)
    ws, ws8 = new(n, dtype=torch.uint8), new(max(m, 16), dtype=torch.uint8)

    def calls():
        d.glu_forward(capi.TYPE_BF16, capi.GLU_SILU, x, D, wg, wu, D, h, F, G, U, F, T, F, D)
        d.glu_backward(capi.TYPE_BF16, capi.GLU_SILU, h, F, x, D, wg, wu, D, G, U, F, dx, D, dwg, dwu, D, T, F, D, ws, n)
        d.quantize_i8(capi.TYPE_BF16, x, D, q, D, s, T, D, D)
        d.glu_i8(capi.GLU_SILU, q, D, qw[0], qw[1], D, s, sw[0], sw[1], capi.TYPE_BF16, h8, F, T, F, D)
        d.gemm_i8_scaled(q, D, qw[0], D, s, sw[0], None, capi.TYPE_BF16, c, F, T, F, D, ws8, m)

    outs = (h, G, U, dx, dwg, dwu, q, s, h8, c)
    x.normal_(generator=g)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        calls()
    for k in range(4):
        x.normal_(generator=g)
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        assert all(bool(o.float().abs().sum() > 0) for o in got)
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        calls()
        d.sync()
        assert all(torch.equal(a, b) for a, b in zip(got, outs)), k
    del graph
    d.close()


def test_a_borrowed_stream_survives_its_handle():
    st = torch.cuda.Stream()
    for _ in range(2):
        d = capi.Device(0, stream=st.cuda_stream)
        x = torch.randn(4, 128, device="cuda")
        st.wait_stream(torch.cuda.current_stream())
        q, s = torch.empty(4, 128, dtype=torch.int8, device="cuda"), torch.empty(4, device="cuda")
        d.quantize_i8(capi.TYPE_F32, x, 128, q, 128, s, 4, 128, 128)
        d.close()
        st.synchronize()
        assert torch.equal(q.double(), quantized(x)[0])


@pytest.mark.parametrize("type", list(TYPES))
def test_quantize_rows_whose_largest_is_a_multiple_of_127(dv, type):
    """amax = 127 c 2^n: there whole families of values lie exactly on a border, and 127 / amax is exact for powers of two c
    only.  Every value of the type up to amax is tried (fp32: a step of 2^-10 of amax)."""
    dt = TYPES[type]
    for c in range(1, 17):
        for n in (-9, 0, 5):
            top = 127 * c * 2.0 ** n
            if float(torch.tensor(top).to(dt)) != top:
                continue
            if dt == torch.float32:
                x = torch.arange(0, 1025, dtype=torch.float64) * top / 1024
            else:
                x = torch.arange(0, 1 << 15, dtype=torch.int32).to(torch.int16).view(dt).double()
                x = x[x <= top]
            x = torch.cat((x, -x)).to(dt)[None].cuda()
            K = x.shape[1]
            q, s = torch.empty(1, K, dtype=torch.int8, device="cuda"), torch.empty(1, device="cuda")
            dv.quantize_i8(type, x, K, q, K, s, 1, K, K)
            rq, rs = quantized(x)
            assert torch.equal(q.double(), rq) and torch.equal(s, rs), (c, n)


@pytest.mark.parametrize("type", [capi.TYPE_BF16, capi.TYPE_F16])
def test_quantize_every_value_against_every_mantissa(dv, type):
    """Every mantissa amax can have (128 of bf16, every fifth of the 1024 of fp16) against every value of the type that is
    no larger and no smaller than amax / 512."""
    dt = TYPES[type]
    bits = torch.arange(0, 1 << 15, dtype=torch.int32, device="cuda").to(torch.int16).view(dt)
    vals = bits[torch.isfinite(bits)]
    tops = vals[(vals >= 16.0) & (vals < 32.0)][:: 1 if type == capi.TYPE_BF16 else 5]
    vals = vals[(vals >= 1 / 32) & (vals < 32.0)]
    x = torch.where(vals[None] <= tops[:, None], vals[None], torch.zeros_like(vals)[None]).contiguous()
    x[:, 1::2] *= -1
    x = torch.cat((x, tops[:, None]), 1).contiguous()
    M, K = x.shape
    q, s = torch.empty(M, K, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    dv.quantize_i8(type, x, K, q, K, s, M, K, K)
    rq, rs = quantized(x)
    assert torch.equal(q.double(), rq) and torch.equal(s, rs)


# ---- where offsets, values and calls are unusual ------------------------------------------------------------------------

@pytest.mark.parametrize("M", [3, 70])
def test_operands_whose_rows_are_far_apart(tiled, M):
    """Rows 64 MiB apart, the most that is taken: the last of 70 is more than 4 GiB behind the first."""
    dv = tiled
    N, K, far = 70, 256, 64 << 20
    g = gen(M)
    a, b, b2 = (torch.randint(-128, 128, (r, K), generator=g, device="cuda").to(torch.int8) for r in (M, N, N))
    big = torch.empty((N - 1) * far + 2 * K, dtype=torch.int8, device="cuda")
    rows, rows2 = big.as_strided((N, K), (far, 1)), big.as_strided((N, K), (far, 1), K)
    rows.copy_(b)
    rows2.copy_(b2)
    one = torch.ones(N, device="cuda")
    c = torch.empty(M, N, device="cuda")
    dv.gemm_i8_scaled(a, K, rows, far, one, one, None, capi.TYPE_F32, c, N, M, N, K)
    assert torch.equal(c.double(), a.double() @ b.double().T)
    dv.glu_i8(capi.GLU_RELU, a, K, rows, rows2, far, one, one, one, capi.TYPE_F32, c, N, M, N, K)
    want = (a.double() @ b.double().T).clamp(min=0) * (a.double() @ b2.double().T)
    within(c, want, 4 * E * want.abs(), torch.float32)
    dv.gemm_i8_scaled(rows, far, a, K, one, one, None, capi.TYPE_F32, c.view(N, M), M, N, M, K)
    assert torch.equal(c.view(N, M).double(), b.double() @ a.double().T)
    D = 64
    x = (torch.randn(N, D, generator=g, device="cuda")).bfloat16()
    w = (torch.randn(2, M, D, generator=g, device="cuda") / 8).bfloat16()
    xs = big.view(torch.bfloat16).as_strided((N, D), (far // 2, 1))
    xs.copy_(x)
    h, G, U = (torch.empty(N, M, dtype=torch.bfloat16, device="cuda") for _ in range(3))
    dv.glu_forward(capi.TYPE_BF16, capi.GLU_RELU, xs, far // 2, w[0], w[1], D, h, M, G, U, M, N, M, D)
    g64, u64 = x.double() @ w[0].double().T, x.double() @ w[1].double().T
    s = 2 * D * E * (x.double().abs() @ w.double().abs().amax(0).T)
    within(h, g64.clamp(min=0) * u64, s * (g64.abs() + u64.abs()), torch.bfloat16)
    n = dv.glu_backward_workspace(N, M, D)
    dw = torch.empty(2, M, D, dtype=torch.bfloat16, device="cuda")
    dv.glu_backward(capi.TYPE_BF16, capi.GLU_RELU, h, M, xs, far // 2, None, None, D, G, U, M, None, D, dw[0], dw[1], D, N, M, D,
                    torch.empty(n, dtype=torch.uint8, device="cuda"), n)
    dU = h.double() * G.double().clamp(min=0)
    within(dw[1], dU.T @ x.double(), (UNIT[torch.bfloat16] + 2 * N * E) * (dU.abs().T @ x.double().abs()), torch.bfloat16)


def test_outputs_whose_rows_are_far_apart(tiled):
    """Rows of 2^31 elements: the second one's bytes are past 32 bits."""
    dv = tiled
    M, N, K, far = 3, 40, 128, 1 << 31
    g = gen(2)
    a, b = (torch.randint(-128, 128, (r, K), generator=g, device="cuda").to(torch.int8) for r in (M, N))
    one = torch.ones(N, device="cuda")
    big = torch.empty((M - 1) * far + 64, dtype=torch.bfloat16, device="cuda")
    c = big.as_strided((M, N), (far, 1))
    c.zero_()
    dv.gemm_i8_scaled(a, K, b, K, one, one, None, capi.TYPE_BF16, c, far, M, N, K)
    ref = a.double() @ b.double().T
    within(c, ref, 4 * E * ref.abs(), torch.bfloat16)
    c.zero_()
    dv.glu_i8(capi.GLU_RELU, a, K, b, b, K, one, one, one, capi.TYPE_BF16, c, far, M, N, K)     # (the same weights twice)
    want = ref.clamp(min=0) * ref
    within(c, want, 4 * E * want.abs(), torch.bfloat16)
    # as inputs of the quantiser and of the gradients
    q, s = torch.empty(M, N, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    dv.quantize_i8(capi.TYPE_BF16, c, far, q, N, s, M, N, N)
    assert torch.equal(q.double(), quantized(c)[0])
    c.copy_(torch.randn(M, N, generator=g, device="cuda"))
    D = 64
    w = torch.randn(N, D, generator=g, device="cuda").bfloat16()
    dx = torch.empty(M, D, dtype=torch.bfloat16, device="cuda")
    n = dv.glu_backward_workspace(M, N, D)
    dv.glu_backward(capi.TYPE_BF16, capi.GLU_RELU, c, far, None, D, w, w, D, c, c, far, dx, D, None, None, D, M, N, D, torch.empty(n, dtype=torch.uint8, device="cuda"), n)
    v = c.double()
    d = torch.where(v > 0, v * v, 0.0)                       # dG and dU of relu with dH = G = U
    within(dx, 2 * d @ w.double(), 2 * (UNIT[torch.bfloat16] + 4 * N * E) * (d.abs() @ w.double().abs()), torch.bfloat16)


def test_a_product_out_of_the_types_range_is_infinite(tiled):
    """fp16 holds 65504: what is past half a step above is infinity, with its sign, and nothing else changes."""
    dv = tiled
    T, F, D = 80, 90, 64
    x = torch.zeros(T, D, dtype=torch.float16, device="cuda")
    x[:, 0] = torch.linspace(-300, 300, T, device="cuda")
    wg, wu = torch.zeros(F, D, dtype=torch.float16, device="cuda"), torch.zeros(F, D, dtype=torch.float16, device="cuda")
    wg[:, 0] = 1.0
    wu[:, 0] = torch.linspace(-2, 2, F, device="cuda")
    h = torch.empty(T, F, dtype=torch.float16, device="cuda")
    dv.glu_forward(capi.TYPE_F16, capi.GLU_RELU, x, D, wg, wu, D, h, F, None, None, 0, T, F, D)
    g64 = x.double()[:, :1]
    ref = g64.clamp(min=0) * (g64 * wu.double()[:, 0][None])
    assert bool(torch.isinf(h).any())
    assert torch.equal(h, ref.to(torch.float16))             # two roundings in fp32, exact here: 11-bit factors


def test_a_refused_call_leaves_the_handle_usable(dv):
    x = torch.randn(4, 256, device="cuda")
    q, s = torch.full((4, 256), 5, dtype=torch.int8, device="cuda"), torch.zeros(4, device="cuda")
    with pytest.raises(capi.Mi355Error) as e:
        dv.quantize_i8(capi.TYPE_F32, x, 100, q, 256, s, 4, 256, 256)
    assert e.value.code == capi.ERR_ARG and "do not fit" in str(e.value)
    assert bool((q == 5).all())
    dv.quantize_i8(capi.TYPE_F32, x, 256, q, 256, s, 4, 256, 256)
    assert torch.equal(q.double(), quantized(x)[0])
    n = dv.glu_backward_workspace(300, 400, 128)
    with pytest.raises(capi.Mi355Error) as e:
        dv.glu_backward(capi.TYPE_BF16, 0, x, 400, x, 128, x, x, 128, x, x, 400, x, 128, x, x, 128, 300, 400, 128, torch.empty(n, dtype=torch.uint8, device="cuda"), n - 1)
    assert "are needed" in str(e.value)


def test_the_handles_own_stream():
    """A handle that owns its stream: its calls are in order among themselves and wait for mi355_sync."""
    d = capi.Device(0)
    M, K = 33, 512
    x = torch.randn(M, K, device="cuda")
    torch.cuda.synchronize()
    w = torch.randint(-127, 128, (40, K), device="cuda").to(torch.int8)
    q, s, one, c = d.alloc(M * K), d.alloc(M * 4), torch.ones(40, device="cuda"), d.alloc(M * 40 * 4)
    torch.cuda.synchronize()
    d.quantize_i8(capi.TYPE_F32, x, K, q, K, s, M, K, K)
    d.gemm_i8_scaled(q, K, w, K, s, one, None, capi.TYPE_F32, c, 40, M, 40, K)
    d.sync()
    got = torch.from_numpy(c.download(np.float32, M * 40)).view(M, 40).cuda()
    rq, rs = quantized(x)
    ref = (rq @ w.double().T) * rs.double()[:, None]
    within(got, ref, 4 * E * ref.abs(), torch.float32)
    for b in (q, s, c):
        b.free()
    d.close()


@pytest.mark.parametrize("M", [(1 << 21) - 1, 1 << 21, (1 << 22) + 5])
def test_quantize_more_rows_than_a_launch_takes(dv, M):
    K, ldx, ldq = 13, 14, 16
    x = torch.randn(M, ldx, generator=gen(M), device="cuda").to(torch.bfloat16)
    q, s = torch.full((M, ldq), 77, dtype=torch.int8, device="cuda"), torch.empty(M + 1, device="cuda").fill_(-1.0)
    dv.quantize_i8(capi.TYPE_BF16, x, ldx, q, ldq, s, M, K, K)
    rq, rs = quantized(x[:, :K])
    assert torch.equal(q[:, :K].double(), rq) and torch.equal(s[:-1], rs) and s[-1] == -1
    assert bool((q[:, K:] == 77).all())
