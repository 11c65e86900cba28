"""What the feed-forward entry points refuse, and that they do so before any HIP call: a handle with no device behind it
(tests/ffn_handle.cpp) on a machine without a GPU.  A call that passes its checks comes back with MI355_ERR_HIP there."""
import ctypes as C
import os
import subprocess

import pytest

from clpeak_amd import capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20            # an aligned address that nothing reads


@pytest.fixture(scope="module")
def lib():
    lib = capi.load_library()
    n = C.c_int(-1)
    if lib.mi355_device_count(C.byref(n)) == capi.OK and n.value > 0:
        pytest.skip("a GPU is present: calls with made-up addresses are for machines without one")
    return lib


@pytest.fixture(scope="module")
def handle(lib, tmp_path_factory):
    so = tmp_path_factory.mktemp("handle") / "ffn_handle.so"
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    os.path.join(ROOT, "tests", "ffn_handle.cpp"), "-o", str(so)], check=True, capture_output=True, timeout=300)
    make = C.CDLL(str(so)).ffn_test_handle
    make.restype = C.c_void_p
    return make()


def forward(**k):
    a = dict(type=0, act=0, X=P, ldx=128, Wg=P, Wu=P, ldw=128, H=P, ldh=33, G=P, U=P, ldg=33, T=5, F=33, D=128)
    a.update(k)
    return "mi355_glu_forward", list(a.values())


def backward(**k):
    a = dict(type=0, act=0, dH=P, lddh=33, X=P, ldx=128, Wg=P, Wu=P, ldw=128, G=P, U=P, ldg=33, dX=P, lddx=128, dWg=P, dWu=P, lddw=128,
             T=5, F=33, D=128, ws=P, bytes=1 << 40)
    a.update(k)
    return "mi355_glu_backward", list(a.values())


def quantize(**k):
    a = dict(type=0, X=P, ldx=100, Q=P, ldq=128, scale=P, M=3, K=100, k_pad=128)
    a.update(k)
    return "mi355_quantize_i8", list(a.values())


def product(**k):
    a = dict(A=P, lda=256, B=P, ldb=256, sa=P, sb=P, bias=P, type=0, C=P, ldc=33, M=5, N=33, K=256, ws=None, bytes=0)
    a.update(k)
    return "mi355_gemm_i8_scaled", list(a.values())


def glu_i8(**k):
    a = dict(act=0, A=P, lda=256, Bg=P, Bu=P, ldb=256, sa=P, sg=P, su=P, type=0, H=P, ldh=33, M=5, F=33, K=256)
    a.update(k)
    return "mi355_glu_i8", list(a.values())


GOOD = [
    forward(), forward(type=1, act=3), forward(G=None, U=None, ldg=0), forward(H=P + 2, ldh=35), forward(T=1, F=1, D=64, ldx=64, ldw=64),
    forward(D=33554432, ldx=33554432, ldw=33554432),
    backward(), backward(dX=None), backward(dX=None, Wg=None, Wu=None), backward(dWg=None, dWu=None), backward(dWg=None, dWu=None, X=None),
    backward(T=0, dH=None, G=None, U=None, X=None, Wg=None, Wu=None, dX=None),
    quantize(), quantize(type=2, X=P + 4, Q=P + 1), quantize(X=P + 2, k_pad=100, ldq=100), quantize(M=1, K=1, k_pad=1),
    product(), product(bias=None), product(type=2, C=P + 4), product(K=130944, lda=130944, ldb=130944), product(ws=P, bytes=16),
    glu_i8(), glu_i8(type=2, act=2),
]
# no rows: nothing to do, and nothing is looked at
NOTHING = [
    forward(T=0, X=None, H=None, G=None, U=None), quantize(M=0, X=None, Q=None, scale=None), product(M=0, A=None, sa=None, C=None),
    glu_i8(M=0, A=None, sa=None, H=None), backward(dX=None, dWg=None, dWu=None, ws=None, bytes=0), backward(T=0, dWg=None, dWu=None, ws=None, bytes=0),
]
BAD = [
    forward(type=2), forward(type=-1), forward(act=4), forward(act=-1), forward(F=0), forward(D=0), forward(D=96), forward(D=32, ldx=64, ldw=64),
    forward(X=None), forward(X=P + 8), forward(ldx=64), forward(ldx=129), forward(ldx=1 << 40), forward(Wg=None), forward(Wu=None), forward(Wu=P + 2),
    forward(ldw=0), forward(H=None), forward(H=P + 1), forward(ldh=32), forward(G=None), forward(U=None), forward(G=P + 1), forward(ldg=32),
    forward(T=(1 << 30) + 1), forward(F=(1 << 30) + 1), forward(D=33554432 + 64, ldx=33554432 + 64, ldw=33554432 + 64), forward(ldh=(1 << 40) + 1),
    backward(type=2), backward(act=9), backward(dH=None), backward(lddh=32), backward(G=None), backward(U=None), backward(ldg=1), backward(X=None),
    backward(Wg=None), backward(ldw=120), backward(dWg=None), backward(dWu=None), backward(lddw=127), backward(lddx=127), backward(dX=P + 1),
    backward(ws=None), backward(ws=P + 128), backward(bytes=1000), backward(T=(1 << 25) + 1), backward(F=1 << 24), backward(D=0), backward(F=0),
    backward(X=P + 8), backward(ldx=132),
    quantize(type=3), quantize(type=-1), quantize(X=None), quantize(Q=None), quantize(scale=None), quantize(K=0), quantize(k_pad=99),
    quantize(ldx=99), quantize(ldq=127), quantize(X=P + 1), quantize(type=2, X=P + 2), quantize(scale=P + 2), quantize(M=1 << 31),
    quantize(K=(1 << 30) + 1, k_pad=(1 << 30) + 1, ldx=1 << 31, ldq=1 << 31), quantize(ldx=(1 << 40) + 1), quantize(k_pad=1 << 31, ldq=1 << 31),
    product(type=3), product(A=None), product(A=P + 8), product(lda=128), product(lda=264), product(B=None), product(B=P + 4), product(ldb=255),
    product(sa=None), product(sb=None), product(sa=P + 1), product(sb=P + 2), product(bias=P + 1), product(C=None), product(type=2, C=P + 2),
    product(ldc=32), product(N=0), product(K=0), product(K=192), product(K=131072, lda=131072, ldb=131072), product(ws=P + 8, bytes=64),
    product(M=(1 << 30) + 1), product(N=(1 << 30) + 1), product(N=(1 << 26) + 1, ldc=1 << 27), forward(F=(1 << 26) + 1, ldh=1 << 27, ldg=1 << 27),
    glu_i8(act=4), glu_i8(type=5), glu_i8(A=None), glu_i8(Bg=None), glu_i8(Bu=P + 8), glu_i8(sg=None), glu_i8(su=None), glu_i8(sa=None),
    glu_i8(H=None), glu_i8(ldh=10), glu_i8(F=0), glu_i8(K=64), glu_i8(K=131072, lda=131072, ldb=131072), glu_i8(ldb=128), glu_i8(H=P + 1),
]


def _id(call):
    return "%s-%d" % (call[0][6:], abs(hash(str(call[1]))) % 9973)


@pytest.mark.parametrize("call", GOOD, ids=_id)
def test_accepted(lib, handle, call):
    rc = getattr(lib, call[0])(handle, *call[1])
    assert rc == capi.ERR_HIP, (rc, lib.mi355_last_error(handle))


@pytest.mark.parametrize("call", NOTHING, ids=_id)
def test_nothing_to_do(lib, handle, call):
    assert getattr(lib, call[0])(handle, *call[1]) == capi.OK, lib.mi355_last_error(handle)


@pytest.mark.parametrize("call", BAD, ids=_id)
def test_refused(lib, handle, call):
    rc = getattr(lib, call[0])(handle, *call[1])
    text = lib.mi355_last_error(handle).decode()
    assert rc == capi.ERR_ARG, (rc, text)
    assert text.startswith(call[0][6:] + ":"), text
    assert getattr(lib, call[0])(None, *call[1]) == capi.ERR_ARG


def test_workspaces(lib, handle):
    n = C.c_size_t(7)
    assert lib.mi355_glu_backward_workspace(handle, 5, 33, 128, C.byref(n)) == capi.OK
    need = n.value
    assert lib.mi355_glu_backward(handle, *backward(bytes=need)[1]) == capi.ERR_HIP
    assert lib.mi355_glu_backward(handle, *backward(bytes=need - 1)[1]) == capi.ERR_ARG
    # what the passes before the products write: dG and dU both ways and the operands turned
    assert need >= 2 * (2 * 5 * 33 * 2 + 128 * 2 * 33 + 128 * 5)
    assert lib.mi355_glu_backward_workspace(handle, 1 << 25, (1 << 24) - 64, 64, C.byref(n)) == capi.OK and n.value > 1 << 50
    assert lib.mi355_glu_backward_workspace(handle, 0, 33, 128, C.byref(n)) == capi.OK
    for T, F, D in [(5, 0, 128), (5, 33, 0), (5, 33, 100), ((1 << 25) + 1, 33, 128), (5, 1 << 24, 128)]:
        assert lib.mi355_glu_backward_workspace(handle, T, F, D, C.byref(n)) == capi.ERR_ARG and n.value == 0
    assert lib.mi355_glu_backward_workspace(handle, 5, 33, 128, None) == capi.ERR_ARG
    assert lib.mi355_gemm_i8_scaled_workspace(handle, 5, 33, 256, None) == capi.ERR_ARG
    assert lib.mi355_gemm_i8_scaled_workspace(handle, 5, 33, 100, C.byref(n)) == capi.ERR_ARG
    assert lib.mi355_gemm_i8_scaled_workspace(handle, 0, 33, 128, C.byref(n)) == capi.OK and n.value == 0


def test_a_stream_of_no_device_is_an_error(lib):
    h = C.c_void_p()
    assert lib.mi355_open_on_stream(0, None, C.byref(h)) in (capi.ERR_NODEV, capi.ERR_HIP)
    assert lib.mi355_open_on_stream(0, None, None) == capi.ERR_ARG
