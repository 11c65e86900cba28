"""What the entry points do on the host, on a HIP runtime without a GPU (tests/hip_stub.cpp), in a process of their own."""
import json
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PRELUDE = """
import ctypes as C, json, sys
stub = C.CDLL(%r, mode=C.RTLD_GLOBAL)
stub.stub_stream.restype = C.c_void_p
sys.path.insert(0, %r)
from clpeak_amd import capi
P = 1 << 20        # an address that nothing reads
def counts():
    a = (C.c_int * 4)()
    stub.stub_counts(a)
    return dict(zip(("launches", "refused", "wrong_device", "big_lds"), a))
def gradients(d, type, T, F, D, dx=True, dw=True):
    n = d.glu_backward_workspace(T, F, D)
    d.glu_backward(type, 0, P, F, P, D, P, P, D, P, P, F, P if dx else None, D, P if dw else None, P if dw else None, D, T, F, D, P, n)
"""


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("hip") / "hip_stub.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-Wno-deprecated-declarations",
                    os.path.join(ROOT, "tests", "hip_stub.cpp"), "-o", so], check=True, capture_output=True, timeout=300)

    def run(code):
        r = subprocess.run([sys.executable, "-c", PRELUDE % (so, ROOT) + code], capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stderr[-3000:]
        return json.loads(r.stdout.splitlines()[-1])
    return run


# One call for each kernel that takes more than 64 KiB of LDS, by name.
LDS_CALLS = """
def tiled(d, tiling, call):
    d.gemm_tiling(tiling)
    call()
    d.gemm_tiling(capi.GEMM_TILING_AUTO)
def glu(d, type, T):
    d.glu_forward(type, 0, P, 128, P, P, 128, P, 512, None, None, 0, T, 512, 128)
def i8(d, type, ws):
    n = d.gemm_i8_scaled_workspace(512, 512, 16384) if ws else 0
    d.gemm_i8_scaled(P, 16384, P, 16384, P, P, None, type, P, 512, 512, 512, 16384, P if ws else None, n)
def glu_i8(d, type):
    d.glu_i8(0, P, 128, P, P, 128, P, P, P, type, P, 512, 512, 512, 128)
raw = lambda d, name, *a: d._check(getattr(d.lib, "mi355_" + name)(d.h, *a))
big, mid, low, tall = capi.GEMM_TILING_256, capi.GEMM_TILING_128, capi.GEMM_TILING_64, capi.GEMM_TILING_256X128
calls = {"f32": lambda d: raw(d, "gemm_f32", P, P, P, 512, 512, 512)}
for t in (big, mid):
    for name, more in (("gemm_bf16", ()), ("gemm_f16", ()), ("gemm_i8", ()), ("gemm_fp8_e4m3", (1.0, 1.0)), ("gemm_fp8_e5m2", (1.0, 1.0))):
        calls["%s %d" % (name, t)] = lambda d, t=t, name=name, more=more: tiled(d, t, lambda: raw(d, name, P, P, P, 512, 512, 512, *more))
calls["mxfp4"] = lambda d: raw(d, "gemm_mxfp4", P, P, P, P, P, 512, 512, 512)
for t in (big, mid, low, tall):
    for type in (0, 1):
        calls["glu %d %d" % (type, t)] = lambda d, t=t, type=type: tiled(d, t, lambda: glu(d, type, 512))
        calls["gradients %d %d" % (type, t)] = lambda d, t=t, type=type: tiled(d, t, lambda: gradients(d, type, 512, 512, 512))
        calls["dW in slices %d %d" % (type, t)] = lambda d, t=t, type=type: tiled(d, t, lambda: gradients(d, type, 8192, 256, 256, dx=False))
        calls["dX in slices %d %d" % (type, t)] = lambda d, t=t, type=type: tiled(d, t, lambda: gradients(d, type, 256, 8192, 256, dw=False))
    for type in (0, 1, 2):
        calls["int8 %d %d" % (type, t)] = lambda d, t=t, type=type: tiled(d, t, lambda: i8(d, type, False))
        calls["int8 in slices %d %d" % (type, t)] = lambda d, t=t, type=type: tiled(d, t, lambda: i8(d, type, True))
        calls["gated int8 %d %d" % (type, t)] = lambda d, t=t, type=type: tiled(d, t, lambda: glu_i8(d, type))
"""


def test_every_kernel_that_takes_a_whole_cus_lds_is_allowed_to_whatever_ran_before(stub):
    """Every ordered pair of such calls on a handle of its own: no launch asks for more LDS than its kernel was allowed."""
    got = stub(LDS_CALLS + """
pairs = {}
for a in calls:
    for b in calls:
        d = capi.Device(0)
        before = counts()["refused"]
        stub.stub_forget()
        calls[a](d)
        calls[b](d)
        if counts()["refused"] != before:
            pairs[a + ", " + b] = counts()["refused"] - before
        d.close()
print(json.dumps({"pairs": pairs, "counts": counts(), "calls": len(calls)}))
""")
    assert got["calls"] == 80 and got["counts"]["big_lds"] >= 2 * got["calls"] ** 2
    assert got["pairs"] == {}


def test_dW_of_a_training_batch_and_the_fp8_product(stub):
    """The library's own choices: the sums of dW in slices in fp16, then the fp8 product on 256x256 tiles, and the other way."""
    got = stub("""
seen = []
for order in (0, 1):
    stub.stub_forget()
    d = capi.Device(0)
    one = lambda: gradients(d, capi.TYPE_F16, 8192, 1024, 4096)
    two = lambda: d._check(d.lib.mi355_gemm_fp8_e4m3(d.h, P, P, P, 8192, 8192, 8192, 1.0, 1.0))
    for call in ((one, two) if order else (two, one)):
        call()
    seen.append(counts()["refused"])
print(json.dumps(seen))
""")
    assert got == [0, 0]


def test_calls_leave_the_current_device_as_they_found_it(stub):
    """A program with torch on one GPU and a handle on another: what the handle launches runs on its device, refused calls and
    errors included, and the thread's current device is the program's again afterwards."""
    got = stub(LDS_CALLS + """
moved, n = [], 0
def check(what, at):
    global n
    n += 1
    if stub.stub_current() != at:
        moved.append([what, at, stub.stub_current()])
        stub.stub_make_current(at)
for at in (0, 1):
    for on in (0, 1):
        for borrowed in (False, True, None):
            stub.stub_make_current(at)
            d = capi.Device(on, stream=None if borrowed is None else stub.stub_stream(on) if borrowed else 0)
            check("open", at)
            for name, call in calls.items():
                call(d)
                check(name, at)
            d.quantize_i8(0, P, 128, P, 128, P, 5, 128, 128)
            check("quantize_i8", at)
            b = d.alloc(4096)
            check("alloc", at)
            d._check(d.lib.mi355_memset(d.h, P, 0, 64))
            check("memset", at)
            d.fill_f32(b, 64, 1, 0, 0)
            check("fill_f32", at)
            d.timer_start(); check("timer_start", at)
            d.timer_stop(); check("timer_stop", at)
            d.sync(); check("sync", at)
            try:
                d.glu_forward(7, 0, P, 128, P, P, 128, P, 512, None, None, 0, 5, 512, 128)
            except capi.Mi355Error:
                check("refused", at)
            try:
                raw(d, "gemm_bf16", P, P, P, 100, 100, 100)
            except capi.Mi355Error:
                check("refused later", at)
            b.free()
            check("free", at)
            d.close()
            check("close", at)
try:
    capi.Device(5)
except capi.Mi355Error:
    check("open of no device", 1)
print(json.dumps({"moved": moved[:10], "all": len(moved), "checked": n, "counts": counts()}))
""")
    assert got["checked"] > 12 * 85 and got["counts"]["launches"] > 12 * 85
    assert got["moved"] == [] and got["all"] == 0
    assert got["counts"]["wrong_device"] == 0


def test_tensors_that_a_call_cannot_take_are_refused_before_it(stub):
    """Each buffer of each Python call in turn: a tensor in host memory, on another GPU, of another type; a workspace shorter
    than said; buffers of a handle on another GPU.  Nothing is launched.  The same calls with tensors that fit go through."""
    got = stub("""
import torch
class Tensor:      # as much of a tensor as is looked at
    def __init__(self, dtype, gpu=0, nbytes=1 << 30):
        self.dtype, self.gpu, self.nbytes, self.device = dtype, gpu, nbytes, "cuda:%d" % gpu
    def get_device(self):
        return self.gpu
    def data_ptr(self):
        return P
d, other = capi.Device(0), capi.Device(1)
h, i8, f32 = torch.float16, torch.int8, torch.float32
calls = {
    "glu_forward": (lambda X, Wg, Wu, H, G, U: d.glu_forward(1, 0, X, 128, Wg, Wu, 128, H, 64, G, U, 64, 5, 64, 128), [h] * 6),
    "glu_backward": (lambda dH, X, Wg, Wu, G, U, dX, dWg, dWu, ws: d.glu_backward(1, 0, dH, 64, X, 128, Wg, Wu, 128, G, U, 64, dX, 128, dWg, dWu, 128, 5, 64, 128, ws,
                     d.glu_backward_workspace(5, 64, 128)), [h] * 9 + [None]),
    "quantize_i8": (lambda X, Q, scale: d.quantize_i8(1, X, 128, Q, 128, scale, 5, 128, 128), [h, i8, f32]),
    "gemm_i8_scaled": (lambda A, B, sa, sb, bias, C, ws: d.gemm_i8_scaled(A, 128, B, 128, sa, sb, bias, 1, C, 64, 5, 64, 128, ws, 64), [i8, i8, f32, f32, f32, h, None]),
    "glu_i8": (lambda A, Bg, Bu, sa, sg, su, H: d.glu_i8(0, A, 128, Bg, Bu, 128, sa, sg, su, 1, H, 64, 5, 64, 128), [i8, i8, i8, f32, f32, f32, h]),
}
fits = lambda t: Tensor(t or torch.uint8)
passed, refused, wrong = 0, 0, []
for name, (call, types) in calls.items():
    for buffers in ([fits(t) for t in types], [P] * len(types), [d.alloc(1 << 20) for _ in types]):
        before = counts()["launches"]
        call(*buffers)
        passed += counts()["launches"] > before
    for k, t in enumerate(types):
        bad = [torch.zeros(64, dtype=t or torch.uint8), Tensor(t or torch.uint8, gpu=1), other.alloc(1 << 20)]
        bad.append(Tensor(torch.bfloat16 if t in (h, f32) else torch.uint8) if t else Tensor(torch.uint8, nbytes=63))
        for b in bad:
            before = counts()["launches"]
            try:
                call(*[b if j == k else fits(u) for j, u in enumerate(types)])
                wrong.append([name, k, "taken"])
            except capi.Mi355Error as e:
                refused += 1
                if e.code != capi.ERR_ARG or name + ":" not in str(e):
                    wrong.append([name, k, str(e)])
            if counts()["launches"] != before:
                wrong.append([name, k, "launched"])
# no rows: nothing is looked at
f = Tensor(torch.float64, gpu=1)
d.glu_forward(1, 0, f, 128, f, f, 128, f, 64, f, f, 64, 0, 64, 128)
d.quantize_i8(1, f, 128, f, 128, f, 0, 128, 128)
d.gemm_i8_scaled(f, 128, f, 128, f, f, f, 1, f, 64, 0, 64, 128)
d.glu_i8(0, f, 128, f, f, 128, f, f, f, 1, f, 64, 0, 64, 128)
d.glu_backward(1, 0, f, 64, f, 128, f, f, 128, f, f, 64, f, 128, fits(h), fits(h), 128, 0, 64, 128, P, d.glu_backward_workspace(0, 64, 128))
print(json.dumps({"passed": passed, "refused": refused, "wrong": wrong}))
""")
    assert got["wrong"] == []
    assert got["passed"] == 15 and got["refused"] == 4 * 33
