"""Cases of the feed-forward operators: the gated projection with its gradients in 16 bits, and its 8-bit integer serving form.

  glu         H = act(X Wg^T) * (X Wu^T), with G = X Wg^T and U = X Wu^T where a backward pass follows
  glu_grad    dX, dWg, dWu of that, from dH, X, the weights and the kept G and U
  quant       every row to int8 with its scale: s = amax / 127, q = 127 x / amax rounded to nearest even
  gemm_i8     C[m][n] = sa[m] sb[n] (A B^T)[m][n] + bias[n], int8 operands with a scale for each token and channel
  glu_i8      H = act(sa sg (A Bg^T)) * (sa su (A Bu^T)) on the same kind of operands

`own` chooses between the plain form of each (elementary torch operations in 32 bits, one rounding at the end) and the
calls of this package.  exact() evaluates the definitions in 64 bits.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_devices = {}


def listed():
    return [
        # one token of a stream being generated, through the gated half of a block
        {"name": "glu 1 token", "op": "glu", "type": "bf16", "act": "silu", "T": 1, "F": 8192, "D": 4096, "keep": False},
        # a short ragged batch; odd numbers of tokens and of channels
        {"name": "glu ragged", "op": "glu", "type": "f16", "act": "gelu", "T": 333, "F": 2731, "D": 1024, "keep": True},
        # a training batch's forward pass
        {"name": "glu batch", "op": "glu", "type": "bf16", "act": "silu", "T": 8192, "F": 8192, "D": 4096, "keep": True},
        # the gradients of a small model's block on a ragged batch
        {"name": "glu_grad ragged", "op": "glu_grad", "type": "f16", "act": "gelu_tanh", "T": 1009, "F": 2752, "D": 1024},
        # the gradients of a training batch
        {"name": "glu_grad batch", "op": "glu_grad", "type": "bf16", "act": "silu", "T": 8192, "F": 8192, "D": 4096},
        # one token's activations on their way into an 8-bit product
        {"name": "quant 1 token", "op": "quant", "type": "bf16", "M": 1, "K": 4096},
        # a prompt's activations; rows that are not a multiple of anything
        {"name": "quant prompt", "op": "quant", "type": "bf16", "M": 8191, "K": 8200},
        # one token against a square projection
        {"name": "gemm_i8 1 token", "op": "gemm_i8", "type": "bf16", "M": 1, "N": 4096, "K": 4096, "bias": False},
        # some dozens of streams, one token each, through the projection back to the model's width
        {"name": "gemm_i8 48 tokens", "op": "gemm_i8", "type": "f32", "M": 48, "N": 4096, "K": 16384, "bias": True},
        # a prompt, ragged in both directions
        {"name": "gemm_i8 prompt", "op": "gemm_i8", "type": "bf16", "M": 4099, "N": 8190, "K": 8192, "bias": True},
        # a few streams through the gated half of an 8-bit block
        {"name": "glu_i8 7 tokens", "op": "glu_i8", "type": "f16", "act": "gelu_tanh", "M": 7, "F": 8192, "K": 4096},
        # a prompt through it
        {"name": "glu_i8 prompt", "op": "glu_i8", "type": "bf16", "act": "silu", "M": 6000, "F": 16384, "K": 4096},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["glu", "glu_grad", "quant", "gemm_i8", "glu_i8"])
    act = rng.choice(["silu", "gelu", "gelu_tanh", "relu"])
    while True:
        if op == "quant":
            c = {"op": op, "type": rng.choice(["bf16", "f16", "f32"]), "M": _spread(rng, 1, 8192), "K": _spread(rng, 16, 16384)}
        elif op == "gemm_i8":
            c = {"op": op, "type": rng.choice(["bf16", "f16", "f32"]), "M": _spread(rng, 1, 8192), "N": _spread(rng, 16, 16384),
                 "K": 128 * _spread(rng, 1, 128), "bias": rng.random() < 0.5}
        elif op == "glu_i8":
            c = {"op": op, "type": rng.choice(["bf16", "f16", "f32"]), "act": act, "M": _spread(rng, 1, 8192), "F": _spread(rng, 16, 16384),
                 "K": 128 * _spread(rng, 1, 64)}
        else:
            c = {"op": op, "type": rng.choice(["bf16", "f16"]), "act": act, "T": _spread(rng, 1, 8192), "F": _spread(rng, 16, 16384),
                 "D": 64 * _spread(rng, 1, 128)}
            if op == "glu":
                c["keep"] = rng.random() < 0.5
        w = work(c)
        if w["flops"] <= 1.6e12 and w["bytes"] <= 1e9:
            return c


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _normal(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * scale


def _activations(g, rows, cols):
    """Activations as they come out of a norm: about unit size, a few channels several times larger."""
    x = _normal(g, rows, cols)
    loud = torch.rand(cols, generator=g, device="cuda") < 0.01
    return x * torch.where(loud, 6.0, 1.0)


def _i8_rows(g, rows, cols):
    """Rows quantised with a scale each, as a program keeps its 8-bit weights: int8 values that reach 127 in about every row."""
    w = _normal(g, rows, cols)
    s = w.abs().amax(1, keepdim=True) / 127
    return (w / s).round().clamp(-127, 127).to(torch.int8), (s[:, 0] / math.sqrt(cols)).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) & 0x7FFFFFFFFFFF)
    s, t = {"case": case}, TYPES[case["type"]]
    if case["op"] in ("glu", "glu_grad"):
        T, F, D = case["T"], case["F"], case["D"]
        s["x"] = _activations(g, T, D).to(t)
        s["wg"] = _normal(g, F, D, scale=1 / math.sqrt(D)).to(t)
        s["wu"] = _normal(g, F, D, scale=1 / math.sqrt(D)).to(t)
        if case["op"] == "glu_grad":
            s["dh"] = _normal(g, T, F).to(t)
            s["g"] = (s["x"].float() @ s["wg"].float().t()).to(t)
            s["u"] = (s["x"].float() @ s["wu"].float().t()).to(t)
    elif case["op"] == "quant":
        s["x"] = _activations(g, case["M"], case["K"]).to(t)
    else:
        M, K = case["M"], case["K"]
        s["a"], s["sa"] = _i8_rows(g, M, K)
        s["sa"] = s["sa"] * math.sqrt(K)
        if case["op"] == "gemm_i8":
            s["b"], s["sb"] = _i8_rows(g, case["N"], K)
            s["bias"] = _normal(g, case["N"]) if case["bias"] else None
        else:
            s["bg"], s["sg"] = _i8_rows(g, case["F"], K)
            s["bu"], s["su"] = _i8_rows(g, case["F"], K)
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------------

def _act(name, x):
    if name == "silu":
        return x / (1 + torch.exp(-x))
    if name == "gelu":
        return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))
    return torch.where(x > 0, x, torch.zeros_like(x))


def _act_grad(name, x):
    if name == "silu":
        p = 1 / (1 + torch.exp(-x))
        return p * (1 + x * (1 - p))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(x * math.sqrt(0.5))) + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (x + 0.044715 * x * x * x))
        return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * c * (1 + 3 * 0.044715 * x * x)
    return torch.where(x > 0, torch.ones_like(x), torch.zeros_like(x))


def _plain(s):
    case = s["case"]
    op, t = case["op"], TYPES[case["type"]]
    if op == "glu":
        x = s["x"].float()
        g, u = x @ s["wg"].float().t(), x @ s["wu"].float().t()
        h = (_act(case["act"], g) * u).to(t)
        return {"h": h, "g": g.to(t), "u": u.to(t)} if case["keep"] else {"h": h}
    if op == "glu_grad":
        g, u, dh = s["g"].float(), s["u"].float(), s["dh"].float()
        dg, du = dh * u * _act_grad(case["act"], g), dh * _act(case["act"], g)
        x = s["x"].float()
        dx = dg @ s["wg"].float() + du @ s["wu"].float()
        return {"dx": dx.to(t), "dwg": (dg.t() @ x).to(t), "dwu": (du.t() @ x).to(t)}
    if op == "quant":
        # in 64 bits: a value next to the border between two whole numbers has to fall on the right side
        x = s["x"].double()
        top = x.abs().amax(1, keepdim=True)
        q = torch.where(top > 0, x * 127 / top, torch.zeros_like(x)).round().to(torch.int8)
        return {"q": q, "scale": (top[:, 0] / 127).float()}
    a = s["a"].float()
    if op == "gemm_i8":
        c = (a @ s["b"].float().t()) * s["sa"][:, None] * s["sb"][None, :]
        return {"c": (c if s["bias"] is None else c + s["bias"][None, :]).to(t)}
    g = (a @ s["bg"].float().t()) * s["sa"][:, None] * s["sg"][None, :]
    u = (a @ s["bu"].float().t()) * s["sa"][:, None] * s["su"][None, :]
    return {"h": (_act(case["act"], g) * u).to(t)}


# ---- this package's calls ---------------------------------------------------------------------------------------------

def _device():
    """The handle of a program that computes with torch too: one for each of its streams, kept."""
    from clpeak_amd import capi
    stream = torch.cuda.current_stream().cuda_stream
    key = (torch.cuda.current_device(), stream)
    if key not in _devices:
        _devices[key] = capi.Device(key[0], stream=stream)
    return capi, _devices[key]


def _own(s):
    capi, dev = _device()
    case = s["case"]
    op, t = case["op"], TYPES[case["type"]]
    kind = {"bf16": capi.TYPE_BF16, "f16": capi.TYPE_F16, "f32": capi.TYPE_F32}[case["type"]]
    new = lambda *shape, dtype=t: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
    if "act" in case:
        act = {"silu": capi.GLU_SILU, "gelu": capi.GLU_GELU, "gelu_tanh": capi.GLU_GELU_TANH, "relu": capi.GLU_RELU}[case["act"]]
    if op in ("glu", "glu_grad"):
        T, F, D = case["T"], case["F"], case["D"]
        x, wg, wu = s["x"], s["wg"], s["wu"]
    if op == "glu":
        h = new(T, F)
        g, u = (new(T, F), new(T, F)) if case["keep"] else (None, None)
        dev.glu_forward(kind, act, x, D, wg, wu, D, h, F, g, u, F, T, F, D)
        return {"h": h, "g": g, "u": u} if case["keep"] else {"h": h}
    if op == "glu_grad":
        dx, dwg, dwu = new(T, D), new(F, D), new(F, D)
        n = dev.glu_backward_workspace(T, F, D)
        dev.glu_backward(kind, act, s["dh"], F, x, D, wg, wu, D, s["g"], s["u"], F, dx, D, dwg, dwu, D, T, F, D,
                         new(n, dtype=torch.uint8), n)
        return {"dx": dx, "dwg": dwg, "dwu": dwu}
    if op == "quant":
        M, K = case["M"], case["K"]
        q, scale = new(M, K, dtype=torch.int8), new(M, dtype=torch.float32)
        dev.quantize_i8(kind, s["x"], K, q, K, scale, M, K, K)
        return {"q": q, "scale": scale}
    M, K = case["M"], case["K"]
    if op == "gemm_i8":
        N = case["N"]
        c, n = new(M, N), dev.gemm_i8_scaled_workspace(M, N, K)
        dev.gemm_i8_scaled(s["a"], K, s["b"], K, s["sa"], s["sb"], s["bias"], kind, c, N, M, N, K,
                           new(n, dtype=torch.uint8) if n else None, n)
        return {"c": c}
    h = new(M, case["F"])
    dev.glu_i8(act, s["a"], K, s["bg"], s["bu"], K, s["sa"], s["sg"], s["su"], kind, h, case["F"], M, case["F"], K)
    return {"h": h}


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    e = {"bf16": 2, "f16": 2, "f32": 4}[case["type"]]
    op = case["op"]
    if op == "quant":
        M, K = case["M"], case["K"]
        return {"bytes": M * K * (e + 1) + 4 * M, "flops": 3 * M * K}
    if op == "gemm_i8":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": (M + N) * K + 4 * (M + N * (2 if case["bias"] else 1)) + e * M * N, "flops": 2 * M * N * K}
    if op == "glu_i8":
        M, F, K = case["M"], case["F"], case["K"]
        return {"bytes": (M + 2 * F) * K + 4 * (M + 2 * F) + e * M * F, "flops": 4 * M * F * K}
    T, F, D = case["T"], case["F"], case["D"]
    if op == "glu":
        return {"bytes": e * (T * D + 2 * F * D + T * F * (3 if case["keep"] else 1)), "flops": 4 * T * F * D}
    return {"bytes": e * (2 * T * D + 4 * F * D + 3 * T * F), "flops": 8 * T * F * D}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------

def _sigmoid64(x):
    e = torch.exp(-x.abs())
    return torch.where(x >= 0, 1 / (1 + e), e / (1 + e))


def _phi64(x):
    """The normal distribution's function and its density."""
    return 0.5 * torch.erfc(-x / math.sqrt(2.0)), torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)


def _gate64(name, x):
    """An activation and its derivative.  The tanh form of gelu is x sigmoid(2 y), y = sqrt(2/pi) (x + 0.044715 x^3)."""
    if name == "silu":
        p = _sigmoid64(x)
        return x * p, p + x * p * _sigmoid64(-x)
    if name == "gelu":
        cdf, pdf = _phi64(x)
        return x * cdf, cdf + x * pdf
    if name == "gelu_tanh":
        k = math.sqrt(8 / math.pi)
        p = _sigmoid64(k * (x + 0.044715 * x ** 3))
        return x * p, p + x * p * (1 - p) * k * (1 + 0.134145 * x ** 2)
    return x.clamp(min=0), (x > 0).double()


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    v = {k: x.double() for k, x in s.items() if torch.is_tensor(x)}
    if op == "glu":
        g, u = torch.mm(v["x"], v["wg"].T), torch.mm(v["x"], v["wu"].T)
        h = _gate64(case["act"], g)[0] * u
        return {"h": h, "g": g, "u": u} if case["keep"] else {"h": h}
    if op == "glu_grad":
        a, da = _gate64(case["act"], v["g"])
        dg, du = v["dh"] * v["u"] * da, v["dh"] * a
        return {"dx": torch.mm(torch.cat((dg, du), 1), torch.cat((v["wg"], v["wu"]), 0)), "dwg": torch.mm(dg.T, v["x"]), "dwu": torch.mm(du.T, v["x"])}
    if op == "quant":
        # whole numbers are the nearest to 127 x / amax: found here from below, a tie going to the even one
        top = v["x"].abs().max(1).values
        at = v["x"] * 127 / top.where(top > 0, torch.ones_like(top))[:, None]
        low = torch.floor(at)
        odd = torch.remainder(low, 2) == 1
        return {"q": (low + ((at - low > 0.5) | ((at - low == 0.5) & odd))).to(torch.int8), "scale": top / 127}
    if op == "gemm_i8":
        c = torch.mm(v["a"] * v["sa"][:, None], (v["b"] * v["sb"][:, None]).T)
        return {"c": c + v["bias"] if "bias" in v else c}
    a = v["a"] * v["sa"][:, None]
    return {"h": _gate64(case["act"], torch.mm(a, (v["bg"] * v["sg"][:, None]).T))[0] * torch.mm(a, (v["bu"] * v["su"][:, None]).T)}
