"""What the operators of a feed-forward training sub-layer -- layer norm, dropout, the gated block -- are measured on: their plain forms in
elementary torch operations, and the calls a user makes of the framework's own.

A case is a dict of plain values. Inputs are made on the GPU from a seed. Forward cases call the C ABI on buffers that the program keeps,
as the JVM host does; training cases go through the Tensor layer and its backward pass.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_TORCH = {"float32": torch.float32, "float64": torch.float64}
_BYTES = {"float32": 4, "float64": 8}
_EPS = 1e-5


def listed():
    return [
        # one token's activations before a layer
        {"name": "norm_token", "op": "norm", "train": False, "dtype": "float32", "rows": 1, "n": 4096, "affine": True},
        # a training batch of long sequences
        {"name": "norm_train_large", "op": "norm", "train": True, "dtype": "float32", "rows": 16384, "n": 4096, "affine": True},
        # a batch of odd extents: no row after the first starts on a vector's boundary
        {"name": "norm_train_ragged", "op": "norm", "train": True, "dtype": "float32", "rows": 4093, "n": 777, "affine": True},
        # few, very long rows in double precision
        {"name": "norm_train_long_f64", "op": "norm", "train": True, "dtype": "float64", "rows": 37, "n": 50001, "affine": True},
        # a small layer's output: the cost of a call
        {"name": "dropout_small", "op": "dropout", "train": False, "dtype": "float32", "rows": 64, "n": 1000, "p": 0.1, "residual": False},
        # the end of a sub-layer: dropped and added to the residual stream, and its backward pass
        {"name": "dropout_train_large", "op": "dropout", "train": True, "dtype": "float32", "rows": 8192, "n": 8192, "p": 0.1, "residual": True},
        # odd extents in double precision
        {"name": "dropout_train_f64", "op": "dropout", "train": True, "dtype": "float64", "rows": 1023, "n": 1537, "p": 0.5, "residual": False},
        # one token through a large block: its weights read once
        {"name": "gated_token", "op": "gated", "train": False, "dtype": "float32", "tokens": 1, "model": 4096, "hidden": 8192, "fun": "silu", "turned": False},
        # a few sequences' next tokens, weights stored the other way round
        {"name": "gated_few_tokens", "op": "gated", "train": False, "dtype": "float32", "tokens": 24, "model": 2048, "hidden": 5461, "fun": "silu", "turned": True},
        # a training step on a large batch
        {"name": "gated_train_large", "op": "gated", "train": True, "dtype": "float32", "tokens": 4096, "model": 2048, "hidden": 8192, "fun": "silu", "turned": False},
        # a training step at odd extents
        {"name": "gated_train_ragged", "op": "gated", "train": True, "dtype": "float32", "tokens": 1023, "model": 777, "hidden": 2051, "fun": "gelu", "turned": False},
        # a small training step in double precision
        {"name": "gated_train_f64", "op": "gated", "train": True, "dtype": "float64", "tokens": 300, "model": 512, "hidden": 1365, "fun": "sig", "turned": True},
    ]


def _log(rng, lo, hi):
    """an integer spread over the logarithm of its range, odd values as likely as even ones"""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "dropout", "gated", "gated"])
    dtype = rng.choice(["float32", "float32", "float32", "float64"])
    case = {"op": op, "train": rng.choice([True, True, False]), "dtype": dtype}
    if op == "gated":
        most = 4096 * 2048 * 8192 // (32 if dtype == "float64" else 1)
        while True:
            t, d, h = _log(rng, 1, 4096), _log(rng, 64, 4096), _log(rng, 64, 16384)
            if t * d * h <= most and d * h <= 4096 * 8192:
                break
        case.update(tokens=t, model=d, hidden=h, fun=rng.choice(["silu", "gelu", "sig", "relu", "tanh", "idy"]), turned=rng.choice([True, False]))
        return case
    while True:
        rows, n = _log(rng, 1, 65536), _log(rng, 8, 65536)   # (below some features the gradient of a norm is what cancellation leaves)
        if 64 <= rows * n <= (1 << 26) // (2 if dtype == "float64" else 1):
            break
    case.update(rows=rows, n=n)
    if op == "norm":
        case["affine"] = rng.choice([True, True, False])
    else:
        case.update(p=rng.choice([0.0, 0.1, 0.25, 0.5, 0.9]), residual=rng.choice([True, False]))
    return case


# ---- inputs ------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    td = _TORCH[case["dtype"]]

    def normal(std, *shape):
        return torch.empty(shape, dtype=td, device="cuda").normal_(0.0, std, generator=g)

    s = {"case": case}
    if case["op"] == "gated":
        t, d, h = case["tokens"], case["model"], case["hidden"]
        s["x"] = normal(1.0, t, d)
        shape = (h, d) if case["turned"] else (d, h)   # as stored; the block takes [model, hidden] views of either
        s["wg"], s["wu"] = normal(1.0 / math.sqrt(d), *shape), normal(1.0 / math.sqrt(d), *shape)
        out = (t, h)
    else:
        out = (case["rows"], case["n"])
        s["x"] = normal(1.0, *out)
        if case["op"] == "norm":   # activations: each feature with a level and a spread of its own
            s["x"].mul_(1.0 + normal(0.5, 1, case["n"]).abs_()).add_(normal(1.0, 1, case["n"]))
            if case["affine"]:
                s["gain"], s["shift"] = normal(0.1, case["n"]).add_(1.0), normal(0.1, case["n"])
        else:
            s["seed"], s["stream"] = seed, seed % 1000
            if case["residual"]:
                s["r"] = normal(1.0, *out)
    if case["train"]:
        s["e"] = normal(1.0, *out)
    else:
        s["y"] = torch.empty(out, dtype=td, device="cuda")   # the buffer a program keeps for the result
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------
def _norm_plain(s, train):
    x, gain, shift = s["x"], s.get("gain"), s.get("shift")
    c = x - x.mean(1, keepdim=True)
    r = 1.0 / torch.sqrt((c * c).mean(1, keepdim=True) + _EPS)
    xh = c * r
    y = xh if gain is None else xh * gain + shift
    if not train:
        return y
    e = s["e"]
    gy = e if gain is None else e * gain
    dx = r * (gy - gy.mean(1, keepdim=True) - xh * (gy * xh).mean(1, keepdim=True))
    return [y, dx] if gain is None else [y, dx, (e * xh).sum(0), e.sum(0)]


def _words(n, seed, stream):
    """the first n words of Philox4x32-10 with the key `seed` and the counters (0, stream), (1, stream), ..., in 64-bit integers"""
    low = 0xFFFFFFFF
    block = torch.arange((n + 3) // 4, dtype=torch.int64, device="cuda")
    c0, c1 = block & low, block >> 32
    c2, c3 = torch.full_like(block, stream & low), torch.full_like(block, (stream >> 32) & low)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57   # the low 64 bits; >> keeps the sign, the mask drops it
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack((c0, c1, c2, c3), 1).reshape(-1)[:n]


def _dropout_plain(s, train):
    x, p = s["x"], s["case"]["p"]
    keep = (_words(x.numel(), s["seed"], s["stream"]) >= int(p * 4294967296.0)).reshape(x.shape)
    scale, zero = 1.0 / (1.0 - p), torch.zeros((), dtype=x.dtype, device="cuda")
    y = torch.where(keep, x * scale, zero)
    if "r" in s:
        y = s["r"] + y
    return [y, torch.where(keep, s["e"] * scale, zero)] if train else y


def _function_plain(fun, g):
    """the function and its derivative, as the framework defines them (gelu by the sigmoid, relu with a slope of 0.01 below zero)"""
    if fun == "idy":
        return g, torch.ones_like(g)
    if fun == "relu":
        slope = torch.where(g >= 0, 1.0, 0.01).to(g.dtype)
        return g * slope, slope
    if fun == "tanh":
        t = torch.tanh(g)
        return t, 1.0 - t * t
    k = 1.702 if fun == "gelu" else 1.0
    sig = 1.0 / (1.0 + torch.exp(-k * g))
    if fun == "sig":
        return sig, sig * (1.0 - sig)
    return g * sig, sig + k * g * sig * (1.0 - sig)


def _gated_plain(s, train):
    case, x, wg, wu = s["case"], s["x"], s["wg"], s["wu"]
    if case["turned"]:
        wg, wu = wg.T, wu.T
    g, u = x @ wg, x @ wu
    f, df = _function_plain(case["fun"], g)
    y = f * u
    if not train:
        return y
    e = s["e"]
    dg, du = e * u * df, e * f
    return [y, dg @ wg.T + du @ wu.T, x.T @ dg, x.T @ du]


# ---- the framework's operators -----------------------------------------------------------------------------------
class _Wrapped:
    """the C ABI's handle of a program's own device memory and its view descriptor; freed with the object"""

    def __init__(self, device, values):
        import ctypes as C
        from neureka_b200 import _lib as L
        from neureka_b200.ndconf import NDConfiguration
        self.device, self.values, self.handle = device, values, C.c_void_p()
        L.check(L.lib.nk_wrap(device.ctx, L.NK_F32 if values.dtype == torch.float32 else L.NK_F64, C.c_void_p(values.data_ptr()), values.numel(),
                              C.byref(self.handle)), device.ctx)
        self.conf = NDConfiguration.of_shape(tuple(values.shape))
        self.describe(self.conf)

    def describe(self, conf):
        import ctypes as C
        self._inline = conf.as_inline_array()
        self.cfg = self._inline.ctypes.data_as(C.POINTER(C.c_int32))

    def __del__(self):
        from neureka_b200 import _lib as L
        L.lib.nk_free(self.device.ctx, self.handle)


def _tensor(device, values):
    """a framework tensor holding the given values"""
    from neureka_b200.tensor import Tensor
    t = Tensor.of(np.float32 if values.dtype == torch.float32 else np.float64, tuple(values.shape), 0).to(device).set_is_virtual(False)
    device.sync()
    _as_torch(t).copy_(values)
    torch.cuda.current_stream().synchronize()
    return t


class _Pointer:
    """what a view of a tensor's memory holds on to"""


def _as_torch(tensor):
    """a tensor's memory as torch sees it (no copy); keeps the tensor alive"""
    import ctypes as C
    from neureka_b200 import _lib as L
    ptr = C.c_void_p()
    L.check(L.lib.nk_buf_info(tensor._data.buf, C.byref(ptr), None, None))
    at = _Pointer()
    at.tensor = tensor
    at.__cuda_array_interface__ = {"shape": tensor.shape, "typestr": "<f4" if tensor.dtype == np.float32 else "<f8", "data": (ptr.value, False), "version": 3}
    return torch.as_tensor(at, device="cuda")


def _held(s):
    """What a program of the framework has in hand: buffers for the C ABI, tensors for a training step. Made on a state's first pass and
    kept as such a program keeps them."""
    if "held" not in s:
        from neureka_b200.device import CudaDevice
        device = CudaDevice.get(0)
        make = _tensor if s["case"]["train"] else _Wrapped
        held = {k: make(device, v) for k, v in s.items() if isinstance(v, torch.Tensor)}
        held["device"] = device
        turned = s["case"].get("turned", False)
        for k in ("wg", "wu"):
            if k in held and turned:
                if s["case"]["train"]:
                    held[k + "_stored"], held[k] = held[k], held[k].permute(1, 0)
                else:
                    held[k].describe(held[k].conf.reshaped((1, 0)))
        if s["case"]["train"]:
            for k in ("x", "gain", "shift", "wg", "wu"):
                if k in held:
                    held[k].set_rqs_gradient(True)
        s["held"] = held
    return s["held"]


def _forward_own(s):
    from neureka_b200 import _lib as L
    case, b = s["case"], _held(s)
    ctx, dt = b["device"].ctx, L.NK_F32 if case["dtype"] == "float32" else L.NK_F64
    x, y = b["x"], b["y"]
    if case["op"] == "norm":
        gain, shift = b.get("gain"), b.get("shift")
        L.check(L.lib.nk_layer_norm(ctx, dt, 2, y.handle, y.cfg, x.handle, x.cfg, gain and gain.handle, gain and gain.cfg,
                                    shift and shift.handle, shift and shift.cfg, _EPS, None), ctx)
    elif case["op"] == "dropout":
        r = b.get("r")
        L.check(L.lib.nk_dropout(ctx, dt, 2, y.handle, y.cfg, x.handle, x.cfg, r and r.handle, r and r.cfg, case["p"], s["seed"], s["stream"]), ctx)
    else:
        wg, wu = b["wg"], b["wu"]
        L.check(L.lib.nk_gated(ctx, L.FUN[case["fun"]], dt, y.handle, y.cfg, x.handle, x.cfg, wg.handle, wg.cfg, wu.handle, wu.cfg, None), ctx)
    return s["y"]


def _train_own(s):
    case, t = s["case"], _held(s)
    leaves = [t[k] for k in ("x", "gain", "shift", "wg", "wu") if k in t]
    for leaf in leaves:
        leaf.gradient = None   # a new step
    if case["op"] == "norm":
        y = t["x"].layer_norm(t.get("gain"), t.get("shift"), _EPS)
    elif case["op"] == "dropout":
        y = t["x"].dropout(case["p"], s["seed"], s["stream"], t.get("r"))
    else:
        y = t["x"].gated(t["wg"], t["wu"], case["fun"])
    y.backward(t["e"])
    return [_as_torch(y)] + [_as_torch(leaf.gradient) for leaf in leaves]


def run(s):
    train = s["case"]["train"]
    if own:
        return _train_own(s) if train else _forward_own(s)
    return {"norm": _norm_plain, "dropout": _dropout_plain, "gated": _gated_plain}[s["case"]["op"]](s, train)


# ---- the definition in 64 bits -----------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double().requires_grad_(case["train"])
    leaves = [x]
    if case["op"] == "dropout":
        n = x.numel()
        i = np.arange((n + 3) // 4, dtype=np.uint64)
        mask, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
        c = [i & mask, i >> shift, np.full_like(i, s["stream"]) & mask, np.full_like(i, s["stream"]) >> shift]
        for r in range(10):
            key = [np.uint64(((s["seed"] & 0xFFFFFFFF) + r * 0x9E3779B9) & 0xFFFFFFFF), np.uint64(((s["seed"] >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF)]
            first, second = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
            c = [(second >> shift) ^ c[1] ^ key[0], second & mask, (first >> shift) ^ c[3] ^ key[1], first & mask]
        dropped = np.stack(c, 1).reshape(-1)[:n] < np.uint64(math.floor(case["p"] * 2.0 ** 32))
        factor = torch.from_numpy(np.where(dropped, 0.0, 1.0 / (1.0 - case["p"]))).cuda().reshape(x.shape)
        y = x * factor + (s["r"].double() if "r" in s else 0.0)
    elif case["op"] == "norm":
        deviation = torch.sqrt(((x - x.mean(1, keepdim=True)) ** 2).sum(1, keepdim=True) / case["n"] + _EPS)
        y = (x - x.sum(1, keepdim=True) / case["n"]) / deviation
        if case["affine"]:
            leaves += [s[k].double().requires_grad_(case["train"]) for k in ("gain", "shift")]
            y = y * leaves[1] + leaves[2]
    else:
        weights = [s[k].double() for k in ("wg", "wu")]
        weights = [(w.T if case["turned"] else w).contiguous().requires_grad_(case["train"]) for w in weights]
        leaves += weights
        a = x @ weights[0]
        f = {"idy": lambda: a, "relu": lambda: torch.maximum(a, 0.01 * a), "tanh": lambda: (torch.exp(a) - torch.exp(-a)) / (torch.exp(a) + torch.exp(-a)),
             "sig": lambda: torch.sigmoid(a), "silu": lambda: a * torch.sigmoid(a), "gelu": lambda: a * torch.sigmoid(1.702 * a)}[case["fun"]]()
        y = f * (x @ weights[1])
    if not case["train"]:
        return y.detach()
    gradients = torch.autograd.grad(y, leaves, s["e"].double())
    return [y.detach(), *gradients]


def work(case):
    size = _BYTES[case["dtype"]]
    if case["op"] == "gated":
        t, d, h = case["tokens"], case["model"], case["hidden"]
        if case["train"]:
            return {"bytes": size * (2 * t * d + 4 * d * h + 2 * t * h), "flops": 12.0 * t * d * h}
        return {"bytes": size * (t * d + 2 * d * h + t * h), "flops": 4.0 * t * d * h}
    full = case["rows"] * case["n"]
    if case["op"] == "norm":
        vectors = 4 * case["n"] if case["affine"] else 0
        return {"bytes": size * ((4 * full + vectors) if case["train"] else (2 * full + vectors // 2)), "flops": (20.0 if case["train"] else 8.0) * full}
    passes = (4 if case["train"] else 2) + (1 if case["residual"] else 0)
    return {"bytes": size * passes * full, "flops": (4.0 if case["train"] else 2.0) * full}
