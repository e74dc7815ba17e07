"""Layer norm, dropout and the gated block on the GPU, beside tests/test_gpu_sublayer.py: memory that a step gives back, sums that
rounding could carry away, operands that are not finite, and the precision of small calls."""
import gc

import numpy as np
import pytest

import sublayer as S
from neureka_b200 import _lib as L
from neureka_b200 import functions as F
from test_gpu_sublayer import put, sub_layer_calls

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("through", [False, True], ids=["forward", "backward"])
@pytest.mark.parametrize("what", ["layer_norm", "gated", "dropout", "sub_layer"])
def test_a_step_gives_its_memory_back_with_the_last_reference(device, what, through):
    rng = np.random.default_rng(51)
    leaves = {k: put(device, rng.standard_normal(s).astype(np.float32)).set_rqs_gradient(True)
              for k, s in (("x", (20, 24)), ("gain", (24,)), ("shift", (24,)), ("wg", (24, 40)), ("wu", (24, 40)), ("wd", (40, 24)))}

    def step():
        x = leaves["x"]
        if what == "layer_norm":
            return x.layer_norm(leaves["gain"], leaves["shift"])
        if what == "gated":
            return x.gated(leaves["wg"], leaves["wu"])
        if what == "dropout":
            return x.dropout(0.5, 1, 2, x)
        return (x.layer_norm(leaves["gain"], leaves["shift"]).gated(leaves["wg"], leaves["wu"]) @ leaves["wd"]).dropout(0.5, 1, 2, x)

    gc.collect()
    gc.disable()
    try:
        before = device.number_of_data_objects(), device.number_of_stored()
        for _ in range(3):
            y = step()
            assert device.number_of_data_objects() > before[0]
            if through:
                y.backward()
                for t in leaves.values():
                    t.gradient = None
            del y
            assert (device.number_of_data_objects(), device.number_of_stored()) == before
    finally:
        gc.enable()


# ---- rounding that could carry something away ----------------------------------------------------------------------------------------
# forms of the kernel: groups of lanes, a CTA, a cluster, rows fetched ahead (by one CTA, by a cluster), chunks
CONSTANT = [(8, 1000), (5000, 96), (2500, 1000), (6000, 300), (1300, 2047), (700, 4096), (310, 12001), (80, 40004), (2, 20000), (3, 300007)]


@pytest.mark.parametrize("shape", CONSTANT, ids=str)
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_layer_norm_of_a_constant_row_is_the_shift(device, dtype, shape):
    """However many rows there are, and however small eps: the mean of equal values is that value."""
    levels = np.array([3.0, 100.0, 1000.0, 0.1, 1000.1, -1e-3, 12345.678, 0.0], dtype=dtype)
    x = np.repeat(levels[np.arange(shape[0]) % len(levels)][:, None], shape[1], 1)
    gain, shift = np.linspace(0.5, 2, shape[1]).astype(dtype), np.linspace(-1, 1, shape[1]).astype(dtype)
    for eps in (1e-5, 1e-12):
        y = put(device, x).layer_norm(put(device, gain), put(device, shift), eps).numpy()
        assert np.array_equal(y, np.repeat(shift[None], shape[0], 0)), np.abs(y - shift).max(1)[:8]


@pytest.mark.parametrize("shape", [(6000, 300), (2500, 777), (5000, 64), (6000, 256), (700, 4096), (310, 12001), (160, 16384), (4, 1024), (2, 140001), (3, 262144)], ids=str)
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_layer_norm_column_sums_take_every_row_once(device, dtype, shape):
    """An error of small integers: dshift is the integer sum itself. With rows of pairs of 1 and -1 (mean 0, variance 1) and eps 0, the normalised
    values are 1 and -1 and dgain is an integer sum too."""
    rng = np.random.default_rng(52)
    rows, n = shape
    x = np.ones(shape, dtype)
    x[:, 1::2] = -1
    x *= np.repeat(rng.choice([-1, 1], (rows, (n + 1) // 2)), 2, 1)[:, :n].astype(dtype)   # (pairs, so that parts of a row have mean 0 too)
    e = rng.integers(-8, 9, shape).astype(dtype)
    tx, gain, shift = put(device, x), put(device, np.ones(n, dtype)).set_rqs_gradient(True), put(device, np.zeros(n, dtype)).set_rqs_gradient(True)
    tx.layer_norm(gain, shift, 0.0).backward(put(device, e))
    assert np.array_equal(shift.gradient.numpy(), e.sum(0))
    if n & (n - 1) == 0:   # (the variance is exactly 1)
        assert np.array_equal(gain.gradient.numpy(), (e * x).sum(0))


LONG = [(1 << 21, 4, 4), (200000, 48, 48), (70000, 20, 100), (9, 400000, 12), (12, 14, 300000)]


@pytest.mark.parametrize("size", LONG, ids=str)
def test_gated_of_narrow_blocks_with_long_sums_of_one_sign(device, size):
    """A block with a narrow side and very many tokens (or the other way round): nothing cancels, so what a running sum loses shows. Each product within the
    framework's bound for a product, 1e-5 of sum |a||b|; what the gate's small products before it were off by comes on top."""
    t, d, h = size
    rng = np.random.default_rng(53)
    x, wg, wu, e = (rng.uniform(0.5, 1.5, s).astype(np.float32) for s in ((t, d), (d, h), (d, h), (t, h)))
    tx, tg, tu = (put(device, a).set_rqs_gradient(True) for a in (x, wg, wu))
    y = tx.gated(tg, tu, "idy")
    y.backward(put(device, e))
    X, G, U, E = (a.astype(np.float64) for a in (x, wg, wu, e))
    g, u = X @ G, X @ U
    tol = 1e-5
    assert (np.abs(y.numpy() / (g * u) - 1) < 2 * tol + 1e-6).all()
    dg, du = E * u, E * g
    for name, got, want in (("dx", tx, dg @ G.T + du @ U.T), ("dwg", tg, X.T @ dg), ("dwu", tu, X.T @ du)):
        # dg and du follow from one product each: off by `tol` where that one is long, by d roundings where it is short
        first = tol if d > 1000 else d * S.unit(np.float32)
        off = np.abs(got.gradient.numpy() / want - 1).max()
        assert off < tol + first + 4 * S.unit(np.float32), (name, off)
    again = put(device, x).gated(put(device, wg), put(device, wu), "idy")
    assert np.array_equal(again.numpy(), y.numpy())


def test_gated_sums_of_4096_terms_take_the_short_accumulation_chunks(device):
    """The tensor core truncates when it accumulates. n = 3 c / 8 accumulations in a chunk of c terms of one sign lose half a unit in the last place of a growing
    partial sum each: the sum over i of 0.5 * 0.72 * 2^-23 * i / n (0.72: a unit in the last place over 2^-23 of the value, on average), 5e-7 for 64
    terms and 10e-7 for 128. The mean over many sums shows which it was."""
    rng = np.random.default_rng(54)
    x, w, one = rng.uniform(0.5, 1.5, (256, 4096)).astype(np.float32), rng.uniform(0.5, 1.5, (4096, 256)).astype(np.float32), np.zeros((4096, 256), np.float32)
    one[0] = 1
    x[:, 0] = 1
    y = put(device, x).gated(put(device, one), put(device, w), "idy").numpy()   # 1 * (x @ w)
    want = x.astype(np.float64) @ w.astype(np.float64)
    assert abs((y / want - 1).mean()) < 7e-7


@pytest.mark.parametrize("fun", L.GATES)
def test_gates_of_plain_products_are_right_to_the_last_bit(device, fun):
    """Where the products are F32 multiply-adds, sig, silu, gelu, relu and idy are the very values of the framework's functions, and tanh and all derivatives
    the true ones rounded once from F64 (half a unit in the last place; what F64 was off by, and denormals, on top). x = [v, 1] with weights [1, 0] and
    [0, 1] gives g = v, u = 1, y = f(v) and, for an error of ones, dx = [f'(v), f(v)]; tokens of [1, 1] with rows of v and ones the same for many columns."""
    v = np.concatenate([np.linspace(-20, 20, 4001), np.linspace(-120, 120, 999), np.geomspace(1e-30, 3e38, 400), -np.geomspace(1e-30, 3e38, 400)]).astype(np.float32)
    w, k = v.astype(S.WIDE), S.WIDE({"gelu": 1.702, "tanh": 2}.get(fun, 1))
    e = np.exp(-k * np.abs(w))
    s, rest = np.where(w < 0, e, 1) / (1 + e), np.where(w < 0, 1, e) / (1 + e)
    if fun == "tanh":
        f = np.tanh(w)
    else:
        f = F.run_function(fun, put(device, v)).numpy()
    df = {"idy": lambda: np.ones_like(w), "relu": lambda: np.where(w >= 0, np.float32(1), np.float32(0.01)), "tanh": lambda: 4 * s * rest, "sig": lambda: s * rest}.get(
        fun, lambda: s + k * w * s * rest)()

    def same(got, want, what):
        if want.dtype == np.float32:
            assert np.array_equal(got, want), what
        else:   # 2^-46: some hundred units in the last place of F64, relative to the terms, which a derivative's sum may cancel
            bound = S.unit(np.float32) * np.abs(want) + 2.0 ** -46 * (np.abs(want) + s + np.abs(k * w) * s * rest) + 2.0 ** -149
            S.assert_within(got, (want, bound), what)

    column = [put(device, np.array(c, np.float32)) for c in ([[1], [0]], [[0], [1]])]
    tx = put(device, np.stack([v, np.ones_like(v)], 1)).set_rqs_gradient(True)
    y = tx.gated(*column, fun)
    y.backward()
    same(y.numpy()[:, 0], f, "f")
    same(tx.gradient.numpy()[:, 1], f, "f again")
    same(tx.gradient.numpy()[:, 0], df, "f'")
    zero, one = np.zeros_like(v), np.ones_like(v)
    for t in (1, 3, 8):
        x = np.ones((t, 2), np.float32)
        rows = [put(device, np.stack(r)).set_rqs_gradient(True) for r in ((v, zero), (zero, one))]
        y = put(device, x).gated(*rows, fun)
        y.backward()
        for i in range(t):
            same(y.numpy()[i], f, f"f of token {i}")
        if t == 1:   # dWg = x^T (u f'(g)), dWu = x^T f(g)
            for i in range(2):
                same(rows[0].gradient.numpy()[i], df, "dWg")
                same(rows[1].gradient.numpy()[i], f, "dWu")


@pytest.mark.parametrize("one_sign", [False, True], ids=["normal", "one_sign"])
@pytest.mark.parametrize("size", [(2, 1024, 1024), (24, 515, 900), (60, 512, 512), (150, 256, 300), (200, 64, 128), (200, 256, 300), (1023, 64, 64)], ids=str)
def test_gated_small_products_are_as_close_as_multiply_adds(device, size, one_sign):
    """Below 2^24 multiply-adds `@` uses those, which are 1e-7 sqrt(K / 64) off (2-norm). With weights [1, 0, 0, ...] for the gate, x of ones in its
    first column and the gate `idy`, y = x @ wu, dwu = x^T @ e and dx = e @ wu^T (but for its first column). 3xTF32 itself: the low parts are rounded to 2^-23 of a
    value and 2^-22 is dropped, 1e-7; accumulations in chunks of 64 terms at most lose 2e-7 of a sum of one sign, as derived above: 3e-7."""
    t, d, h = size
    rng = np.random.default_rng(57)
    draw = (lambda *s: rng.uniform(0.5, 1.5, s).astype(np.float32)) if one_sign else (lambda *s: rng.standard_normal(s).astype(np.float32))
    x, wg, wu, e = draw(t, d), np.zeros((d, h), np.float32), draw(d, h), draw(t, h)
    x[:, 0], wg[0] = 1, 1
    tx, tg, tu = (put(device, a).set_rqs_gradient(True) for a in (x, wg, wu))
    y = tx.gated(tg, tu, "idy")
    y.backward(put(device, e))
    X, U, E = (a.astype(np.float64) for a in (x, wu, e))
    for name, got, want in (("y", y.numpy(), X @ U), ("dwu", tu.gradient.numpy(), X.T @ E), ("dx", tx.gradient.numpy()[:, 1:], (E @ U.T)[:, 1:])):
        assert np.linalg.norm(got - want) < 3e-7 * np.linalg.norm(want), (name, np.linalg.norm(got - want) / np.linalg.norm(want))


# ---- operands that are not finite ----------------------------------------------------------------------------------------------------
def product(a, b):
    """a @ b in F64, from products of finite matrices alone: which terms of a sum are infinite, of which sign, or no number, counted"""
    def count(p, q):
        return p.astype(np.float64) @ q.astype(np.float64) > 0
    (ai, ap, an, a0), (bi, bp, bn, b0) = ((np.isinf(m), m > 0, m < 0, m == 0) for m in (a, b))
    plus = count(ai & ap, bp) | count(ai & an, bn) | count(ap, bi & bp) | count(an, bi & bn)
    minus = count(ai & ap, bn) | count(ai & an, bp) | count(ap, bi & bn) | count(an, bi & bp)
    none = np.isnan(a).any(1)[:, None] | np.isnan(b).any(0)[None] | count(ai, b0) | count(a0, bi)
    c = np.where(np.isfinite(a), a, 0).astype(np.float64) @ np.where(np.isfinite(b), b, 0).astype(np.float64)
    return np.where(none | (plus & minus), np.nan, np.where(plus, np.inf, np.where(minus, -np.inf, c)))


def same_kind(got, want, what):
    """NaN where the plain form has NaN, the same infinity where it has one, finite elsewhere"""
    def kind(a):
        return np.where(np.isnan(a), 9, np.where(np.isinf(a), np.sign(np.where(np.isnan(a), 0, a)), 0)).astype(int)
    a, b = kind(got), kind(want)
    assert np.array_equal(a, b), f"{what}: {int((a != b).sum())} of {a.size} of another kind"


# one token; some; a lone CTA's tiles, their k split, pairs; narrow sides
INFINITE = [(1, 96, 128), (2, 96, 128), (8, 100, 72), (24, 300, 257), (24, 4100, 136), (64, 130, 260), (150, 96, 200), (300, 260, 130), (300, 2100, 130), (2600, 300, 1100), (300, 30, 500)]


@pytest.mark.parametrize("turned", [False, True], ids=["", "turned"])
@pytest.mark.parametrize("size", INFINITE, ids=str)
def test_gated_of_infinite_operands(device, size, turned):
    """An infinity times a finite value is an infinity, whatever the other value's low bits are and however many tokens there are."""
    t, d, h = size
    rng = np.random.default_rng(55)

    def draw(*shape):   # values whose low bits are zero, positive or negative, in turn, and a few zeros
        a = rng.standard_normal(shape).astype(np.float32)
        a = np.where(rng.random(shape) < 0.3, np.round(a * 4) / 4, a)
        return np.where(rng.random(shape) < 0.01, 0, a).astype(np.float32)

    x, wg, wu, e = draw(t, d), draw(d, h), draw(d, h), draw(t, h)
    for place in ("x", "w", "both", "e"):
        X, G, U, E = x.copy(), wg.copy(), wu.copy(), e.copy()
        if place in ("x", "both"):
            X[t // 2, d // 3] = np.inf
            X[t - 1, d - 1] = -np.inf
        if place in ("w", "both"):
            G[d // 2, h // 3] = -np.inf
            U[d - 1, h - 1] = np.inf
        if place == "e":
            E[t // 2, h // 2] = np.inf
            E[t - 1, 0] = -np.inf
        tx, tg, tu = (put(device, a, "turned" if turned and k else "dense").set_rqs_gradient(True) for k, a in enumerate((X, G, U)))
        y = tx.gated(tg, tu, "idy")
        y.backward(put(device, E))
        with np.errstate(invalid="ignore"):
            g, u = product(X, G), product(X, U)
            dg, du = E * u, E * g
            same_kind(y.numpy(), g * u, f"y {place}")
            same_kind(tx.gradient.numpy(), product(dg, G.T) + product(du, U.T), f"dx {place}")
            same_kind(tg.gradient.numpy(), product(X.T, dg), f"dwg {place}")
            same_kind(tu.gradient.numpy(), product(X.T, du), f"dwu {place}")


@pytest.mark.parametrize("size", [(256, 256, 300), (300, 4100, 70), (1100, 300, 1030)], ids=str)
def test_matrix_product_of_infinite_operands(device, size):
    """... and so for `@`, whose large products are computed the same way"""
    m, k, n = size
    rng = np.random.default_rng(56)
    a, b = (np.where(rng.random(s) < 0.3, 0.5, rng.standard_normal(s)).astype(np.float32) for s in ((m, k), (k, n)))
    a[m // 2, k // 3], a[m - 1, k - 1], b[k // 2, n // 3], a[3, 5] = np.inf, -np.inf, np.inf, np.nan
    b[k // 3, 7] = 0
    got = (put(device, a) @ put(device, b)).numpy()
    with np.errstate(invalid="ignore"):
        same_kind(got, product(a, b), "a @ b")


def test_split_sums_and_sums_taken_again_captured_and_replayed(device):
    """What takes memory for the length of a call, or looks at its sums again, does so under capture as well: a narrow block of many tokens, and infinities."""
    import torch
    for case, place in (((np.float32, 20000, 40, 48), None), ((np.float32, 300, 260, 515), (7, 9)), ((np.float32, 24, 300, 257), (3, 5))):
        (x, wg), results, run, raw = sub_layer_calls(device.ctx, *case)
        stream = torch.cuda.ExternalStream(L.lib.nk_stream(device.ctx))
        run()
        device.sync()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
            run()
        for _ in range(2):
            wg.mul_(-1.25)
            if place is not None:
                wg[place] = float("inf")
            torch.cuda.synchronize()
            run()
            device.sync()
            want = [r.clone() for r in results]
            for r in results:
                r.fill_(-7)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(torch.nan_to_num(a, nan=-3.5), torch.nan_to_num(b, nan=-3.5)) and torch.equal(a.isnan(), b.isnan()) for a, b in zip(results, want))
            assert bool(torch.isinf(results[1]).any()) == (place is not None)


def test_two_contexts_split_long_sums_at_once(device):
    import ctypes as C
    import torch
    second = C.c_void_p()
    L.check(L.lib.nk_device_open(device.ordinal, C.byref(second)))
    try:
        sides = []
        for ctx in (device.ctx, second):
            _, results, run, raw = sub_layer_calls(ctx, np.float32, 30000, 24, 40)
            run()
            L.check(L.lib.nk_sync(ctx), ctx)
            sides.append((results, [r.clone() for r in results], run, raw))
        for _ in range(10):
            for _, _, run, _ in sides:
                run()
        torch.cuda.synchronize()
        for results, want, _, _ in sides:
            assert all(torch.equal(a, b) for a, b in zip(results, want))
        del sides, results, want, run, raw
    finally:
        L.lib.nk_device_close(second)
