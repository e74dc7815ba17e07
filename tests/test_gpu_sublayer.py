"""Layer norm, dropout and the gated block on the GPU against plain implementations in at least 64 bits (tests/sublayer.py, where the
bounds are derived)."""
import ctypes as C

import numpy as np
import pytest

import sublayer as S
from neureka_b200 import _lib as L
from neureka_b200.ndconf import Layout
from neureka_b200.tensor import Tensor

pytestmark = pytest.mark.gpu
TYPES = [np.float32, np.float64]


def put(device, a, view="dense"):
    """a's values as a tensor on the device, laid out as asked"""
    a = np.ascontiguousarray(a)
    if view == "dense":
        return Tensor.of(a.dtype, a.shape, a.reshape(-1)).to(device)
    if view == "column":
        return Tensor.of(a.dtype, a.shape, a.reshape(-1)).to_layout(Layout.COLUMN_MAJOR).to(device)
    if view == "turned":
        order = tuple(reversed(range(a.ndim)))
        return Tensor.of(a.dtype, a.T.shape, np.ascontiguousarray(a.T).reshape(-1)).to(device).permute(*order)
    step = 2 if view == "stepped" else 1   # a part of a larger tensor whose other elements are NaN
    whole = np.full([1 + s * step + 2 for s in a.shape], np.nan, dtype=a.dtype)
    at = tuple(slice(1, 1 + s * step, step) for s in a.shape)
    whole[at] = a
    return Tensor.of(a.dtype, whole.shape, whole.reshape(-1)).to(device)[at]


VIEWS = ["dense", "part", "stepped", "turned", "column"]


# ---- layer norm ------------------------------------------------------------------------------------------------------------------
def norm_case(device, rng, dtype, shape, affine=True, view="dense", spread=1.0, level=0.0):
    n, u = shape[-1], S.unit(dtype)
    x = (rng.standard_normal(shape) * spread + level).astype(dtype)
    e = rng.standard_normal(shape).astype(dtype)
    gain = (1 + 0.3 * rng.standard_normal(n)).astype(dtype) if affine else None
    shift = rng.standard_normal(n).astype(dtype) if affine else None
    tx, te = put(device, x, view).set_rqs_gradient(True), put(device, e, view)
    tg = put(device, gain).set_rqs_gradient(True) if affine else None
    ts = put(device, shift).set_rqs_gradient(True) if affine else None
    y = tx.layer_norm(tg, ts, 1e-5)
    want, xh, r = S.norm(x, gain, shift, 1e-5)
    S.assert_within(y.numpy(), (want, S.norm_bound(x, gain, want, xh, r, u)), f"y {shape}")
    y.backward(te)
    dx, dgain, dshift = S.norm_gradients(x, gain, e, 1e-5, u)
    S.assert_within(tx.gradient.numpy(), dx, f"dx {shape}")
    if affine:
        S.assert_within(tg.gradient.numpy(), dgain, f"dgain {shape}")
        S.assert_within(ts.gradient.numpy(), dshift, f"dshift {shape}")


NORM_SHAPES = [(1, 1), (5, 1), (3, 2), (1, 3), (7, 8), (33, 16), (129, 31), (5, 64), (1, 100), (65, 128), (17, 129), (300, 255), (9, 256), (4, 1000), (2, 1023), (3, 1024),
               (3, 1025), (600, 1024), (2, 2047), (5, 4096), (301, 2048), (2, 8191), (3, 8192), (2, 8193), (1, 16384), (2, 32768), (1, 50001), (2, 65536), (1, 131072), (1, 300007),
               (5000, 8), (4100, 33), (2, 3, 5, 40), (9,), (777,)]


@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_and_its_gradients(device, dtype, shape):
    norm_case(device, np.random.default_rng(sum(shape)), dtype, shape)


# enough rows that they are fetched ahead: teams of one to sixteen warps and clusters, rows that start anywhere
@pytest.mark.parametrize("shape", [(5000, 257), (6000, 300), (2500, 777), (2400, 1024), (1300, 2047), (1200, 2500), (620, 4096), (700, 4097), (400, 8000), (300, 8192), (310, 12001), (160, 16384),
                                   (90, 30001), (80, 40004)], ids=str)
@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_of_many_rows(device, dtype, shape):
    norm_case(device, np.random.default_rng(sum(shape)), dtype, shape)
    norm_case(device, np.random.default_rng(sum(shape)), dtype, shape, affine=False, view="part")


def test_layer_norm_rows_at_the_ends_of_odd_memory(device):
    """A program's own memory, adopted at an address that is no multiple of 16 and as long as the tensor: nothing outside it is read."""
    import torch
    rows, n = 2500, 777
    rng = np.random.default_rng(9)
    x = rng.standard_normal((rows, n)).astype(np.float32)
    for shift in (1, 2, 3):
        memory = torch.full((rows * n + 8,), float("nan"), dtype=torch.float32, device="cuda")
        memory[shift:shift + rows * n] = torch.from_numpy(x.reshape(-1)).cuda()
        torch.cuda.synchronize()
        buf = C.c_void_p()
        L.check(L.lib.nk_wrap(device.ctx, L.NK_F32, C.c_void_p(memory.data_ptr() + 4 * shift), rows * n, C.byref(buf)), device.ctx)
        try:
            out, stats = put(device, np.zeros((rows, n), np.float32)), put(device, np.zeros((2, rows), np.float32))
            c = out.ndconf.inline_pointer
            L.check(L.lib.nk_layer_norm(device.ctx, L.NK_F32, 2, out._data.buf, c, buf, c, None, None, None, None, 1e-5, stats._data.buf), device.ctx)
            want, xh, r = S.norm(x, None, None, 1e-5)
            S.assert_within(out.numpy(), (want, S.norm_bound(x, None, want, xh, r, S.unit(np.float32))), f"shift {shift}")
            L.check(L.lib.nk_layer_norm_grad(device.ctx, L.NK_F32, 2, out._data.buf, c, None, None, None, None, buf, c, buf, c, None, None, stats._data.buf), device.ctx)
            S.assert_within(out.numpy(), S.norm_gradients(x, None, x, 1e-5, S.unit(np.float32))[0], f"dx, shift {shift}")
        finally:
            L.lib.nk_free(device.ctx, buf)


@pytest.mark.parametrize("view", VIEWS[1:])
@pytest.mark.parametrize("shape", [(5, 7), (40, 96), (3, 4, 130), (3, 2050), (2, 9000)], ids=str)
@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_of_views(device, dtype, shape, view):
    norm_case(device, np.random.default_rng(1), dtype, shape, view=view)


@pytest.mark.parametrize("shape", [(6, 12), (40, 777), (3, 20000)], ids=str)
def test_layer_norm_without_gain_and_shift_and_far_from_zero(device, shape):
    norm_case(device, np.random.default_rng(2), np.float32, shape, affine=False)
    norm_case(device, np.random.default_rng(2), np.float32, shape, level=1000.0)      # the variance is a millionth of the mean's square
    norm_case(device, np.random.default_rng(2), np.float64, shape, spread=1e-8, level=1.0)
    norm_case(device, np.random.default_rng(2), np.float32, shape, spread=1e15)


def test_layer_norm_vectors_of_other_layouts(device):
    rng = np.random.default_rng(5)
    x, e = rng.standard_normal((6, 48)).astype(np.float32), rng.standard_normal((6, 48)).astype(np.float32)
    gain, shift = rng.standard_normal((1, 48)).astype(np.float32), rng.standard_normal((1, 48)).astype(np.float32)
    for view in VIEWS[1:]:
        tx, tg, ts = put(device, x).set_rqs_gradient(True), put(device, gain, view).set_rqs_gradient(True), put(device, shift, view).set_rqs_gradient(True)
        y = tx.layer_norm(tg, ts)
        want, xh, r = S.norm(x, gain[0], shift[0], 1e-5)
        S.assert_within(y.numpy(), (want, S.norm_bound(x, gain[0], want, xh, r, S.unit(np.float32))), view)
        y.backward(put(device, e))
        dx, dgain, dshift = S.norm_gradients(x, gain[0], e, 1e-5, S.unit(np.float32))
        assert tg.gradient.shape == (1, 48)
        S.assert_within(tx.gradient.numpy(), dx, "dx")
        S.assert_within(tg.gradient.numpy(), dgain, "dgain")
        S.assert_within(ts.gradient.numpy(), dshift, "dshift")


def test_layer_norm_rows_that_are_not_finite_stay_apart(device):
    """A NaN or an infinity spoils its own row and no other; constant rows give the shift."""
    x = np.random.default_rng(6).standard_normal((8, 300)).astype(np.float32)
    x[1, 7], x[4, 0], x[6] = np.nan, np.inf, 2.5
    shift = np.linspace(-1, 1, 300).astype(np.float32)
    y = put(device, x).layer_norm(None, put(device, shift)).numpy()
    assert np.isnan(y[1]).all() and np.isnan(y[4]).all()
    assert np.isfinite(y[[0, 2, 3, 5, 6, 7]]).all()
    assert np.array_equal(y[6], shift)


def test_layer_norm_gives_the_same_bits_every_time_and_only_the_gradients_asked_for(device):
    rng = np.random.default_rng(7)
    for shape in ((1500, 1000), (3, 70000), (2000, 1003)):
        x, e, gain = (rng.standard_normal(s).astype(np.float32) for s in (shape, shape, shape[-1:]))
        got = []
        for wanted in ("xg", "xg", "x", "g"):
            tx, tg = put(device, x).set_rqs_gradient("x" in wanted), put(device, gain).set_rqs_gradient("g" in wanted)
            y = tx.layer_norm(tg)
            y.backward(put(device, e))
            got.append((y.numpy(), tx.gradient and tx.gradient.numpy(), tg.gradient and tg.gradient.numpy()))
        assert got[2][2] is None and got[3][1] is None
        for other in (got[1], (got[2][0], got[2][1], got[3][2])):
            assert all(np.array_equal(a, b) for a, b in zip(got[0], other))


def test_layer_norm_in_place(device):
    """the drain may be the source, and the gradient's drain the error"""
    rng = np.random.default_rng(8)
    for n in (96, 5000, 40000):
        x, e = rng.standard_normal((4, n)).astype(np.float32), rng.standard_normal((4, n)).astype(np.float32)
        t, r, stats, err = put(device, x), put(device, x), put(device, np.zeros((2, 4), np.float32)), put(device, e)
        arr = t.ndconf.as_inline_array()
        c = arr.ctypes.data_as(C.POINTER(C.c_int32))
        L.check(L.lib.nk_layer_norm(device.ctx, L.NK_F32, 2, t._data.buf, c, t._data.buf, c, None, None, None, None, 1e-5, stats._data.buf), device.ctx)
        assert np.array_equal(t.numpy(), r.layer_norm().numpy())
        L.check(L.lib.nk_layer_norm_grad(device.ctx, L.NK_F32, 2, err._data.buf, c, None, None, None, None, err._data.buf, c, r._data.buf, c, None, None, stats._data.buf), device.ctx)
        S.assert_within(err.numpy(), S.norm_gradients(x, None, e, 1e-5, S.unit(np.float32))[0], "dx")


# ---- dropout ---------------------------------------------------------------------------------------------------------------------
DROP_SHAPES = [(1,), (3,), (4,), (5,), (64, 1000), (33, 7), (2, 3, 4, 5), (1023, 257), (1, 65537), (700, 1028)]


@pytest.mark.parametrize("shape", DROP_SHAPES, ids=str)
@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_and_its_gradients(device, dtype, shape):
    rng = np.random.default_rng(11)
    x, r, e = (rng.standard_normal(shape).astype(dtype) for _ in range(3))
    for p, seed, stream, residual in ((0.1, 7, 0, False), (0.5, -3, 5, True), (0.0, 1 << 40, 1, True), (0.875, (1 << 63) - 1, (1 << 45) + 3, False)):
        tx, tr = put(device, x).set_rqs_gradient(True), put(device, r).set_rqs_gradient(True)
        y = tx.dropout(p, seed, stream, tr if residual else None)
        assert np.array_equal(y.numpy(), S.dropout(x, p, seed, stream, r if residual else None))
        y.backward(put(device, e))
        assert np.array_equal(tx.gradient.numpy(), S.dropout(e, p, seed, stream))
        if residual:
            assert np.array_equal(tr.gradient.numpy(), e)


@pytest.mark.parametrize("view", VIEWS)
@pytest.mark.parametrize("shape", [(5, 7), (12, 64), (3, 4, 20), (40, 130)], ids=str)
def test_dropout_mask_does_not_depend_on_the_layout(device, shape, view):
    rng = np.random.default_rng(12)
    x, r = rng.standard_normal(shape).astype(np.float32), rng.standard_normal(shape).astype(np.float32)
    for other in VIEWS:
        y = put(device, x, view).dropout(0.3, 99, 4, put(device, r, other))
        assert np.array_equal(y.numpy(), S.dropout(x, 0.3, 99, 4, r))


def test_dropped_elements_are_zero_whatever_they_were(device):
    x = np.full(4000, np.nan, dtype=np.float32)
    x[::2] = np.inf
    y = put(device, x).dropout(0.4, 5).numpy()
    keep = S.keeps((4000,), 0.4, 5, 0)
    assert (y[~keep] == 0).all() and not np.isfinite(y[keep]).any()
    assert abs((~keep).mean() - 0.4) < 0.04   # five standard deviations


def test_dropout_of_one_value_standing_for_all(device):
    t = Tensor.of(np.float32, [30, 40], 2.0).to(device)
    assert np.array_equal(t.dropout(0.5, 3).numpy(), S.dropout(np.full((30, 40), 2.0, np.float32), 0.5, 3, 0))
    assert t.is_virtual


def test_dropout_into_its_source_and_into_a_view(device):
    x = np.random.default_rng(13).standard_normal((20, 36)).astype(np.float32)
    t = put(device, x)
    arr = t.ndconf.as_inline_array()
    c = arr.ctypes.data_as(C.POINTER(C.c_int32))
    L.check(L.lib.nk_dropout(device.ctx, L.NK_F32, 2, t._data.buf, c, t._data.buf, c, t._data.buf, c, 0.25, 1, 2), device.ctx)
    assert np.array_equal(t.numpy(), S.dropout(x, 0.25, 1, 2, x))
    big = put(device, np.zeros((24, 40), np.float32))
    part = big[2:22, 3:39]
    parr, s = part.ndconf.as_inline_array(), put(device, x)
    L.check(L.lib.nk_dropout(device.ctx, L.NK_F32, 2, part._data.buf, parr.ctypes.data_as(C.POINTER(C.c_int32)), s._data.buf, c, None, None, 0.25, 1, 2), device.ctx)
    want = np.zeros((24, 40), np.float32)
    want[2:22, 3:39] = S.dropout(x, 0.25, 1, 2)
    assert np.array_equal(big.numpy(), want)


# ---- the gated block -------------------------------------------------------------------------------------------------------------
def gated_case(device, rng, dtype, t, d, h, fun, views=("dense", "dense", "dense", "dense"), positive=False):
    draw = rng.random if positive else rng.standard_normal
    x, wg, wu = draw((t, d)).astype(dtype), (draw((d, h)) / np.sqrt(d)).astype(dtype), (draw((d, h)) / np.sqrt(d)).astype(dtype)
    e = rng.standard_normal((t, h)).astype(dtype)
    tx, tg, tu = (put(device, a, v).set_rqs_gradient(True) for a, v in zip((x, wg, wu), views))
    y = tx.gated(tg, tu, fun)
    S.assert_within(y.numpy(), S.gated(x, wg, wu, fun)[0], f"y {t} {d} {h}")
    free = put(device, x, views[0]).gated(put(device, wg, views[1]), put(device, wu, views[2]), fun)   # nothing kept for a backward pass
    assert np.array_equal(free.numpy(), y.numpy())
    y.backward(put(device, e, views[3]))
    for name, got, want in zip(("dx", "dwg", "dwu"), (tx, tg, tu), S.gated_gradients(x, wg, wu, e, fun)):
        S.assert_within(got.gradient.numpy(), want, f"{name} {t} {d} {h}")


GATED_SIZES = [(1, 1, 1), (1, 5, 3), (2, 64, 64), (1, 300, 129), (3, 257, 96), (4, 96, 260), (7, 33, 65), (8, 1000, 200), (9, 200, 1000), (16, 128, 128), (17, 100, 130),
               (31, 64, 40), (32, 515, 77), (63, 64, 64), (64, 64, 64), (65, 130, 70), (100, 31, 300), (128, 256, 512), (130, 257, 515), (300, 512, 365), (515, 129, 1027)]


@pytest.mark.parametrize("size", GATED_SIZES, ids=str)
@pytest.mark.parametrize("dtype", TYPES)
def test_gated_and_its_gradients(device, dtype, size):
    gated_case(device, np.random.default_rng(sum(size)), dtype, *size, "silu")


# some tokens: tiles shared by several multiprocessors, chunks and tiles that end inside, one chunk or many per tile
SOME_SIZES = [(9, 300, 1027), (10, 128, 1024), (16, 1000, 129), (17, 2050, 64), (24, 515, 900), (32, 64, 2048), (33, 130, 2050), (48, 128, 4096), (64, 777, 260), (50, 4100, 70),
              (12, 66, 20000), (64, 1023, 1025)]


@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("size", SOME_SIZES, ids=str)
def test_gated_some_tokens(device, size, turned):
    gated_case(device, np.random.default_rng(sum(size)), np.float32, *size, "silu", ("dense", "turned" if turned else "dense", "turned" if turned else "dense", "dense"))


@pytest.mark.parametrize("fun", L.GATES)
@pytest.mark.parametrize("size", [(1, 70, 90), (5, 64, 48), (24, 200, 136), (200, 300, 260)], ids=str)
@pytest.mark.parametrize("dtype", TYPES)
def test_gated_functions(device, dtype, size, fun):
    gated_case(device, np.random.default_rng(21), dtype, *size, fun)


@pytest.mark.parametrize("view", VIEWS[1:])
@pytest.mark.parametrize("size", [(1, 70, 90), (6, 72, 40), (40, 100, 60), (200, 260, 300)], ids=str)
@pytest.mark.parametrize("dtype", TYPES)
def test_gated_of_views(device, dtype, size, view):
    rng = np.random.default_rng(22)
    gated_case(device, rng, dtype, *size, "gelu", (view,) * 4)
    gated_case(device, rng, dtype, *size, "silu", ("dense", view, "dense", "dense"))
    gated_case(device, rng, dtype, *size, "silu", ("dense", "turned", view, view))


def test_gated_long_sums_of_one_sign(device):
    """Nothing cancels: a sum that is cut short or truncated on the way shows."""
    rng = np.random.default_rng(23)
    gated_case(device, rng, np.float32, 96, 4096, 80, "idy", positive=True)
    gated_case(device, rng, np.float32, 2, 8192, 40, "idy", positive=True)
    gated_case(device, rng, np.float32, 2048, 96, 100, "idy", positive=True)


def test_gated_tokens_that_are_not_finite_stay_apart(device):
    rng = np.random.default_rng(24)
    for t in (4, 200):
        x, wg, wu = rng.standard_normal((t, 96)).astype(np.float32), rng.standard_normal((96, 128)).astype(np.float32), rng.standard_normal((96, 128)).astype(np.float32)
        clean = put(device, x).gated(put(device, wg), put(device, wu)).numpy()
        x[1, 3], x[2, 95] = np.nan, np.inf
        y = put(device, x).gated(put(device, wg), put(device, wu)).numpy()
        assert np.isnan(y[1]).all() and not np.isfinite(y[2]).all()
        rest = [i for i in range(t) if i not in (1, 2)]
        assert np.array_equal(y[rest], clean[rest])


def test_gated_same_weights_twice_and_the_same_bits_every_time(device):
    rng = np.random.default_rng(25)
    x, w, e = rng.standard_normal((150, 96)).astype(np.float32), (rng.standard_normal((96, 200)) / 10).astype(np.float32), rng.standard_normal((150, 200)).astype(np.float32)
    got = []
    for _ in range(2):
        tx, tw = put(device, x).set_rqs_gradient(True), put(device, w).set_rqs_gradient(True)
        y = tx.gated(tw, tw, "sig")
        y.backward(put(device, e))
        got.append((y.numpy(), tx.gradient.numpy(), tw.gradient.numpy()))
    assert all(np.array_equal(a, b) for a, b in zip(*got))
    dx, dwg, dwu = S.gated_gradients(x, w, w, e, "sig")
    S.assert_within(got[0][1], dx, "dx")
    S.assert_within(got[0][2], (dwg[0] + dwu[0], dwg[1] + dwu[1] + 2 * S.unit(np.float32) * np.abs(dwg[0] + dwu[0])), "dw")


@pytest.mark.parametrize("wanted", ["x", "g", "u", "xu", "gu"])
def test_gated_only_the_gradients_asked_for(device, wanted):
    rng = np.random.default_rng(26)
    for t in (3, 40, 150):
        x, wg, wu, e = (rng.standard_normal(s).astype(np.float32) for s in ((t, 96), (96, 128), (96, 128), (t, 128)))
        tx, tg, tu = (put(device, a).set_rqs_gradient(k in wanted) for a, k in zip((x, wg, wu), "xgu"))
        tx.gated(tg, tu).backward(put(device, e))
        for k, t_, want in zip("xgu", (tx, tg, tu), S.gated_gradients(x, wg, wu, e, "silu")):
            if k in wanted:
                S.assert_within(t_.gradient.numpy(), want, k)
            else:
                assert t_.gradient is None


# ---- together --------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("size", [(1, 64, 96), (12, 96, 160), (200, 128, 256)], ids=str)
def test_a_feed_forward_sub_layer(device, size):
    """y = x + dropout(gated(norm(x)) @ down), forward and backward, in double precision against the same in 64 bits or more and, for one
    element of every leaf, against differences."""
    t, d, h = size
    rng = np.random.default_rng(31)
    leaves = {"x": rng.standard_normal((t, d)), "gain": 1 + 0.1 * rng.standard_normal(d), "shift": 0.1 * rng.standard_normal(d),
              "wg": rng.standard_normal((d, h)) / np.sqrt(d), "wu": rng.standard_normal((d, h)) / np.sqrt(d), "wd": rng.standard_normal((h, d)) / np.sqrt(h)}
    e = rng.standard_normal((t, d))

    def plain(v):
        hidden = S.gated(S.norm(v["x"], v["gain"], v["shift"], 1e-5)[0].astype(np.float64), v["wg"], v["wu"], "silu")[0][0]
        keep = S.keeps((t, d), 0.2, 17, 3)
        return v["x"] + np.where(keep, (hidden @ v["wd"].astype(S.WIDE)) / S.WIDE(0.8), 0)

    T = {k: put(device, v).set_rqs_gradient(True) for k, v in leaves.items()}
    y = (T["x"].layer_norm(T["gain"], T["shift"]).gated(T["wg"], T["wu"]) @ T["wd"]).dropout(0.2, 17, 3, T["x"])
    assert np.abs(y.numpy() - plain(leaves)).max() < 1e-11
    y.backward(put(device, e))
    for k, v in leaves.items():
        at = tuple(int(rng.integers(0, s)) for s in v.shape)
        step, values = 1e-5, []
        for sign in (1, -1):
            moved = {n: a.copy() for n, a in leaves.items()}
            moved[k][at] += sign * step
            values.append((plain(moved) * e).sum())
        slope = float(values[0] - values[1]) / (2 * step)
        got = T[k].gradient.numpy()[at]
        # the difference's own error: the third derivative times step^2 (1e-10), and the sum's rounding over the step
        assert abs(slope - got) < 1e-7 * max(1.0, abs(got)) + 1e-6, (k, at)
    # twice through the same graph: the gradients add up
    once = {k: v.gradient.numpy().copy() for k, v in T.items()}
    y.backward(put(device, e))
    for k in T:
        assert np.abs(T[k].gradient.numpy() - 2 * once[k]).max() <= 4 * S.unit(np.float64) * np.abs(once[k]).max()


def test_two_contexts_at_work_at_once(device):
    """The calls bring their own workspace and share nothing."""
    rng = np.random.default_rng(32)
    x, e = rng.standard_normal((300, 5000)).astype(np.float32), rng.standard_normal((300, 5000)).astype(np.float32)
    want, xh, r = S.norm(x, None, None, 1e-5)
    bound = S.norm_bound(x, None, want, xh, r, S.unit(np.float32))
    second = C.c_void_p()
    L.check(L.lib.nk_device_open(device.ordinal, C.byref(second)))
    try:
        t, out = put(device, x), [put(device, np.zeros_like(x)) for _ in range(2)]
        device.sync()
        arr = t.ndconf.as_inline_array()
        c = arr.ctypes.data_as(C.POINTER(C.c_int32))
        for _ in range(20):
            for ctx, o in ((device.ctx, out[0]), (second, out[1])):
                L.check(L.lib.nk_layer_norm(ctx, L.NK_F32, 2, o._data.buf, c, t._data.buf, c, None, None, None, None, 1e-5, None), ctx)
        L.check(L.lib.nk_sync(second), second)
        device.sync()
        for o in out:
            S.assert_within(o.numpy(), (want, bound), "two contexts")
    finally:
        L.lib.nk_device_close(second)


# ---- refusals --------------------------------------------------------------------------------------------------------------------
def test_refusals(device):
    x, w, v = (put(device, np.ones(s, np.float32)) for s in ((4, 6), (6, 8), (6,)))
    out, stats, kept = put(device, np.zeros((4, 6), np.float32)), put(device, np.zeros(8, np.float32)), put(device, np.zeros(2 * 4 * 8, np.float32))

    def cfg(t, shape=None):
        arr = np.array(t.ndconf.as_inline_array() if shape is None else shape, dtype=np.int32)
        keep.append(arr)
        return arr.ctypes.data_as(C.POINTER(C.c_int32))
    keep = []
    N = (None, None)

    def b(t):
        return t._data.buf, cfg(t)
    virtual = (out._data.buf, cfg(out, [4, 6] + [0] * 8))
    wide = (v._data.buf, cfg(v, [7, 1, 1, 0, 1]))
    small = put(device, np.zeros(7, np.float32))
    double = put(device, np.zeros((4, 6)))
    lib, ctx = L.lib, device.ctx
    BAD, UNS, OUT = L.NK_ERR_BAD_ARG, L.NK_ERR_UNSUPPORTED, L.NK_ERR_BOUNDS

    def norm(d=b(out), s=b(x), g=b(v), sh=b(v), eps=1e-5, st=None, dt=L.NK_F32):
        return lib.nk_layer_norm(ctx, dt, 2, *d, *s, *g, *sh, eps, st)
    assert norm() == L.NK_OK and norm(g=N, sh=N, eps=0.0, st=stats._data.buf) == L.NK_OK
    assert norm(dt=L.NK_I32) == UNS and norm(eps=-1.0) == BAD and norm(eps=float("nan")) == BAD and norm(d=virtual) == BAD
    assert norm(g=wide) == OUT and norm(sh=b(small)) == BAD and norm(d=N) == BAD and norm(s=b(double)) == BAD and norm(s=b(w)) == BAD
    assert norm(st=small._data.buf) == OUT and norm(st=double._data.buf) == BAD

    def ngrad(d=b(out), g=N, s=N, e=b(x), src=b(x), gain=N, st=stats._data.buf):
        return lib.nk_layer_norm_grad(ctx, L.NK_F32, 2, *d, *g, *s, *e, *src, *gain, st)
    assert ngrad() == L.NK_OK and ngrad(d=N) == L.NK_OK
    assert ngrad(st=None) == BAD and ngrad(st=small._data.buf) == OUT and ngrad(d=virtual) == BAD and ngrad(e=b(w)) == BAD and ngrad(g=b(small)) == BAD

    def drop(d=b(out), s=b(x), r=N, p=0.5, dt=L.NK_F32):
        return lib.nk_dropout(ctx, dt, 2, *d, *s, *r, p, 1, 2)
    assert drop() == L.NK_OK
    for p in (1.0, -0.1, 1.5, float("nan"), float("inf")):
        assert drop(p=p) == BAD
    assert drop(dt=L.NK_I64) == UNS and drop(d=virtual) == BAD and drop(r=b(w)) == BAD and drop(s=b(double)) == BAD

    y = put(device, np.zeros((4, 8), np.float32))
    silu = L.FUN["silu"]

    def gated(f=silu, d=b(y), s=b(x), g=b(w), u=b(w), k=None, dt=L.NK_F32):
        return lib.nk_gated(ctx, f, dt, *d, *s, *g, *u, k)
    assert gated() == L.NK_OK and gated(k=kept._data.buf) == L.NK_OK
    assert gated(f=99) == BAD and gated(f=-1) == BAD and gated(f=L.FUN["exp"]) == UNS and gated(dt=L.NK_I8) == UNS
    assert gated(g=b(x)) == BAD and gated(u=b(y)) == BAD and gated(d=b(x)) == BAD and gated(s=b(double)) == BAD and gated(k=stats._data.buf) == OUT

    def ggrad(k=kept._data.buf, e=b(y), d=b(out), g=N, u=N):
        return lib.nk_gated_grad(ctx, silu, L.NK_F32, *d, *g, *u, *e, *b(x), *b(w), *b(w), k)
    assert ggrad() == L.NK_OK and ggrad(d=N) == L.NK_OK
    assert ggrad(k=None) == BAD and ggrad(k=stats._data.buf) == OUT and ggrad(e=b(x)) == BAD and ggrad(g=b(x)) == BAD and ggrad(d=virtual) == BAD
    device.sync()


# ---- calls that are seldom made ----------------------------------------------------------------------------------------------------
class Raw:
    """Buffers of torch's memory for the C entry points"""

    def __init__(self, ctx):
        self.ctx, self.keep = ctx, []

    def __call__(self, values, shape=None, strides=None):
        """a buffer with these values, and the view of it (dense, or of the given shape and strides)"""
        import torch
        t = torch.as_tensor(values, device="cuda").contiguous()
        buf = C.c_void_p()
        L.check(L.lib.nk_wrap(self.ctx, L.NK_F32 if t.dtype == torch.float32 else L.NK_F64, C.c_void_p(t.data_ptr()), t.numel(), C.byref(buf)), self.ctx)
        shape = list(t.shape) if shape is None else list(shape)
        dense = [int(np.prod(shape[k + 1:])) for k in range(len(shape))]
        arr = np.array(shape + (dense if strides is None else list(strides)) + dense + [0] * len(shape) + [1] * len(shape), dtype=np.int32)
        self.keep.append((t, arr))
        return t, (buf, arr.ctypes.data_as(C.POINTER(C.c_int32)))


def sub_layer_calls(ctx, dtype, t, d, h):
    """One pass through everything, forward and backward, on ctx's stream: the inputs, the results, and the calls as a function"""
    import torch
    raw, dt = Raw(ctx), L.NK_F32 if dtype == np.float32 else L.NK_F64
    rng = np.random.default_rng(t + d + h)
    (x, bx), (e, be) = (raw(rng.standard_normal((t, d)).astype(dtype)) for _ in range(2))
    (wg, bwg), (wu, bwu) = (raw((rng.standard_normal((d, h)) / np.sqrt(d)).astype(dtype)) for _ in range(2))
    (wd, bwd), (gain, bgain) = raw(rng.standard_normal((t, h)).astype(dtype)), raw(1 + 0.1 * rng.standard_normal(d).astype(dtype))
    (n, bn), (stats, bstats), (y, by), (kept, bkept), (o, bo) = (raw(np.zeros(s, dtype)) for s in ((t, d), (2, t), (t, h), (2, t, h), (t, h)))
    (dn, bdn), (dg, bdg), (du, bdu), (dx, bdx), (dgain, bdgain), (dshift, bdshift) = (raw(np.zeros(s, dtype)) for s in ((t, d), (d, h), (d, h), (t, d), (d,), (d,)))
    N, lib, silu = (None, None), L.lib, L.FUN["silu"]

    def run():
        L.check(lib.nk_layer_norm(ctx, dt, 2, *bn, *bx, *bgain, *N, 1e-5, bstats[0]), ctx)
        L.check(lib.nk_gated(ctx, silu, dt, *by, *bn, *bwg, *bwu, bkept[0]), ctx)
        L.check(lib.nk_dropout(ctx, dt, 2, *bo, *by, *bwd, 0.25, 7, 8), ctx)
        L.check(lib.nk_gated_grad(ctx, silu, dt, *bdn, *bdg, *bdu, *bo, *bn, *bwg, *bwu, bkept[0]), ctx)
        L.check(lib.nk_layer_norm_grad(ctx, dt, 2, *bdx, *bdgain, *bdshift, *bdn, *bx, *bgain, bstats[0]), ctx)
    torch.cuda.synchronize()
    return (x, wg), (n, y, o, dg, du, dx, dgain, dshift), run, raw


SUB_LAYERS = [(np.float32, 1, 128, 200), (np.float32, 24, 300, 257), (np.float32, 300, 260, 515), (np.float32, 3000, 640, 100), (np.float64, 5, 70, 96), (np.float64, 200, 130, 70),
              (np.float32, 2, 140000, 20)]


@pytest.mark.parametrize("case", SUB_LAYERS, ids=lambda c: f"{c[0].__name__}-{c[1]}-{c[2]}-{c[3]}")
def test_captured_once_and_replayed(device, case):
    import torch
    (x, wg), results, run, raw = sub_layer_calls(device.ctx, *case)
    stream = torch.cuda.ExternalStream(L.lib.nk_stream(device.ctx))
    run()   # (what is looked up once per device has been)
    device.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        run()
    for k in range(3):   # other values in the same places
        x.mul_(0.75).add_(0.125)
        wg.mul_(-1.25)
        torch.cuda.synchronize()
        run()
        device.sync()
        want = [r.clone() for r in results]
        for r in results:
            r.fill_(float("nan"))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
            if k == 2:
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and bool(torch.isfinite(a).all()) for a, b in zip(results, want))


def test_two_graphs_and_eager_calls_at_work_at_once(device):
    import torch
    second = C.c_void_p()
    L.check(L.lib.nk_device_open(device.ordinal, C.byref(second)))
    try:
        sides = []
        for ctx, case in ((device.ctx, (np.float32, 300, 260, 515)), (second, (np.float32, 24, 300, 257)), (second, (np.float32, 500, 200, 300))):
            _, results, run, raw = sub_layer_calls(ctx, *case)
            run()
            L.check(L.lib.nk_sync(ctx), ctx)
            want, stream = [r.clone() for r in results], torch.cuda.ExternalStream(L.lib.nk_stream(ctx))
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
                run()
            sides.append((results, want, graph, torch.cuda.Stream(), run, raw))
        for k in range(10):
            for results, want, graph, own, run, raw in sides:
                with torch.cuda.stream(own):   # a stream of its own: the graphs have memory of their own
                    graph.replay()
            torch.cuda.synchronize()
            for results, want, graph, own, run, raw in sides:
                assert all(torch.equal(a, b) for a, b in zip(results, want))
        for k in range(10):   # both contexts, eagerly
            for results, want, graph, own, run, raw in sides:
                run()
        torch.cuda.synchronize()
        for results, want, graph, own, run, raw in sides:
            assert all(torch.equal(a, b) for a, b in zip(results, want))
        del sides, results, want, graph, own, run, raw
    finally:
        L.lib.nk_device_close(second)


@pytest.mark.parametrize("size", [(1, 70, 90), (5, 64, 48), (24, 96, 130), (200, 260, 300)], ids=str)
@pytest.mark.parametrize("dtype", TYPES)
def test_gated_of_one_value_standing_for_many(device, dtype, size):
    """rows or whole matrices that are one row or one value in memory, as operands and as the error"""
    t, d, h = size
    rng, raw, dt, ctx = np.random.default_rng(41), Raw(device.ctx), L.NK_F32 if dtype == np.float32 else L.NK_F64, device.ctx
    vx, vg, vu, ve = rng.standard_normal(d).astype(dtype), (rng.standard_normal(h) / d).astype(dtype), np.array([0.5 / d], dtype), np.array([0.75], dtype)
    x, wg, wu, e = np.tile(vx, (t, 1)), np.tile(vg, (d, 1)), np.full((d, h), vu[0]), np.full((t, h), ve[0])
    _, bx = raw(vx, (t, d), (0, 1))
    _, bg = raw(vg, (d, h), (0, 1))
    _, bu = raw(vu, (d, h), (0, 0))
    _, be = raw(ve, (t, h), (0, 0))
    (y, by), (kept, bk), (dx, bdx), (dg, bdg), (du, bdu) = (raw(np.zeros(s, dtype)) for s in ((t, h), (2, t, h), (t, d), (d, h), (d, h)))
    import torch
    torch.cuda.synchronize()
    L.check(L.lib.nk_gated(ctx, L.FUN["gelu"], dt, *by, *bx, *bg, *bu, bk[0]), ctx)
    L.check(L.lib.nk_gated_grad(ctx, L.FUN["gelu"], dt, *bdx, *bdg, *bdu, *be, *bx, *bg, *bu, bk[0]), ctx)
    device.sync()
    S.assert_within(y.cpu().numpy(), S.gated(x, wg, wu, "gelu")[0], "y")
    for name, got, want in zip(("dx", "dwg", "dwu"), (dx, dg, du), S.gated_gradients(x, wg, wu, e, "gelu")):
        S.assert_within(got.cpu().numpy(), want, name)


def test_one_leaf_in_every_place(device):
    """The same tensor as several operands: its gradients add up."""
    rng = np.random.default_rng(42)
    u = S.unit(np.float64)
    a, e = rng.standard_normal((60, 60)) / 4, rng.standard_normal((60, 60))
    ta = put(device, a).set_rqs_gradient(True)
    ta.gated(ta, ta, "tanh").backward(put(device, e))
    parts = S.gated_gradients(a, a, a, e, "tanh")
    want, bound = sum(p[0] for p in parts), sum(p[1] for p in parts)
    S.assert_within(ta.gradient.numpy(), (want, bound + 3 * u * sum(np.abs(p[0]) for p in parts)), "a")
    x, v, e = rng.standard_normal((30, 40)), rng.standard_normal(40), rng.standard_normal((30, 40))
    tx, tv = put(device, x), put(device, v).set_rqs_gradient(True)
    tx.layer_norm(tv, tv).backward(put(device, e))
    _, dgain, dshift = S.norm_gradients(x, v, e, 1e-5, u)
    S.assert_within(tv.gradient.numpy(), (dgain[0] + dshift[0], dgain[1] + dshift[1] + 2 * u * (np.abs(dgain[0]) + np.abs(dshift[0]))), "v")
    tx = put(device, x).set_rqs_gradient(True)
    y = tx.dropout(0.5, 3, 4, residual=tx)
    assert np.array_equal(y.numpy(), S.dropout(x, 0.5, 3, 4, x))
    y.backward(put(device, e))
    assert np.array_equal(tx.gradient.numpy(), e + S.dropout(e, 0.5, 3, 4))


def test_backward_without_an_error(device):
    """ones, one value standing for all"""
    rng = np.random.default_rng(43)
    x, wg, wu = rng.standard_normal((20, 30)), rng.standard_normal((30, 50)) / 5, rng.standard_normal((30, 50)) / 5
    tx, tg, tu = (put(device, a).set_rqs_gradient(True) for a in (x, wg, wu))
    tx.gated(tg, tu).backward()
    for got, want in zip((tx, tg, tu), S.gated_gradients(x, wg, wu, np.ones((20, 50)), "silu")):
        S.assert_within(got.gradient.numpy(), want, "gated")
    gain = 1 + rng.standard_normal(30)
    tx, tg = put(device, x).set_rqs_gradient(True), put(device, gain).set_rqs_gradient(True)
    tx.layer_norm(tg).backward()
    dx, dgain, _ = S.norm_gradients(x, gain, np.ones((20, 30)), 1e-5, S.unit(np.float64))
    S.assert_within(tx.gradient.numpy(), dx, "dx")
    S.assert_within(tg.gradient.numpy(), dgain, "dgain")
    tx = put(device, x).set_rqs_gradient(True)
    tx.dropout(0.3, 1).backward()
    assert np.array_equal(tx.gradient.numpy(), S.dropout(np.ones((20, 30)), 0.3, 1, 0))


@pytest.mark.parametrize("shape", [(5000, 96), (3000, 777), (700, 4096), (320, 12001), (2, 140001)], ids=str)
def test_layer_norm_in_place_of_many_and_of_long_rows(device, shape):
    import torch
    rng, raw, ctx = np.random.default_rng(44), Raw(device.ctx), device.ctx
    x, e = rng.standard_normal(shape).astype(np.float32), rng.standard_normal(shape).astype(np.float32)
    (tx, bx), (ty, by), (te, be), (tr, br) = (raw(a) for a in (x, x, e, e))
    (s0, bs), (dx, bdx), (d0, bd0), (d1, bd1) = (raw(np.zeros(s, np.float32)) for s in ((2, shape[0]), shape, shape[1:], shape[1:]))
    N = (None, None)
    torch.cuda.synchronize()
    for drain in (by, by):   # (the second time on what the first one left, as one after the other would)
        L.check(L.lib.nk_layer_norm(ctx, L.NK_F32, 2, *bdx, *by, *N, *N, 1e-5, None), ctx)
        L.check(L.lib.nk_layer_norm(ctx, L.NK_F32, 2, *drain, *by, *N, *N, 1e-5, None), ctx)
    device.sync()
    assert torch.equal(ty, dx)
    L.check(L.lib.nk_layer_norm(ctx, L.NK_F32, 2, *bdx, *bx, *N, *N, 1e-5, bs[0]), ctx)
    L.check(L.lib.nk_layer_norm_grad(ctx, L.NK_F32, 2, *bdx, *bd0, *N, *be, *bx, *N, bs[0]), ctx)
    L.check(L.lib.nk_layer_norm_grad(ctx, L.NK_F32, 2, *br, *bd1, *N, *br, *bx, *N, bs[0]), ctx)
    device.sync()
    assert torch.equal(tr, dx) and torch.equal(d0, d1)
    S.assert_within(tr.cpu().numpy(), S.norm_gradients(x, None, e, 1e-5, S.unit(np.float32))[0], "dx")


@pytest.mark.parametrize("fun", L.GATES)
def test_f32_gates_over_their_whole_range(device, fun):
    """x = [v, 1] with weights [1, 0] and [0, 1] (in one tile of F32 multiply-adds: exact) give g = v, u = 1, y = f(v) and, for an error of ones,
    dx = [f'(v), f(v)]. With e = e^-|k v|: 4 u for e (2 units in the last place), 4 for the quotient, 1 each for 1 + e, e t, v s, 2 for e's share in 1 + e,
    and 3 for gelu's correction: 16 u; the derivatives have two such factors and three operations more: 36 u of their terms."""
    v = np.concatenate([np.linspace(-20, 20, 4001), np.linspace(-120, 120, 999), np.geomspace(1e-30, 3e38, 400), -np.geomspace(1e-30, 3e38, 400), [0.0, -0.0]]).astype(np.float32)
    x = np.stack([v, np.ones_like(v)], 1)
    tx = put(device, x).set_rqs_gradient(True)
    y = tx.gated(put(device, np.array([[1], [0]], np.float32)), put(device, np.array([[0], [1]], np.float32)), fun)
    y.backward()
    w, u = v.astype(S.WIDE), S.unit(np.float32)
    if fun in ("idy", "relu"):
        f, df = S.gate(fun, v)
        f_off, df_off = 2 * u * np.abs(f), 2 * u * np.abs(df)
    else:
        k = S.WIDE({"gelu": 1.702, "tanh": 2}.get(fun, 1))
        e = np.exp(-k * np.abs(w))
        small, large = e / (1 + e), 1 / (1 + e)
        s, rest = np.where(w < 0, small, large), np.where(w < 0, large, small)
        if fun == "tanh":
            f, df = np.tanh(w), 4 * s * rest
            terms = df
        elif fun == "sig":
            f, df = s, s * rest
            terms = df
        else:
            f, df = w * s, s + k * w * s * rest
            terms = s + k * np.abs(w) * s * rest
        f_off, df_off = 16 * u * np.abs(f), 36 * u * terms
    denormal = 2.0 ** -146   # what a result, or a factor of it, may be off by where it is below the normal range
    S.assert_within(y.numpy()[:, 0], (f, f_off + denormal * (1 + np.minimum(np.abs(w), 200))), "f")
    S.assert_within(tx.gradient.numpy()[:, 1], (f, f_off + denormal * (1 + np.minimum(np.abs(w), 200))), "f again")
    S.assert_within(tx.gradient.numpy()[:, 0], (df, df_off + denormal * (1 + 2 * np.minimum(np.abs(w), 200))), "f'")
