"""Layer norm, dropout and the gated block without a GPU: the plain implementations that the GPU tests compare with, and what is refused
before any device is needed."""
import ctypes as C

import numpy as np
import pytest

import sublayer as S


def test_generator_gives_the_published_words():
    """The known answers of Philox4x32-10: counter and key all zeros, all ones, and digits of pi."""
    def words(counter, key):
        return [int(w) for w in S.philox4x32(counter, key)]
    assert words([0, 0, 0, 0], (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert words([0xFFFFFFFF] * 4, (0xFFFFFFFF, 0xFFFFFFFF)) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert words([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], (0xA4093822, 0x299F31D0)) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


@pytest.mark.parametrize("fun", ["sig", "silu", "gelu", "relu", "tanh", "idy"])
def test_plain_gradients_against_differences(fun):
    rng = np.random.default_rng(3)
    x, wg, wu, e = (rng.standard_normal(s) for s in ((3, 4), (4, 5), (4, 5), (3, 5)))
    grads = S.gated_gradients(x, wg, wu, e, fun)
    for i, a in enumerate((x, wg, wu)):
        for at in np.ndindex(a.shape):
            keep, h = a[at], 1e-6
            a[at] = keep + h
            up = (S.gated(x, wg, wu, fun)[0][0] * e).sum()
            a[at] = keep - h
            down = (S.gated(x, wg, wu, fun)[0][0] * e).sum()
            a[at] = keep
            assert abs((up - down) / (2 * h) - grads[i][0][at]) < 1e-7 * max(1, abs(grads[i][0][at]))


def test_plain_norm_gradients_against_differences():
    rng = np.random.default_rng(4)
    x, gain, shift, e = rng.standard_normal((3, 7)), rng.standard_normal(7), rng.standard_normal(7), rng.standard_normal((3, 7))
    grads = S.norm_gradients(x, gain, e, 1e-5, S.unit(np.float64))
    for i, a in enumerate((x, gain, shift)):
        for at in np.ndindex(a.shape):
            keep, h = a[at], 1e-6
            a[at] = keep + h
            up = (S.norm(x, gain, shift, 1e-5)[0] * e).sum()
            a[at] = keep - h
            down = (S.norm(x, gain, shift, 1e-5)[0] * e).sum()
            a[at] = keep
            assert abs((up - down) / (2 * h) - grads[i][0][at]) < 1e-7 * max(1, abs(grads[i][0][at]))


def test_refused_before_a_device_is_needed():
    from neureka_b200 import _lib as L
    from neureka_b200.tensor import Tensor
    x, v = Tensor.of(np.float32, [4, 6], np.zeros(24)), Tensor.of(np.float32, [5], np.zeros(5))
    w, w2 = Tensor.of(np.float32, [6, 3], np.zeros(18)), Tensor.of(np.float32, [6, 2], np.zeros(12))
    with pytest.raises(ValueError, match="does not fit rows of 6"):
        x.layer_norm(v)
    with pytest.raises(ValueError, match="does not fit rows of 6"):
        x.layer_norm(None, Tensor.of(np.float32, [4, 6], np.zeros(24)))
    with pytest.raises(ValueError, match="residual"):
        x.dropout(0.5, 1, 0, v)
    with pytest.raises(ValueError, match="64 bits"):
        x.dropout(0.5, 1 << 63)
    with pytest.raises(ValueError, match="no gate"):
        x.gated(w, w, "softplus")
    with pytest.raises(ValueError, match="do not make"):
        x.gated(w, w2)
    with pytest.raises(ValueError, match="rank-2"):
        x.gated(w, v)
    for call in (lambda: x.layer_norm(), lambda: x.dropout(0.5, 1), lambda: x.gated(w, w)):
        with pytest.raises(L.NeurekaCudaError, match="no CPU execution"):
            call()


def test_entry_points_refuse_a_missing_context():
    from neureka_b200 import _lib as L
    none = [None, None]
    assert L.lib.nk_layer_norm(None, L.NK_F32, 2, *none * 4, 1e-5, None) == L.NK_ERR_BAD_ARG
    assert L.lib.nk_layer_norm_grad(None, L.NK_F32, 2, *none * 6, None) == L.NK_ERR_BAD_ARG
    assert L.lib.nk_dropout(None, L.NK_F32, 2, *none * 3, 0.5, 0, 0) == L.NK_ERR_BAD_ARG
    assert L.lib.nk_gated(None, L.FUN["silu"], L.NK_F32, *none * 4, None) == L.NK_ERR_BAD_ARG
    assert L.lib.nk_gated_grad(None, L.FUN["silu"], L.NK_F32, *none * 7, None) == L.NK_ERR_BAD_ARG
    assert b"invalid context" in L.lib.nk_last_error(None)


def test_registered_beside_the_other_operations():
    from neureka_b200 import backend as B
    pairs = set(B.CudaBackend().pairs())
    assert {("layerNorm", B.LAYER_NORM), ("dropout", B.DROPOUT), ("gated", B.GATED)} <= pairs


def test_vectors_of_any_view_are_described_with_one_dim():
    """A gain or shift may be a row of a matrix, a slice with a step, or turned: the descriptor of rank 1 names the same elements."""
    from neureka_b200 import backend as B
    from neureka_b200.ndconf import NDConfiguration as ND
    from neureka_b200.tensor import Tensor
    m = Tensor.of(np.float32, [4, 12], np.arange(48))
    column = Tensor.of(np.float32, [12, 4], np.arange(48))
    for t in (m[2:3, 1:12:2], m[0:1, 0:12], column[2:9, 3:4].permute(1, 0), Tensor.of(np.float32, [5], np.arange(5))):
        _, at = B._cfg_vector(t)
        shape, strides, indices_map, offset, spread = (at[i] for i in range(5))
        flat = ND((shape,), (strides,), (indices_map,), (spread,), (offset,))
        assert flat.element_offsets().tolist() == t.ndconf.element_offsets().tolist()


@pytest.mark.parametrize("through", [False, True])
def test_a_node_lets_go_of_what_it_kept_with_its_last_reference(monkeypatch, through):
    """The operands, the statistics and the kept products of a step go with its result, not with the next run of the cycle collector."""
    import gc
    import weakref
    from neureka_b200 import functions as F
    from neureka_b200.tensor import Tensor

    def tensor(*shape):
        return Tensor.of(np.float32, shape, np.zeros(int(np.prod(shape))))

    def made(t):
        seen.append(weakref.ref(t))
        return t
    seen = []
    monkeypatch.setattr(F, "run_layer_norm", lambda x, gain, shift, eps, keep: (made(tensor(2, 3)), made(tensor(2, 2))))
    monkeypatch.setattr(F, "run_gated", lambda x, w_gate, w_up, fun, keep: (made(tensor(2, 5)), made(tensor(2, 2, 5))))
    monkeypatch.setattr(F, "run_layer_norm_gradients", lambda err, x, gain, shift, stats, wanted: [made(tensor(2, 3)), made(tensor(3)), made(tensor(3))])
    monkeypatch.setattr(F, "run_gated_gradients", lambda err, x, w_gate, w_up, kept, fun, wanted: [made(tensor(2, 3)), made(tensor(3, 5)), made(tensor(3, 5))])
    gc.collect()
    gc.disable()
    try:
        x, gain, shift, w_gate, w_up = (made(tensor(*s).set_rqs_gradient(True)) for s in ((2, 3), (3,), (3,), (3, 5), (3, 5)))
        y = x.layer_norm(gain, shift).gated(w_gate, w_up)
        if through:   # what the backward pass does with a node's parents
            errors = [act(y) for _, act in y.graph_node.parents]
            errors += [act(errors[0]) for _, act in y.graph_node.parents[0][0].graph_node.parents]
            assert [e.shape for e in errors] == [(2, 3), (3, 5), (3, 5), (2, 3), (3,), (3,)]
            del errors
        del x, gain, shift, w_gate, w_up, y
        assert [r for r in seen if r() is not None] == []
    finally:
        gc.enable()


def test_a_configuration_that_served_a_call_can_be_copied_and_pickled():
    import copy
    import pickle
    from neureka_b200.ndconf import NDConfiguration as ND
    from neureka_b200.tensor import Tensor
    t = Tensor.of(np.float32, [4, 6], np.arange(24))
    for c in (ND.of_shape((2, 3)), ND.virtual_of((5,)), t.ndconf, ND.of_shape((4, 6)).sliced([2, 3], [1, 0], [1, 2])):
        before = c.inline_pointer[0], c.rank, c.size, c.is_compact()
        for other in (pickle.loads(pickle.dumps(c)), copy.deepcopy(c), copy.copy(c)):
            assert other == c and hash(other) == hash(c)
            assert (other.inline_pointer[0], other.rank, other.size, other.is_compact()) == before
            assert [other.inline_pointer[i] for i in range(5 * c.rank)] == c.as_inline_array().tolist()
    assert np.array_equal(copy.deepcopy(t).numpy(), t.numpy())


def test_extents_of_any_kind_that_converts_to_a_number():
    from neureka_b200.ndconf import Layout, NDConfiguration as ND
    for shape in ((2, 3), [2, 3], (np.int64(2), np.int32(3)), (np.array(2), np.array(3)), [np.array(2), 3], iter((2, 3)), np.array([2, 3]), (2.0, 3.0)):
        c = ND.of_shape(shape)
        assert c.shape == (2, 3) and all(type(x) is int for x in c.shape) and c.strides == (3, 1)
    assert ND.of_shape((np.array(2), 3), Layout.COLUMN_MAJOR) == ND.of_shape((2, 3), Layout.COLUMN_MAJOR)
    assert ND.virtual_of((np.array(2), 3)) == ND.virtual_of([2, 3])
    for shape in ((2, 0), (np.array(0),)):
        with pytest.raises(ValueError, match="greater than 0"):
            ND.of_shape(shape)
    with pytest.raises(TypeError):
        ND.of_shape((2, None))


def test_a_device_has_nothing_that_is_no_tensor():
    from neureka_b200.device import CudaDevice
    from neureka_b200.tensor import Tensor
    device = object.__new__(CudaDevice)   # (none of these calls reaches the library)
    for what in (None, "a", 3, [], Tensor.of(np.float32, [2], [1, 2])):
        assert not device.has(what) and not device.contains(what)
        with pytest.raises(ValueError, match="not stored on this device"):
            device.restore(what)
        assert device.free(what) is device
