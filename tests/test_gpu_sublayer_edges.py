"""Layer norm, dropout and the gated block on the GPU, beside tests/test_gpu_sublayer.py: memory that a step gives back, sums that
rounding could carry away, operands that are not finite, and the precision of small calls."""
import gc

import numpy as np
import pytest

import sublayer as S
from test_gpu_sublayer import put

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
