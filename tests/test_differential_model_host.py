"""Differential layers of a Kipizen configuration, without a device."""
import copy

import numpy as np
import pytest

import differential_model as model
from onyxia_b200 import checkpoint, ir, kipizen
from onyxia_b200.ir import HostTensor
from onyxia_b200.kipizen import KipizenConfig

CFG = KipizenConfig.from_dict(model.CONFIG)


def weights():
    return checkpoint.Weights.from_bf16({k: HostTensor.bf16(v).data.view(np.uint16).reshape(v.shape) for k, v in model.weights(model.CONFIG).items()})


def test_shapes_are_those_that_the_module_is_built_from():
    assert {k: v.shape for k, v in model.weights(model.CONFIG).items()} == kipizen.tensor_shapes(CFG)
    random = kipizen.random_weights(CFG)
    for w in (weights(), random):
        for dtype in (ir.F32, ir.BF16):
            assert kipizen.build(CFG, w, dtype)


def test_lambda_begins_with_the_layers_number():
    assert [l.mixer.lambda_init for l in CFG.layers if isinstance(l.mixer, kipizen.AttentionConfig)] == [0.6, 0.3, None]


def test_keys_are_not_shared_with_a_differential_layer():
    for reader, source in ((2, 0), (3, 2)):
        c = copy.deepcopy(model.CONFIG)
        c["layers"][reader]["mixer"]["kv_from"] = source
        with pytest.raises(ValueError, match="keys of its own"):
            KipizenConfig.from_dict(c)


@pytest.mark.parametrize("name", ["l0.mix.lam.q1", "l0.mix.lam.k2", "l2.mix.head_norm", "l2.mix.q", "l0.mix.k.b"])
def test_a_tensor_of_another_size_is_refused(name):
    w = {k: HostTensor.bf16(v).data.view(np.uint16).reshape(v.shape) for k, v in model.weights(model.CONFIG).items()}
    w[name] = np.ascontiguousarray(w[name][:-1])
    with pytest.raises(ValueError):
        kipizen.build(CFG, checkpoint.Weights.from_bf16(w), ir.BF16)


def test_equal_maps_take_their_share_from_the_first():
    """The plain form itself: two equal maps and no window leave (1 - lambda) of one map, which the norm makes 1 again."""
    r = np.random.default_rng(0)
    c = dict(model.differential(heads=1, kv_heads=1, dim=8, vdim=8, lambda_init=0.5, window=64, rot=0), softcap=0.0)
    w = {n: r.standard_normal((16, 12)) for n in ("q", "k")} | {"q.b": np.zeros(16), "k.b": np.zeros(16), "v": r.standard_normal((8, 12)), "v.b": np.zeros(8), "o": np.eye(8)}
    for n in ("q", "k"):
        w[n][8:] = w[n][:8]
    w |= {"lam." + n: np.zeros(8) for n in ("q1", "k1", "q2", "k2")} | {"head_norm": np.full(8, 2.0)}
    got = model.mixer(r.standard_normal((5, 12)), w, c, 0.0)[0]
    assert np.allclose(np.sqrt((got ** 2).mean(-1)), 1.0)
