"""Layers of a Kipizen configuration whose keys and values are held in 4 bits, without a device."""
import copy

import numpy as np
import pytest

import packed_model as model
from onyxia_b200 import checkpoint, ir, kipizen
from onyxia_b200.ir import HostTensor
from onyxia_b200.kipizen import KipizenConfig

CFG = KipizenConfig.from_dict(model.CONFIG)


def test_modules_are_built_with_pools_of_bytes():
    assert [l.mixer.packed for l in CFG.layers if isinstance(l.mixer, kipizen.AttentionConfig)] == [True, True, True, False]
    stored = checkpoint.Weights.from_bf16({k: HostTensor.bf16(v).data.view(np.uint16).reshape(v.shape) for k, v in model.weights(model.CONFIG).items()})
    for w in (stored, kipizen.random_weights(CFG)):
        for dtype in (ir.F32, ir.BF16):
            assert kipizen.build(CFG, w, dtype)
    assert {k: v.shape for k, v in model.weights(model.CONFIG).items()} == kipizen.tensor_shapes(CFG)


@pytest.mark.parametrize("layer,changed,match", [
    (0, {"cache": "int4"}, "unknown cache type"), (0, {"dim": 24, "rot": None}, "multiples"), (2, {"vdim": 72}, "multiples"), (3, {"cache": "e2m1"}, "of the layer's own"),
    (0, {"differential": {"lambda_init": 0.5}}, "of the layer's own")], ids=str)
def test_layers_that_are_refused(layer, changed, match):
    c = copy.deepcopy(model.CONFIG)
    c["layers"][layer]["mixer"].update(changed)
    with pytest.raises(ValueError, match=match):
        KipizenConfig.from_dict(c)


def test_a_layer_without_a_cache_type_is_as_it_was():
    c = copy.deepcopy(model.CONFIG)
    for l in c["layers"]:
        l["mixer"].pop("cache", None)
    assert not any(l.mixer.packed for l in KipizenConfig.from_dict(c).layers if isinstance(l.mixer, kipizen.AttentionConfig))
