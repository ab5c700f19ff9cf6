"""A small Kipizen configuration whose keys and values are held in 4 bits, and the mixer's plain form for kipizen_ref.py."""
import numpy as np

import kipizen_ref as ref
import kipizen_util as util
import packed_util


def packed(heads=4, kv_heads=2, dim=32, vdim=64, scale=0.2, **more):
    return dict(util.attention(heads=heads, kv_heads=kv_heads, dim=dim, vdim=vdim, scale=scale, **more), cache="e2m1")


CONFIG = util.config(131, 64, 1e-5, 3.0, [
    util.layer(packed(window=1000, rot=32, softcap=8.0)), util.layer(util.lightning([0.9, 0.97], dim=32, vdim=16), experts=0),
    util.layer(packed(heads=6, kv_heads=1, dim=64, vdim=128, window=40, rot=16), experts=5, top=2, ff=24),
    util.layer(util.attention(dim=32, vdim=64, window=90, rot=32, kv_from=0, scale=0.2), experts=0), util.layer(util.attention(window=30), experts=0)])


def weights(c, seed=0):
    return util.weights(c, seed)


plain_mixer = ref.attention_mixer


def stored(x, round_to=lambda a: np.asarray(a, np.float32)):
    """What a pool gives back of x [T, heads, n] that a module of a type stores."""
    one = np.ones(x.shape[1], np.float32)
    return packed_util.valued(*packed_util.packed(round_to(x.astype(np.float32)), one), one)


def mixer(h, w, c, eps, shared=None, round_to=lambda a: np.asarray(a, np.float32)):
    """As kipizen_ref.attention_mixer; keys and values go through 4 bits where they are the layer's own."""
    if not c.get("cache"):
        return plain_mixer(h, w, c, eps, shared)
    T, H, G, d = h.shape[0], c["heads"], c["kv_heads"], c["dim"]
    rot = c["rot"]

    def place(x):
        return ref.unit_rms(ref.rotate(x, rot["base"], rot["dims"], rot["scaling"]["factor"]), eps)

    q = place((h @ w["q"].T + w["q.b"]).reshape(T, H, d))
    k = stored(place((h @ w["k"].T + w["k.b"]).reshape(T, G, d)), round_to)
    v = stored((h @ w["v"].T + w["v.b"]).reshape(T, G, c["vdim"]), round_to)
    o = ref.attention(q, k, v, c["scale"], c["softcap"], c["mask"]["size"])
    return o.reshape(T, -1) @ w["o"].T, (k, v)
