"""A small Kipizen configuration with differential layers, and the mixer's plain form for kipizen_ref.py."""
import numpy as np

import kipizen_ref as ref
import kipizen_util as util


def differential(heads=4, kv_heads=2, dim=32, vdim=64, lambda_init=0.6, **more):
    m = util.attention(heads=heads, kv_heads=kv_heads, dim=dim, vdim=vdim, **more)
    m["differential"] = {"lambda_init": lambda_init}
    return m


CONFIG = util.config(131, 64, 1e-5, 3.0, [
    util.layer(differential(window=1000, rot=32, softcap=8.0)), util.layer(util.lightning([0.9, 0.97], dim=32, vdim=16), experts=0),
    util.layer(differential(heads=6, kv_heads=1, dim=64, vdim=128, window=40, rot=16, lambda_init=0.3), experts=5, top=2, ff=24),
    util.layer(util.attention(window=30), experts=0)])


def weights(c, seed=0):
    """kipizen_util's tensors; those of differential layers in their sizes, and their own."""
    r, out = np.random.default_rng(seed + 100), util.weights(c, seed)
    for i, l in enumerate(c["layers"]):
        m, p = l["mixer"], f"l{i}.mix."
        if not m.get("differential"):
            continue
        for n, heads in (("q", m["heads"]), ("k", m["kv_heads"])):
            out[p + n] = util.to_bf16(r.standard_normal((2 * heads * m["dim"], c["width"])) / np.sqrt(c["width"]))
            out[p + n + ".b"] = util.to_bf16(0.5 * r.standard_normal(2 * heads * m["dim"]))
        out.update({p + "lam." + n: util.to_bf16(0.1 * r.standard_normal(m["dim"])) for n in ("q1", "k1", "q2", "k2")})
        out[p + "head_norm"] = util.to_bf16(1 + 0.2 * r.standard_normal(m["vdim"]))
    return out


plain_mixer = ref.attention_mixer


def mixer(h, w, c, eps, shared=None):
    if not c.get("differential"):
        return plain_mixer(h, w, c, eps, shared)
    T, H, G, d = h.shape[0], c["heads"], c["kv_heads"], c["dim"]
    rot, first = c["rot"], c["differential"]["lambda_init"]

    def place(x):
        return ref.unit_rms(ref.rotate(x, rot["base"], rot["dims"], rot["scaling"]["factor"]), eps)

    q = place((h @ w["q"].T + w["q.b"]).reshape(T, 2 * H, d)).reshape(T, H, 2, d)
    k = place((h @ w["k"].T + w["k.b"]).reshape(T, 2 * G, d)).reshape(T, G, 2, d)
    v = (h @ w["v"].T + w["v.b"]).reshape(T, G, c["vdim"])
    lam = np.exp(w["lam.q1"] @ w["lam.k1"]) - np.exp(w["lam.q2"] @ w["lam.k2"]) + first
    a, b = (ref.attention(q[:, :, m], k[:, :, m], v, c["scale"], c["softcap"], c["mask"]["size"]) for m in (0, 1))
    o = ref.unit_rms(a - lam * b, eps) * w["head_norm"] * (1 - first)
    return o.reshape(T, -1) @ w["o"].T, None
