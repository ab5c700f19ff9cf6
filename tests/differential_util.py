"""Differential attention written out in 64 bits, batch steps over paged pools, and the module of the one composite."""
import dataclasses
import math

import numpy as np

from kipizen_util import to_bf16
from onyxia_b200 import ir
from onyxia_b200.ir import HostTensor
from onyxia_b200.kipizen import turns_per_position


@dataclasses.dataclass
class Form:
    heads: int
    kv_heads: int
    dim: int
    vdim: int
    rot_dims: int = 0
    page: int = 64
    window: int = 0
    softcap: float = 0.0
    norm: int = 0
    sink: int = 0
    head_norm: int = 1
    scale: float = 0.0
    eps: float = 1e-5
    head_eps: float = 1e-5
    gap: int = 0          # columns of the projection between and behind its parts

    def __post_init__(self):
        self.scale = self.scale or self.dim ** -0.5

    @property
    def offsets(self):
        q, k = self.heads * 2 * self.dim, self.kv_heads * 2 * self.dim
        return self.gap, q + 2 * self.gap, q + k + 3 * self.gap

    @property
    def width(self):
        return self.offsets[2] + self.kv_heads * self.vdim + self.gap


def module(f: Form, dtype, lam, gain, **changed):
    """`changed`: attributes, or shapes and types of operands by name, that are not what they should be."""
    b = ir.GraphBuilder()
    N, R, NP, TW = b.sym("num_tokens"), b.sym("num_seqs"), b.sym("num_pages"), b.sym("table_width")
    shape = lambda name, dt, dims: changed.get(name, (dt, dims))  # noqa: E731
    ins = {name: b.input(name, *shape(name, dt, dims)) for name, dt, dims in (
        ("proj", dtype, [N, f.width]), ("pages.keys", dtype, [NP, f.kv_heads, f.page, 2 * f.dim]), ("pages.values", dtype, [NP, f.kv_heads, f.page, f.vdim]),
        ("seq_info", ir.I32, [R, 4]), ("page_table", ir.I32, [R, TW]))}
    q, k, v = f.offsets
    attrs = {"heads": f.heads, "kv_heads": f.kv_heads, "dim": f.dim, "vdim": f.vdim, "q_offset": q, "k_offset": k, "v_offset": v, "rot_dims": f.rot_dims, "window": f.window,
             "scale": float(f.scale), "softcap": float(f.softcap), "norm": f.norm, "epsilon": f.eps, "sink": f.sink, "head_norm": f.head_norm, "head_epsilon": f.head_eps}
    attrs.update({k: v for k, v in changed.items() if k in attrs})
    const = lambda a: b.constant(HostTensor.from_numpy(np.ascontiguousarray(a, np.float32)))  # noqa: E731
    operands = [ins["proj"], const(changed.get("turns", turns_per_position(f.rot_dims, 10000.0, 1.0))), ins["pages.keys"], ins["pages.values"], ins["seq_info"], ins["page_table"], const(lam)]
    operands += [const(gain)] if f.head_norm else []
    b.set_loc("mix", "DifferentialAttention")
    outs = b.composite("onyxia.DifferentialAttention", attrs, operands[:changed.get("operands", 8)], [
        changed.get("out", (dtype, [N, f.heads * f.vdim])), (changed.get("pages.keys", (dtype,))[0], changed.get("pages.keys", (0, [NP, f.kv_heads, f.page, 2 * f.dim]))[1]),
        (changed.get("pages.values", (dtype,))[0], changed.get("pages.values", (0, [NP, f.kv_heads, f.page, f.vdim]))[1])])
    for name, v in zip(("out", "updated.pages.keys", "updated.pages.values"), outs):
        b.output(name, v)
    return b.finish()


@dataclasses.dataclass
class Step:
    proj: np.ndarray
    keys: np.ndarray
    values: np.ndarray
    seqs: np.ndarray
    table: np.ndarray
    lam: np.ndarray
    gain: np.ndarray


def step(f: Form, lengths, seed=0, spare=2, tail=0, spread=1.5, round_to=to_bf16):
    """`lengths`: (new, past) of every sequence; `tail`: rows behind the last one; `spare`: pages that nobody has. What no sequence has written is NaN."""
    r = np.random.default_rng(seed)
    held = [-(-(n + p) // f.page) for n, p in lengths]
    pages = sum(held) + spare
    order, width = r.permutation(pages).astype(np.int32), max(held + [1])
    table, seqs = np.full((len(lengths), width), -1, np.int32), np.zeros((len(lengths), 4), np.int32)
    keys, values = np.full((pages, f.kv_heads, f.page, 2 * f.dim), np.nan, np.float32), np.full((pages, f.kv_heads, f.page, f.vdim), np.nan, np.float32)
    at = row = 0
    for i, (n, past) in enumerate(lengths):
        table[i, :held[i]] = order[at:at + held[i]]
        seqs[i] = row, n, past, i
        for j in range(past):
            pg, off = table[i, j // f.page], j % f.page
            keys[pg, :, off] = round_to(r.standard_normal((f.kv_heads, 2 * f.dim)))
            values[pg, :, off] = round_to(r.standard_normal((f.kv_heads, f.vdim)))
        at, row = at + held[i], row + n
    proj = r.standard_normal((row + tail, f.width)).astype(np.float32)
    q, k, _ = f.offsets
    proj[:, q:k] *= spread
    return Step(round_to(proj), keys, values, seqs, table, (0.2 + 0.6 * r.random(f.heads)).astype(np.float32), (0.2 + 0.02 * r.standard_normal(f.vdim)).astype(np.float32))


def feed(s: Step, act):
    return {"proj": act(s.proj), "pages.keys": act(s.keys), "pages.values": act(s.values), "seq_info": HostTensor.from_numpy(s.seqs), "page_table": HostTensor.from_numpy(s.table)}


def reference(f: Form, s: Step, stored=to_bf16):
    """(results [rows, heads · vdim], keys, values) in 64 bits; new keys are rounded by `stored` when they go to the pool. Rows of no sequence are NaN."""
    x, keys, values = s.proj.astype(np.float64), s.keys.astype(np.float64), s.values.astype(np.float64)
    turns = turns_per_position(f.rot_dims, 10000.0, 1.0).astype(np.float64).sum(0)
    out = np.full((len(x), f.heads, f.vdim), np.nan)
    q0, k0, v0 = f.offsets
    half = f.rot_dims // 2

    def prepared(part, positions):
        part = part.copy()
        if half:
            a = 2.0 * math.pi * positions[:, None] * turns
            cos, sin = np.cos(a)[:, None, None], np.sin(a)[:, None, None]
            u, v = part[..., :half].copy(), part[..., half:2 * half].copy()
            part[..., :half], part[..., half:2 * half] = u * cos - v * sin, v * cos + u * sin
        return part / np.sqrt((part ** 2).mean(-1, keepdims=True) + f.eps) if f.norm else part

    for i, (row, n, past, _) in enumerate(s.seqs):
        if n == 0:
            continue
        mine, new = x[row:row + n], np.arange(past, past + n)
        q = prepared(mine[:, q0:q0 + f.heads * 2 * f.dim].reshape(n, f.heads, 2, f.dim), new.astype(np.float64))
        k = prepared(mine[:, k0:k0 + f.kv_heads * 2 * f.dim].reshape(n, f.kv_heads, 2, f.dim), new.astype(np.float64))
        pg, off = s.table[i, new // f.page], new % f.page
        keys[pg, :, off] = stored(k).astype(np.float64).reshape(n, f.kv_heads, -1)
        values[pg, :, off] = mine[:, v0:v0 + f.kv_heads * f.vdim].reshape(n, f.kv_heads, f.vdim)
        for t, pos in enumerate(new):
            seen = np.arange(max(0, pos - f.window + 1) if f.window else 0, pos + 1)
            pg, off = s.table[i, seen // f.page], seen % f.page
            for h in range(f.heads):
                g, w = h // (f.heads // f.kv_heads), []
                for m in (0, 1):
                    z = keys[pg, g, off, m * f.dim:(m + 1) * f.dim] @ q[t, h, m] * f.scale
                    if f.softcap:
                        z = f.softcap * np.tanh(z / f.softcap)
                    top = max(z.max(), 0.0) if f.sink else z.max()
                    e = np.exp(z - top)
                    w.append(e / (e.sum() + (np.exp(-top) if f.sink else 0.0)))
                o = (w[0] - float(s.lam[h]) * w[1]) @ values[pg, g, off]
                out[row + t, h] = o / np.sqrt((o ** 2).mean() + f.head_eps) * s.gain if f.head_norm else o
    return out.reshape(len(x), -1), keys, values
