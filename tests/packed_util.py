"""Keys and values in 4 bits written out in 64 bits, batch steps over their paged pools, and modules of the composites that write, read and attend to them."""
import dataclasses
import math

import numpy as np

from kipizen_util import to_bf16
from onyxia_b200 import ir
from onyxia_b200.ir import HostTensor
from onyxia_b200.kipizen import turns_per_position

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


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
    scale: float = 0.0
    eps: float = 1e-5
    factors: int = 0
    gap: int = 0          # columns of the projection between and behind its parts
    shared: bool = False  # nothing is appended

    def __post_init__(self):
        self.scale = self.scale or self.dim ** -0.5

    @property
    def offsets(self):
        q, k = self.heads * self.dim, self.kv_heads * self.dim
        return self.gap, q + 2 * self.gap, q + k + 3 * self.gap

    @property
    def width(self):
        return self.offsets[2] + self.kv_heads * self.vdim + self.gap

    def factor_pair(self):
        if not self.factors:
            return [np.ones(self.kv_heads, np.float32)] * 2
        r = np.random.default_rng(99)
        return [np.exp(r.uniform(-1.5, 1.5, self.kv_heads)).astype(np.float32) for _ in range(2)]


# ── the format ──
def scale_values(codes):
    """What e4m3 codes stand for."""
    e, m = codes.astype(np.int64) >> 3 & 15, codes.astype(np.int64) & 7
    v = np.where(e == 0, np.ldexp(m.astype(np.float64), -9), np.ldexp(8.0 + m, e - 10))
    return np.where((codes & 127) == 127, np.nan, v) * np.where(codes & 128, -1.0, 1.0)


SCALES = scale_values(np.arange(127))  # rising


def nearest(x, values):
    """Index of the value next to each x ≥ 0, of two that are as near the even one; the last one for what is beyond."""
    i = np.clip(np.searchsorted(values, x), 1, len(values) - 1)
    low, high = values[i - 1], values[i]
    i = np.where((x - low < high - x) | ((x - low == high - x) & (i % 2 == 1)), i - 1, i)
    return i


def packed(x, factor):
    """(codes, scales) of x [..., kv_heads, n], one value each; factor [kv_heads]. Quotients by the factor and by 6 are rounded to f32."""
    x = np.asarray(x, np.float32)
    y = (x / np.asarray(factor, np.float32)[:, None]).reshape(*x.shape[:-1], x.shape[-1] // 16, 16)
    bad = np.isnan(y).any(-1)
    y = np.where(bad[..., None], 0.0, y).astype(np.float64)
    top = (np.abs(y).max(-1).astype(np.float32) / np.float32(6.0)).astype(np.float64)
    scales = nearest(np.minimum(top, 448.0), SCALES)
    s = SCALES[scales][..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        r = np.where(s > 0, np.abs(y) / s, 0.0)
    codes = nearest(np.minimum(r, 6.0), MAGNITUDES)
    codes += np.where((y < 0) & (codes > 0), 8, 0)  # 0 has no sign
    return codes.reshape(x.shape).astype(np.uint8), np.where(bad, 127, scales).astype(np.uint8)


def valued(codes, scales, factor):
    v = MAGNITUDES[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    v = v.reshape(*scales.shape, 16) * scale_values(scales)[..., None]
    return v.reshape(codes.shape) * np.asarray(factor, np.float64)[:, None]


def bytes_of(codes, scales):
    """Pools [pages, kv_heads, page, n · 9 / 16] from codes [pages, kv_heads, page, n] and scales [pages, kv_heads, page, n / 16]."""
    pages, kv, page, n = codes.shape
    both = codes[..., 0::2] | codes[..., 1::2] << 4
    return np.concatenate([both.reshape(pages, kv, -1), scales.reshape(pages, kv, -1)], -1).reshape(pages, kv, page, n * 9 // 16).astype(np.uint8)


def parts_of(pool):
    """Codes and scales of a pool of bytes."""
    pages, kv, page, w = pool.shape
    n = w * 16 // 9
    flat = pool.reshape(pages, kv, -1)
    both = flat[..., :page * n // 2].reshape(pages, kv, page, n // 2)
    return np.stack([both & 15, both >> 4], -1).reshape(pages, kv, page, n), flat[..., page * n // 2:].reshape(pages, kv, page, n // 16)


# ── modules ──
def module(f: Form, dtype, kind="attend", **changed):
    """`kind`: "attend", "shared", "write", "read", or "chain": keys and values are written, attended to by another node, and read back. `changed`: attributes, or shapes and types of
    operands by name, that are not what they should be."""
    b = ir.GraphBuilder()
    N, R, NP, TW, M = b.sym("num_tokens"), b.sym("num_seqs"), b.sym("num_pages"), b.sym("table_width"), b.sym("num_places")
    given = lambda name, dt, dims: b.input(name, *changed.get(name, (dt, dims)))  # noqa: E731
    shapes = [changed.get(name, (ir.U8, [NP, f.kv_heads, f.page, n // 16 * 9])) for name, n in (("pages.keys", f.dim), ("pages.values", f.vdim))]
    pools = [b.input(name, *s) for name, s in zip(("pages.keys", "pages.values"), shapes)]
    table = given("page_table", ir.I32, [R, TW])
    q, k, v = f.offsets
    sizes = {"kv_heads": f.kv_heads, "dim": f.dim, "vdim": f.vdim, "factors": f.factors}
    attrs = dict(sizes, heads=f.heads, q_offset=q, k_offset=k, v_offset=v, rot_dims=f.rot_dims, window=f.window, scale=float(f.scale), softcap=float(f.softcap), norm=f.norm, epsilon=f.eps,
                 sink=f.sink)
    for a in (sizes, attrs):
        a.update({n: x for n, x in changed.items() if n in a})
    const = lambda a: b.constant(HostTensor.from_numpy(np.ascontiguousarray(a, np.float32)))  # noqa: E731
    factors = [const(x) for x in changed.get("factor_values", f.factor_pair() if f.factors else [])]
    cut = slice(0, changed.get("operands"))
    out, stored = changed.get("out", (dtype, [N, f.heads * f.vdim])), changed.get("out", (dtype, [M, f.kv_heads * (f.dim + f.vdim)]))
    b.set_loc("mix", "packed")
    if kind != "read":
        ins = [given("proj", dtype, [N, f.width]), const(changed.get("turns", turns_per_position(f.rot_dims, 10000.0, 1.0))), *pools, given("seq_info", ir.I32, [R, 4]), table, *factors][cut]
        updated = [changed.get("updated", s) for s in shapes]
        if kind == "attend":
            o, *pools = b.composite("onyxia.PackedKVAttention", attrs, ins, [out, *updated])
        if kind in ("write", "chain"):
            pools = b.composite("onyxia.CacheWrite", {n: x for n, x in attrs.items() if n not in ("heads", "q_offset", "window", "scale", "softcap", "sink")}, ins, updated)
            ins[2:4] = pools
        if kind in ("shared", "chain"):
            o = b.composite("onyxia.SharedPackedKVAttention", attrs, ins, [out])[0]
        if kind != "write":
            b.output("out", o)
    if kind in ("read", "chain"):
        b.output("stored", b.composite("onyxia.CacheRead", sizes, [*pools, given("places", ir.I32, [M, 2]), table, *factors][cut], [stored])[0])
    if kind not in ("read", "shared"):
        for name, x in zip(("updated.pages.keys", "updated.pages.values"), pools):
            b.output(name, x)
    return b.finish()


# ── batch steps ──
@dataclasses.dataclass
class Step:
    proj: np.ndarray
    keys: np.ndarray    # pools of bytes
    values: np.ndarray
    seqs: np.ndarray
    table: np.ndarray


def step(f: Form, lengths, seed=0, spare=2, tail=0, spread=1.5, round_to=to_bf16, size=1.0):
    """`lengths`: (new, past) of every sequence; `tail`: rows behind the last one; `spare`: pages that nobody has. What no sequence has written is bytes of 0xFF: scales that are no numbers.
    Sequences of the shared form have their new tokens in the pools already."""
    r = np.random.default_rng(seed)
    held = [-(-(n + p) // f.page) for n, p in lengths]
    pages = sum(held) + spare
    order, width = r.permutation(pages).astype(np.int32), max(held + [1])
    table, seqs = np.full((len(lengths), width), -1, np.int32), np.zeros((len(lengths), 4), np.int32)
    parts = [[np.full((pages, f.kv_heads, f.page, n), 15, np.uint8), np.full((pages, f.kv_heads, f.page, n // 16), 255, np.uint8)] for n in (f.dim, f.vdim)]
    at = row = 0
    for i, (n, past) in enumerate(lengths):
        table[i, :held[i]] = order[at:at + held[i]]
        seqs[i] = row, n, past, i
        j = np.arange(past + (n if f.shared else 0))
        for part, d, factor in zip(parts, (f.dim, f.vdim), f.factor_pair()):
            codes, scales = packed(size * r.standard_normal((len(j), f.kv_heads, d)), factor)
            part[0][table[i, j // f.page], :, j % f.page] = codes
            part[1][table[i, j // f.page], :, j % f.page] = scales
        at, row = at + held[i], row + n
    proj = size * r.standard_normal((row + tail, f.width)).astype(np.float32)
    q, k, _ = f.offsets
    proj[:, q:k] *= spread / size
    return Step(round_to(proj), bytes_of(*parts[0]), bytes_of(*parts[1]), seqs, table)


def feed(s: Step, act):
    return {"proj": act(s.proj), "pages.keys": HostTensor.from_numpy(s.keys), "pages.values": HostTensor.from_numpy(s.values), "seq_info": HostTensor.from_numpy(s.seqs),
            "page_table": HostTensor.from_numpy(s.table)}


def prepared(f, part, positions):
    """Queries or keys [tokens, heads, dim], rotated and normed in 64 bits."""
    part, half = part.astype(np.float64), f.rot_dims // 2
    if half:
        turns = turns_per_position(f.rot_dims, 10000.0, 1.0).astype(np.float64).sum(0)
        t = positions[:, None].astype(np.float64) * turns
        a = 2.0 * math.pi * (t - np.rint(t))
        cos, sin = np.cos(a)[:, None], np.sin(a)[:, None]
        u, v = part[..., :half].copy(), part[..., half:2 * half].copy()
        part[..., :half], part[..., half:2 * half] = u * cos - v * sin, v * cos + u * sin
    return part / np.sqrt((part ** 2).mean(-1, keepdims=True) + f.eps) if f.norm else part


def written(f: Form, s: Step, round_to=to_bf16):
    """The pools behind a step: bytes."""
    parts = [[x.copy() for x in parts_of(pool)] for pool in (s.keys, s.values)]
    _, k0, v0 = f.offsets
    for i, (row, n, past, _) in enumerate(s.seqs):
        new = np.arange(past, past + n)
        k = round_to(prepared(f, s.proj[row:row + n, k0:k0 + f.kv_heads * f.dim].reshape(n, f.kv_heads, f.dim), new).astype(np.float32))
        v = s.proj[row:row + n, v0:v0 + f.kv_heads * f.vdim].reshape(n, f.kv_heads, f.vdim)
        pg, off = s.table[i, new // f.page], new % f.page
        for part, x, factor in zip(parts, (k, v), f.factor_pair()):
            part[0][pg, :, off], part[1][pg, :, off] = packed(x, factor)
    return [bytes_of(*p) for p in parts]


def read(f: Form, pools, table, places):
    """What the pools hold at places, [places, kv_heads · (dim + vdim)] in 64 bits."""
    seq, pos = np.asarray(places).T
    pg, off = table[seq, pos // f.page], pos % f.page
    both = [valued(codes[pg, :, off], scales[pg, :, off], factor) for (codes, scales), factor in zip((parts_of(p) for p in pools), f.factor_pair())]
    return np.concatenate([x.reshape(len(pg), -1) for x in both], 1)


def reference(f: Form, s: Step, pools):
    """Results [rows, heads · vdim] in 64 bits over pools that hold the new keys and values. Rows of no sequence are NaN."""
    out = np.full((len(s.proj), f.heads, f.vdim), np.nan)
    q0 = f.offsets[0]
    for i, (row, n, past, _) in enumerate(s.seqs):
        if n == 0:
            continue
        q = prepared(f, s.proj[row:row + n, q0:q0 + f.heads * f.dim].reshape(n, f.heads, f.dim), np.arange(past, past + n))
        both = read(f, pools, s.table, [(i, j) for j in range(past + n)])
        keys, values = both[:, :f.kv_heads * f.dim].reshape(-1, f.kv_heads, f.dim), both[:, f.kv_heads * f.dim:].reshape(-1, f.kv_heads, f.vdim)
        at, j = np.arange(past, past + n)[:, None], np.arange(past + n)
        seen = (j <= at) & ((j > at - f.window) | (f.window == 0))
        for h in range(f.heads):
            g = h // (f.heads // f.kv_heads)
            z = q[:, h] @ keys[:, g].T * f.scale
            if f.softcap:
                z = f.softcap * np.tanh(z / f.softcap)
            z = np.where(seen, z, -np.inf)
            top = np.maximum(z.max(1), 0.0) if f.sink else z.max(1)
            e = np.where(seen, np.exp(z - top[:, None]), 0.0)
            out[row:row + n, h] = np.where(seen, e, 0.0) @ values[:, g] / (e.sum(1) + (np.exp(-top) if f.sink else 0.0))[:, None]
    return out.reshape(len(s.proj), -1)
