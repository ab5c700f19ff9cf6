"""Performance cases of single operators: keys and values held in 4 bits, written, read back, and attended to by prompts and by single tokens.

  attention  `onyxia.PackedKVAttention`: the batch's new keys and values go to the pools, its queries attend to what these hold; `onyxia.CacheRead` gives back what was stored
  cache      `onyxia.CacheWrite` of a batch's keys and values, and `onyxia.CacheRead` of them
  read       `onyxia.CacheRead` of tokens that were stored before

All of them are prepared as modules of these nodes and run by `CudaSession.run` on tensors of the device. Where `own` is false, `run` computes the same in elementary torch operations, in 32 bits;
rotations, norms and what is next to a border between two codes in 64.

A pool [pages, kv_heads, page, dim · 9 / 16] of bytes holds of every page and head first the codes (e2m1, two in a byte, the earlier one in the low half), then a scale (e4m3) per 16 dimensions;
a value is code · scale · the head's factor. Widths are those of the three sizes that the whole-pass cases use (1b, 4b, 27b).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

EPS, BLOCK = 1e-6, 16
# heads, kv_heads, dimensions of a key, of a value
SIZES = {"1b": (4, 1, 256, 256), "4b": (16, 4, 128, 128), "27b": (32, 16, 128, 128)}


# ── the cases ──
def _attention(size, seqs, new, past, *, ragged=False, dtype="bf16", page=64, window=0, softcap=0.0, norm=False, sink=False, factors=False):
    heads, kv, dim, vdim = SIZES[size] if isinstance(size, str) else size
    return {"kind": "attention", "heads": heads, "kv_heads": kv, "dim": dim, "vdim": vdim, "seqs": seqs, "new": new, "past": past, "ragged": ragged, "dtype": dtype,
            "page": page, "window": window, "softcap": softcap, "norm": norm, "sink": sink, "factors": factors}


def _cache(kind, size, seqs, new, past, *, ragged=False, dtype="bf16", page=64, norm=False, factors=False):
    return dict(_attention(size, seqs, new, past, ragged=ragged, dtype=dtype, page=page, norm=norm, factors=factors), kind=kind)


def listed():
    cases = {
        # a few short questions of one batch step, none longer than a page
        "prompt_1b_short": _attention("1b", 6, 47, 0, ragged=True),
        # an odd portion of a prompt whose first thousand tokens are cached; capped scores, normed queries and keys, a sink
        "prompt_4b_1999": _attention("4b", 1, 1999, 1000, softcap=30.0, norm=True, sink=True),
        # the longest prompt, at the widest size
        "prompt_27b_4096": _attention("27b", 1, 4096, 0),
        # 32-bit arithmetic, short ragged requests
        "prompt_f32": _attention((4, 2, 32, 64), 3, 101, 20, ragged=True, dtype="f32"),
        # a single user who waits for every token
        "token_1b_single": _attention("1b", 1, 1, 519),
        # a full serving batch behind contexts of different lengths
        "token_4b_batch64": _attention("4b", 64, 1, 8192, ragged=True),
        # few users behind long documents, factors from a calibration
        "token_27b_long": _attention("27b", 4, 1, 32768, sink=True, factors=True),
        # the largest: every sequence sees 8192 keys of every head
        "token_27b_batch64": _attention("27b", 64, 1, 8191),
        # the cache of a prompt whose attention ran elsewhere
        "cache_27b_4096": _cache("cache", "27b", 1, 4096, 0),
        # a few tokens of short requests in 32 bits, odd sizes
        "cache_f32": _cache("cache", (6, 3, 48, 80), 5, 29, 11, ragged=True, dtype="f32", page=16, factors=True),
        # a long document's keys and values, to go on with in another layout
        "read_27b_32768": _cache("read", "27b", 1, 32768, 0),
        # the last page of a sequence
        "read_1b_page": _cache("read", "1b", 1, 64, 512),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _spread(rng, low, high):
    """A whole number from low to high, its logarithm spread evenly."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49))))))


def draw(rng):
    kind = rng.choice(("prompt", "prompt", "prompt", "token", "token", "token", "cache", "read"))
    more = {"ragged": rng.random() < 0.7, "page": rng.choice((16, 32, 64, 64, 128)), "norm": rng.random() < 0.3, "factors": rng.random() < 0.3}
    dims = (32, 48, 64, 64, 80, 96, 128, 128, 256)
    dim, kv = rng.choice(dims), rng.choice((1, 2, 3, 4, 8))
    size = rng.choice(("1b", "4b", "27b", (kv * rng.randint(1, 9), kv, dim, rng.choice((dim, rng.choice(dims))))))
    if kind in ("cache", "read"):
        seqs = _spread(rng, 1, 16)
        return _cache(kind, size, seqs, _spread(rng, 1, 8192 // seqs), rng.choice((0, _spread(rng, 1, 2000))) // seqs, dtype=rng.choice(("bf16", "bf16", "f32")), **more)
    more |= {"sink": rng.random() < 0.3, "softcap": rng.choice((0.0, 0.0, 30.0)), "window": rng.choice((0, 0, _spread(rng, 64, 4096)))}
    if rng.random() < 0.15:
        dim = rng.choice((16, 32, 48, 64))
        return _attention((kv * rng.randint(1, 3), kv, dim, 2 * dim), _spread(rng, 1, 4), rng.choice((1, _spread(rng, 2, 150))), _spread(rng, 1, 200), dtype="f32", **more)
    if kind == "token":
        seqs = _spread(rng, 1, 64)
        return _attention(size, seqs, 1, _spread(rng, 1, min(32768, 262144 // seqs)), **more)
    seqs = _spread(rng, 1, 16)
    return _attention(size, seqs, _spread(rng, 2, 4096 // seqs), rng.choice((0, _spread(rng, 1, 2000))) // seqs, **more)


# ── the sequences of a case ──
def _lengths(case):
    """(new, past) of every sequence."""
    new, past = case["new"], case["past"]
    if not case["ragged"]:
        return [(new, past)] * case["seqs"]
    return [(max(1, new - (i * 37) % (new // 2 + 1)), past - (i * 53) % (past // 2 + 1)) for i in range(case["seqs"])]


def _seen(case):
    """How many keys each new row sees, added over the rows; how many keys each sequence reads, added over the sequences; rows."""
    pairs = keys = rows = 0
    for new, past in _lengths(case):
        w = case["window"] or past + new
        pairs += sum(min(w, past + i + 1) for i in range(new))
        keys += min(past + new, w + new - 1)
        rows += new
    return pairs, keys, rows


def work(case):
    pairs, keys, rows = _seen(case)
    heads, kv, dim, vdim, size = case["heads"], case["kv_heads"], case["dim"], case["vdim"], 2 if case["dtype"] == "bf16" else 4
    per_key = kv * (dim + vdim)
    held = per_key * 9 // 16
    if case["kind"] == "read":
        return {"bytes": rows * (held + per_key * size), "flops": rows * per_key}
    if case["kind"] == "cache":  # in, stored, out
        return {"bytes": rows * (2 * per_key * size + held), "flops": rows * per_key}
    moved = rows * (heads * dim + per_key) + rows * heads * vdim + rows * per_key  # projections in, results and what was stored out
    return {"bytes": moved * size + keys * held, "flops": pairs * heads * 2 * (dim + vdim)}


# ── inputs ──
def _turns(dim):
    """[2, dim / 2] f32: turns per position of each pair of dimensions, as the sum of two f32."""
    turns = np.array([10000.0 ** (-2.0 * i / dim) / (2.0 * math.pi) for i in range(dim // 2)])
    high = turns.astype(np.float32)
    return np.stack([high, (turns - high).astype(np.float32)])


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    heads, kv, dim, vdim, page = case["heads"], case["kv_heads"], case["dim"], case["vdim"], case["page"]
    lengths = _lengths(case)
    rows = sum(n for n, _ in lengths)
    held = [-(-(n + past) // page) for n, past in lengths]
    pages, width = sum(held), max(held)
    host = np.random.default_rng(seed)
    order, table, at, row = host.permutation(pages).astype(np.int32), np.zeros((len(lengths), width), np.int32), 0, 0
    seqs, places = np.zeros((len(lengths), 4), np.int32), []
    for i, (n, past) in enumerate(lengths):
        table[i, :held[i]] = order[at:at + held[i]]
        seqs[i] = row, n, past, i
        places += [(i, past + t) for t in range(n)]
        at, row = at + held[i], row + n
    state = {"case": case, "turns": torch.from_numpy(_turns(dim)).cuda(), "seqs": torch.from_numpy(seqs).cuda(), "table": torch.from_numpy(table).cuda(),
             "rows": torch.from_numpy(np.array(places, np.int32)).cuda()}
    # some dimensions of a key are larger than others for every token
    sizes = torch.exp(0.5 * randn(kv, dim))
    if case["kind"] != "read":
        # queries of a spread that lets some keys stand out
        q = 1.5 * randn(rows, heads * dim) if case["kind"] == "attention" else randn(rows, 0)
        state["proj"] = torch.cat([q, (randn(rows, kv, dim) * sizes).reshape(rows, -1), randn(rows, kv * vdim)], 1).to(dtype)
    if case["factors"]:
        state["factors"] = [0.5 + torch.rand(kv, generator=gen, device="cuda") for _ in range(2)]
    for name, d, by in (("keys", dim, sizes), ("values", vdim, 1.0)):
        pool = torch.empty(pages, kv, page, d * 9 // 16, dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 27) // (kv * page * d))
        for p in range(0, pages, step):
            x = randn(min(step, pages - p), kv, page, d) * (by[:, None] if name == "keys" else by)
            for part, to in zip(_packed(x), _parts(pool[p:p + step], d)):
                to.copy_(part)
        state[name] = pool
    if own:
        _own_handles(state)
    return state


# ── the framework's calls ──
def _own_handles(state):
    """The session, and what a program has on the device between steps."""
    from onyxia_b200 import ir
    from onyxia_b200.backend import CudaBackend

    case = state["case"]
    b = ir.GraphBuilder()
    dtype = ir.BF16 if case["dtype"] == "bf16" else ir.F32
    heads, kv, dim, vdim, page = case["heads"], case["kv_heads"], case["dim"], case["vdim"], case["page"]
    N, R, NP, TW = b.sym("num_tokens"), b.sym("num_seqs"), b.sym("num_pages"), b.sym("table_width")
    const = lambda x: b.constant(ir.HostTensor.from_numpy(x.cpu().numpy()))  # noqa: E731
    shapes = [(ir.U8, [NP, kv, page, d * 9 // 16]) for d in (dim, vdim)]
    pools = [b.input("pages." + name, *t) for name, t in zip(("keys", "values"), shapes)]
    rows, table = b.input("rows", ir.I32, [N, 2]), b.input("page_table", ir.I32, [R, TW])
    factors = [const(f) for f in state.get("factors", ())]
    sizes = {"kv_heads": kv, "dim": dim, "vdim": vdim, "factors": int(bool(factors))}
    named = {"pages.keys": "keys", "pages.values": "values", "rows": "rows", "page_table": "table"}
    if case["kind"] != "read":
        q = heads * dim if case["kind"] == "attention" else 0
        proj, seqs = b.input("proj", dtype, [N, q + kv * (dim + vdim)]), b.input("seq_info", ir.I32, [R, 4])
        named |= {"proj": "proj", "seq_info": "seqs"}
        attrs = dict(sizes, k_offset=q, v_offset=q + kv * dim, rot_dims=dim, norm=int(case["norm"]), epsilon=EPS)
        ins = [proj, const(state["turns"]), *pools, seqs, table, *factors]
        if case["kind"] == "attention":
            attrs |= {"heads": heads, "q_offset": 0, "scale": dim ** -0.5, "window": case["window"], "softcap": float(case["softcap"]), "sink": int(case["sink"])}
            out, *pools = b.composite("onyxia.PackedKVAttention", attrs, ins, [(dtype, [N, heads * vdim]), *shapes])
            b.output("out", out)
        else:
            pools = b.composite("onyxia.CacheWrite", attrs, ins, shapes)
    b.output("stored", b.composite("onyxia.CacheRead", sizes, [*pools, rows, table, *factors], [(dtype, [N, kv * (dim + vdim)])])[0])
    if case["kind"] != "read":
        for name, pool in zip(("keys", "values"), pools):
            b.output("updated.pages." + name, pool)
    session = CudaBackend((0,)).prepare(b.finish())
    state["session"] = session
    kinds = {torch.float32: ir.F32, torch.bfloat16: ir.BF16, torch.int32: ir.I32, torch.uint8: ir.U8}
    state["feed"] = [(name, session.upload_device(kinds[x.dtype], tuple(x.shape), x.data_ptr(), torch.cuda.current_stream().cuda_stream))
                     for name, x in ((name, state[key]) for name, key in named.items())]


def _view(session, t):
    """A tensor of the session as torch sees it: the same memory."""
    from onyxia_b200 import ir

    x = torch.as_tensor(session.view(t, torch.cuda.current_stream().cuda_stream), device="cuda")
    return x.view(torch.bfloat16) if t.dtype == ir.BF16 else x


def run(state):
    if own:
        return {name: _view(state["session"], t) for name, t in state["session"].run(state["feed"]) if name in ("out", "stored")}
    case = state["case"]
    found = {}
    if case["kind"] != "read":
        q = _plain_write(state)
        if case["kind"] == "attention":
            found["out"] = _plain_attention(state, q)
    return dict(found, stored=_plain_read(state))


# ── plain forms ──
def _parts(pool, dim):
    """The codes [pages, kv_heads, page, dim / 2] and the scales [..., dim / 16] of a pool: views."""
    pages, kv, page, _ = pool.shape
    flat = pool.view(pages, kv, -1)
    return flat[..., :page * dim // 2].unflatten(-1, (page, dim // 2)), flat[..., page * dim // 2:].unflatten(-1, (page, dim // BLOCK))


def _packed(x):
    """Codes and scales of x [..., dim] f32."""
    x = x.unflatten(-1, (-1, BLOCK))
    scale = (x.abs().amax(-1, keepdim=True) / 6.0).clamp_max_(448.0).to(torch.float8_e4m3fn)
    r = (x.abs() / scale.float()).nan_to_num_(0.0, 6.0)  # a block of zeros
    code = (r > 0.25).byte() + (r >= 0.75) + (r > 1.25) + (r >= 1.75) + (r > 2.5) + (r >= 3.5) + (r > 5.0)
    code = (code + 8 * (x < 0)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, scale.squeeze(-1).view(torch.uint8)


def _valued(codes, scales):
    """What codes [..., dim / 2] and scales [..., dim / 16] stand for, f32 [..., dim], without the factor."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device="cuda")
    table = torch.cat([table, -table])
    x = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], -1).flatten(-2)
    return (x.unflatten(-1, (-1, BLOCK)) * scales.view(torch.float8_e4m3fn).float()[..., None]).flatten(-2)


def _factors(state):
    return [f[:, None] for f in state.get("factors", ())] or [1.0, 1.0]


def _rotate(x, turns, pos):
    """x [rows, heads, dim] in 64 bits at positions pos [rows]: dimension i turns with i + dim / 2."""
    t = pos[:, None].double() * turns.double().sum(0)
    t = (t - t.round()) * (2.0 * math.pi)
    cos, sin = t.cos()[:, None], t.sin()[:, None]
    a, b = x.double().chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_write(s):
    """The new keys and values go to the pools; returns the rotated queries."""
    c = s["case"]
    kv, dim, vdim, page = c["kv_heads"], c["dim"], c["vdim"], c["page"]
    seq, pos = s["rows"].long().unbind(1)
    rows, heads = len(seq), c["heads"] if c["kind"] == "attention" else 0
    qk = _rotate(s["proj"][:, :(heads + kv) * dim].reshape(rows, -1, dim), s["turns"], pos)
    if c["norm"]:
        qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + EPS)
    pg, off = s["table"].long()[seq, pos // page], pos % page
    new = qk[:, heads:].to(s["proj"].dtype).float(), s["proj"][:, (heads + kv) * dim:].reshape(rows, kv, vdim).float()
    for name, x, f in zip(("keys", "values"), new, _factors(s)):
        for part, to in zip(_packed(x / f), _parts(s[name], x.shape[-1])):
            to[pg, :, off] = part
    return qk[:, :heads].float()


def _plain_read(s):
    c = s["case"]
    seq, pos = s["rows"].long().unbind(1)
    pg, off = s["table"].long()[seq, pos // c["page"]], pos % c["page"]
    parts = [(_valued(*(part[pg, :, off] for part in _parts(s[name], d))) * f).flatten(1) for name, d, f in zip(("keys", "values"), (c["dim"], c["vdim"]), _factors(s))]
    return torch.cat(parts, 1).to(torch.bfloat16 if c["dtype"] == "bf16" else torch.float32)


def _plain_attention(s, q):
    c = s["case"]
    heads, kv, dim, vdim = c["heads"], c["kv_heads"], c["dim"], c["vdim"]
    rep, start, count, past = heads // kv, s["seqs"][:, 0].long(), s["seqs"][:, 1].long(), s["seqs"][:, 2].long()
    seq, pos = s["rows"].long().unbind(1)
    place, rows = pos - past[seq], len(seq)
    # every sequence's keys and values one behind the other, its rows side by side
    longest, table = c["new"], s["table"].long()
    keys, values = ((_valued(*(part[table] for part in _parts(s[name], d))).transpose(2, 3) * f).reshape(len(count), -1, kv, d)
                    for name, d, f in zip(("keys", "values"), (dim, vdim), _factors(s)))
    queries = torch.zeros(len(count), longest, heads, dim, device="cuda")
    queries[seq, place] = q
    queries = queries.reshape(len(count), longest, kv, rep, dim).permute(0, 2, 3, 1, 4).reshape(len(count), kv, rep * longest, dim)
    scores = (queries @ keys.permute(0, 2, 3, 1)).mul_(dim ** -0.5)
    if c["softcap"]:
        scores = scores.div_(c["softcap"]).tanh_().mul_(c["softcap"])
    at, key = past[:, None] + torch.arange(longest, device="cuda"), torch.arange(keys.shape[1], device="cuda")
    hidden = key > at[..., None]
    if c["window"]:
        hidden |= key <= at[..., None] - c["window"]
    scores = scores.view(len(count), kv, rep, longest, -1).masked_fill_(hidden[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    if c["sink"]:
        top = top.clamp_min_(0.0)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    if c["sink"]:
        total = total + (-top).exp()
    out = weights.div_(total).view(len(count), kv, rep * longest, -1) @ values.transpose(1, 2)
    out = out.view(len(count), heads, longest, vdim)[seq, :, place]
    return out.reshape(rows, heads * vdim).to(s["proj"].dtype)


# ── the same from the definitions, in 64 bits ──
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["kind"] == "attention" and _seen(case)[0] * case["heads"] > 1e9:  # some seconds of 64-bit products
        return None
    kv, dim, vdim, page, dev = case["kv_heads"], case["dim"], case["vdim"], case["page"], "cuda"
    factors = [f.double() for f in s.get("factors", ())] or [torch.ones(kv, dtype=torch.float64, device=dev)] * 2
    magnitudes = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=dev)

    def fetched(name, d, pg, off, f):
        """[tokens, kv_heads, d]: what is stored at places of pages."""
        flat = s[name].view(s[name].shape[0], kv, -1)
        i, h = torch.arange(d, device=dev), torch.arange(kv, device=dev)
        byte = flat[pg[:, None, None], h[:, None], off[:, None, None] * (d // 2) + i // 2].long()
        code = torch.where(i % 2 == 1, byte >> 4, byte & 15)
        e = flat[pg[:, None, None], h[:, None], page * d // 2 + off[:, None, None] * (d // BLOCK) + i // BLOCK].long()
        scale = torch.where(e < 8, torch.ldexp((e % 8).double(), torch.tensor(-9, device=dev)), torch.ldexp(8.0 + (e % 8).double(), e // 8 - 10))
        return magnitudes[code % 8] * torch.where(code >= 8, -1.0, 1.0) * scale * f[:, None]

    def nearest(x, digits, least):
        """x rounded to so many binary digits, in steps of 2^least at least."""
        step = torch.ldexp(torch.ones_like(x), (torch.frexp(x)[1] - digits).clamp_min(least))
        return (x / step).round() * step

    def stored(x, f):
        """What 16 neighbours become."""
        y = (x / f[:, None]).unflatten(-1, (-1, BLOCK))
        scale = nearest(y.abs().amax(-1, keepdim=True) / 6.0, 4, -9).clamp_max(448.0)
        r = torch.where(scale > 0, y.abs() / scale, 0.0)
        return (nearest(r, 2, -1).clamp_max(6.0) * y.sign() * scale).flatten(-2) * f[:, None]

    proj = s["proj"].double() if "proj" in s else None
    heads = case["heads"] if case["kind"] == "attention" else 0
    turns, row, outs, back = s["turns"].double().sum(0), 0, [], []
    for i, (new, past) in enumerate(_lengths(case)):
        spots = torch.arange(past + new, device=dev)
        pg, off = s["table"][i].long()[spots // page], spots % page
        if case["kind"] == "read":
            back.append(torch.cat([fetched(n, d, pg[past:], off[past:], f).flatten(1) for n, d, f in zip(("keys", "values"), (dim, vdim), factors)], 1))
            continue
        angle = 2.0 * math.pi * spots[past:, None].double() * turns
        y = proj[row:row + new, :(heads + kv) * dim].reshape(new, -1, dim)
        z = torch.complex(y[..., :dim // 2], y[..., dim // 2:]) * torch.polar(torch.ones_like(angle), angle)[:, None]
        y = torch.cat([z.real, z.imag], -1)
        if case["norm"]:
            y = y / (y.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
        k, v = y[:, heads:].to(s["proj"].dtype).double(), proj[row:row + new, (heads + kv) * dim:].reshape(new, kv, vdim)
        k, v = stored(k, factors[0]), stored(v, factors[1])
        back.append(torch.cat([k.flatten(1), v.flatten(1)], 1))
        row += new
        if case["kind"] == "cache":
            continue
        k, v = torch.cat([fetched("keys", dim, pg[:past], off[:past], factors[0]), k]), torch.cat([fetched("values", vdim, pg[:past], off[:past], factors[1]), v])
        at = spots[past:, None]
        seen = (spots <= at) & (spots > at - case["window"]) if case["window"] else spots <= at
        out = torch.empty(new, heads, vdim, dtype=torch.float64, device=dev)
        for h in range(heads):
            g = h // (heads // kv)
            t = y[:, h] @ k[:, g].T / math.sqrt(dim)
            if case["softcap"]:
                t = case["softcap"] * torch.tanh(t / case["softcap"])
            t = t.masked_fill(~seen, -math.inf)
            if case["sink"]:
                t = torch.cat([t, torch.zeros(new, 1, dtype=torch.float64, device=dev)], 1)
            out[:, h] = torch.softmax(t, 1)[:, :past + new] @ v[:, g]
        outs.append(out.flatten(1))
    found = {"stored": torch.cat(back)}
    return dict(found, out=torch.cat(outs)) if outs else found
