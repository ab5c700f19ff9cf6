"""Performance cases of single operators: differential attention over paged keys and values, for prompts and for single tokens, and the rules
that a request puts on the logits of its next token.

  attention  `onyxia.DifferentialAttention`, prepared as a module of that one node and run by `CudaSession.run` on tensors of the device
  rules      `CudaSession.constrain_last` on logits of the device

Every attention case is one batch step: sequences with cached tokens behind them bring new ones, whose keys and values go to the pools.
Widths are those of the three sizes that the whole-pass cases use (1b, 4b, 27b): a head of 2 · dim there is a pair of maps of dim here.
Where `own` is false, `run` computes the same in elementary torch operations, in 32 bits.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

EPS, HEAD_EPS = 1e-6, 1e-5
# heads, kv_heads, dimensions of a map, of a value
SIZES = {"1b": (4, 1, 128, 256), "4b": (16, 4, 64, 128), "27b": (32, 16, 64, 128)}


# ── the cases ──
def _attention(size, seqs, new, past, *, ragged=False, dtype="bf16", page=64, window=0, softcap=0.0, norm=False, sink=False):
    heads, kv, dim, vdim = SIZES[size] if isinstance(size, str) else size
    return {"kind": "attention", "heads": heads, "kv_heads": kv, "dim": dim, "vdim": vdim, "seqs": seqs, "new": new, "past": past, "ragged": ragged, "dtype": dtype,
            "page": page, "window": window, "softcap": softcap, "norm": norm, "sink": sink}


def _rules(rows, vocab, history, *, dtype="f32", masks=0, biases=0):
    return {"kind": "rules", "rows": rows, "vocab": vocab, "history": history, "dtype": dtype, "masks": masks, "biases": biases}


def listed():
    cases = {
        # a few short questions of one batch step, none longer than a page
        "prompt_1b_short": _attention("1b", 6, 47, 0, ragged=True),
        # one ordinary prompt
        "prompt_4b_2048": _attention("4b", 1, 2048, 0),
        # an odd portion of a prompt whose first thousand tokens are cached; capped scores, normed queries and keys, a sink
        "prompt_1b_1999": _attention("1b", 1, 1999, 1000, softcap=30.0, norm=True, sink=True),
        # the longest prompt, at the widest size
        "prompt_27b_4096": _attention("27b", 1, 4096, 0),
        # 32-bit arithmetic, short ragged requests
        "prompt_f32": _attention((4, 2, 32, 64), 3, 101, 20, ragged=True, dtype="f32"),
        # a single user who waits for every token
        "token_1b_single": _attention("1b", 1, 1, 519),
        # a full serving batch behind contexts of different lengths
        "token_4b_batch64": _attention("4b", 64, 1, 2048, ragged=True),
        # few users behind long documents, of which a window is seen
        "token_27b_window": _attention("27b", 4, 1, 32768, window=4096),
        # the largest: every sequence sees 2048 keys of every head
        "token_27b_batch64": _attention("27b", 64, 1, 2047),
        # one row of the two-layer decoder's vocabulary: repetitions are penalised
        "rules_single": _rules(1, 32000, 16),
        # answers in a grammar: every row has a mask, half-precision logits
        "rules_grammar": _rules(8, 262144, 512, dtype="f16", masks=8),
        # a full serving batch at the largest vocabulary, all kinds of rules at once
        "rules_batch64": _rules(64, 262144, 2048, masks=16, biases=64),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _spread(rng, low, high):
    """A whole number from low to high, its logarithm spread evenly."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49))))))


def draw(rng):
    kind = rng.choice(("prompt", "prompt", "token", "token", "rules"))
    if kind == "rules":
        vocab = rng.choice((32000, 32768, 262144, _spread(rng, 1000, 262144)))
        return _rules(_spread(rng, 1, 64), vocab, _spread(rng, 1, 4096), dtype=rng.choice(("f32", "f32", "f16")), masks=rng.choice((0, 1, _spread(rng, 1, 64))),
                      biases=rng.choice((0, _spread(rng, 1, 300))))
    more = {"ragged": rng.random() < 0.7, "page": rng.choice((16, 32, 64, 64, 128)), "norm": rng.random() < 0.3, "sink": rng.random() < 0.3,
            "softcap": rng.choice((0.0, 0.0, 30.0)), "window": rng.choice((0, 0, _spread(rng, 64, 4096)))}
    dim = rng.choice((32, 48, 64, 64, 80, 96, 128, 128))
    kv = rng.choice((1, 2, 3, 4, 8))
    size = rng.choice(("1b", "4b", "27b", (kv * rng.randint(1, 6), kv, dim, rng.choice((dim, 2 * dim)))))
    if rng.random() < 0.15:
        dim = rng.choice((24, 32, 40, 64))
        return _attention((kv * rng.randint(1, 3), kv, dim, 2 * dim), _spread(rng, 1, 4), rng.choice((1, _spread(rng, 2, 150))), _spread(rng, 1, 200), dtype="f32", **more)
    if kind == "token":
        seqs = _spread(rng, 1, 64)
        return _attention(size, seqs, 1, _spread(rng, 1, min(32768, 131072 // seqs)), **more)
    seqs = _spread(rng, 1, 16)
    return _attention(size, seqs, _spread(rng, 2, 4096 // seqs), rng.choice((0, _spread(rng, 1, 2000))) // seqs, **more)


# ── the sequences of an attention case ──
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
    if case["kind"] == "rules":
        rows, vocab = case["rows"], case["vocab"]
        read = rows * vocab * (2 if case["dtype"] == "f16" else 4) + case["masks"] * -(-vocab // 32) * 4 + rows * (case["history"] * 4 + case["biases"] * 8)
        return {"bytes": read + rows * vocab * 4, "flops": rows * vocab}
    pairs, keys, rows = _seen(case)
    heads, kv, dim, vdim, size = case["heads"], case["kv_heads"], case["dim"], case["vdim"], 2 if case["dtype"] == "bf16" else 4
    per_key = kv * (2 * dim + vdim)
    moved = rows * (heads * 2 * dim + per_key) + keys * per_key + rows * heads * vdim  # projections in, keys and values (the new ones are written), results
    return {"bytes": moved * size, "flops": pairs * heads * (4 * dim + 2 * vdim)}


# ── inputs ──
def _turns(dim):
    """[2, dim / 2] f32: turns per position of each pair of dimensions, as the sum of two f32."""
    turns = np.array([10000.0 ** (-2.0 * i / dim) / (2.0 * math.pi) for i in range(dim // 2)])
    high = turns.astype(np.float32)
    return np.stack([high, (turns - high).astype(np.float32)])


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    if case["kind"] == "rules":
        state = _rules_inputs(case, seed, gen, randn)
    else:
        state = _attention_inputs(case, seed, gen, randn)
    if own:
        _own_handles(state)
    return state


def _attention_inputs(case, seed, gen, randn):
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    heads, kv, dim, vdim, page = case["heads"], case["kv_heads"], case["dim"], case["vdim"], case["page"]
    lengths = _lengths(case)
    rows = sum(n for n, _ in lengths)
    held = [-(-(n + past) // page) for n, past in lengths]
    pages, width = sum(held), max(held)
    host = np.random.default_rng(seed)
    order, table, at, row = host.permutation(pages).astype(np.int32), np.zeros((len(lengths), width), np.int32), 0, 0
    seqs = np.zeros((len(lengths), 4), np.int32)
    for i, (n, past) in enumerate(lengths):
        table[i, :held[i]] = order[at:at + held[i]]
        seqs[i] = row, n, past, i
        at, row = at + held[i], row + n
    # queries of a spread that lets some keys stand out
    proj = randn(rows, heads * 2 * dim + kv * (2 * dim + vdim))
    proj[:, :heads * 2 * dim] *= 1.5
    return {"case": case, "proj": proj.to(dtype), "keys": randn(pages, kv, page, 2 * dim).to(dtype), "values": randn(pages, kv, page, vdim).to(dtype),
            "turns": torch.from_numpy(_turns(dim)).cuda(), "lambda": 0.2 + 0.6 * torch.rand(heads, generator=gen, device="cuda"), "gain": 0.2 * (1.0 + 0.1 * randn(vdim)),
            "seqs": torch.from_numpy(seqs).cuda(), "table": torch.from_numpy(table).cuda()}


def _rules_inputs(case, seed, gen, randn):
    rows, vocab, n, host = case["rows"], case["vocab"], case["history"], np.random.default_rng(seed)
    # logits with a few that stand out; answers come back to some of their tokens
    logits = (2.0 * randn(rows, vocab) + 6.0 * (torch.rand(rows, vocab, generator=gen, device="cuda") < 0.001)).to(torch.float16 if case["dtype"] == "f16" else torch.float32)
    common = host.integers(0, vocab, 64)
    history = np.where(host.random((rows, n)) < 0.3, common[host.integers(0, 64, (rows, n))], host.integers(0, vocab, (rows, n))).astype(np.int32)
    total = n - np.arange(rows) * 29 % (n // 2 + 1)
    lengths = np.stack([total // 3, total], 1).astype(np.int32)
    penalties = np.stack([host.uniform(1.0, 1.4, rows), host.uniform(0.0, 0.5, rows), host.uniform(0.0, 0.7, rows)], 1).astype(np.float32)
    state = {"case": case, "logits": logits, "history": history, "lengths": lengths, "penalties": penalties}
    if case["biases"]:
        state["bias_ids"] = np.stack([host.permutation(vocab)[:case["biases"]] for _ in range(rows)]).astype(np.int32)
        state["bias"] = host.normal(0.0, 5.0, state["bias_ids"].shape).astype(np.float32)
    state = {k: torch.from_numpy(v).cuda() if isinstance(v, np.ndarray) else v for k, v in state.items()}
    if case["masks"]:
        words = -(-vocab // 32)
        state["masks"] = torch.randint(-2 ** 31, 2 ** 31, (case["masks"], words), generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
        state["mask_of"] = torch.from_numpy((np.arange(rows) % (case["masks"] + 1) - (rows > case["masks"])).astype(np.int32)).cuda()
    return state


# ── the framework's calls ──
def _own_handles(state):
    """The session, and what a program has on the device between steps."""
    from onyxia_b200 import ir
    from onyxia_b200.backend import CudaBackend

    case = state["case"]
    b = ir.GraphBuilder()

    def up(session, name, x):
        kind = {torch.float32: ir.F32, torch.float16: ir.F16, torch.bfloat16: ir.BF16, torch.int32: ir.U32 if name == "masks" else ir.I32}[x.dtype]
        return session.upload_device(kind, tuple(x.shape), x.data_ptr(), torch.cuda.current_stream().cuda_stream)

    if case["kind"] == "rules":
        b.output("one", b.const_f32([1.0], [1]))
        session = CudaBackend((0,)).prepare(b.finish())
        state["session"] = session
        state["handles"] = {k: up(session, k, v) for k, v in state.items() if torch.is_tensor(v)}
        return
    dtype = ir.BF16 if case["dtype"] == "bf16" else ir.F32
    heads, kv, dim, vdim, page = case["heads"], case["kv_heads"], case["dim"], case["vdim"], case["page"]
    N, R, NP, TW = b.sym("num_tokens"), b.sym("num_seqs"), b.sym("num_pages"), b.sym("table_width")
    const = lambda x: b.constant(ir.HostTensor.from_numpy(x.cpu().numpy()))  # noqa: E731
    proj = b.input("proj", dtype, [N, heads * 2 * dim + kv * (2 * dim + vdim)])
    keys, values = b.input("pages.keys", dtype, [NP, kv, page, 2 * dim]), b.input("pages.values", dtype, [NP, kv, page, vdim])
    seqs, table = b.input("seq_info", ir.I32, [R, 4]), b.input("page_table", ir.I32, [R, TW])
    attrs = {"heads": heads, "kv_heads": kv, "dim": dim, "vdim": vdim, "q_offset": 0, "k_offset": heads * 2 * dim, "v_offset": (heads + kv) * 2 * dim, "rot_dims": dim,
             "scale": dim ** -0.5, "window": case["window"], "softcap": float(case["softcap"]), "norm": int(case["norm"]), "epsilon": EPS, "sink": int(case["sink"]),
             "head_norm": 1, "head_epsilon": HEAD_EPS}
    out, new_keys, new_values = b.composite(
        "onyxia.DifferentialAttention", attrs, [proj, const(state["turns"]), keys, values, seqs, table, const(state["lambda"]), const(state["gain"])],
        [(dtype, [N, heads * vdim]), (dtype, [NP, kv, page, 2 * dim]), (dtype, [NP, kv, page, vdim])])
    b.output("out", out)
    b.output("updated.pages.keys", new_keys)
    b.output("updated.pages.values", new_values)
    session = CudaBackend((0,)).prepare(b.finish())
    state["session"] = session
    named = {"proj": "proj", "pages.keys": "keys", "pages.values": "values", "seq_info": "seqs", "page_table": "table"}
    state["feed"] = [(name, up(session, key, state[key])) for name, key in named.items()]
    state["pools"] = {key: _view(session, t) for key, (_, t) in zip(("keys", "values"), state["feed"][1:3])}


def _view(session, t):
    """A tensor of the session as torch sees it: the same memory."""
    from onyxia_b200 import ir

    x = torch.as_tensor(session.view(t, torch.cuda.current_stream().cuda_stream), device="cuda")
    return x.view(torch.bfloat16) if t.dtype == ir.BF16 else x


def run(state):
    if state["case"]["kind"] == "rules":
        if not own:
            return _plain_rules(state)
        h = state["handles"]
        return _view(state["session"], state["session"].constrain_last(h["logits"], **{k: v for k, v in h.items() if k != "logits"}))
    if not own:
        return _plain_attention(state)
    outs = state["session"].run(state["feed"])
    return {"out": _view(state["session"], outs[0][1]), "keys": state["pools"]["keys"], "values": state["pools"]["values"]}


# ── plain forms ──
def _rotate(x, turns, pos):
    """x [rows, heads, dim] at positions pos [rows]: dimension i turns with i + dim / 2. Angles in 64 bits."""
    t = pos[:, None].double() * turns.double().sum(0)
    t = (t - t.round()) * (2.0 * math.pi)
    cos, sin = t.cos().float()[:, None], t.sin().float()[:, None]
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_attention(s):
    c = s["case"]
    heads, kv, dim, vdim, page = c["heads"], c["kv_heads"], c["dim"], c["vdim"], c["page"]
    rep, start, count, past = heads // kv, s["seqs"][:, 0].long(), s["seqs"][:, 1].long(), s["seqs"][:, 2].long()
    rows = s["proj"].shape[0]
    seq = torch.repeat_interleave(torch.arange(len(count), device="cuda"), count, output_size=rows)
    place = torch.arange(rows, device="cuda") - start[seq]
    pos = past[seq] + place
    x = s["proj"].float()
    q, k, v = x.split([heads * 2 * dim, kv * 2 * dim, kv * vdim], 1)
    qk = _rotate(torch.cat([q, k], 1).reshape(rows, -1, dim), s["turns"], pos)
    if c["norm"]:
        qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + EPS)
    q, k = qk.split([heads * 2, kv * 2], 1)
    pg, off = s["table"].long()[seq, pos // page], pos % page
    s["keys"][pg, :, off] = k.reshape(rows, kv, 2 * dim).to(s["keys"].dtype)
    s["values"][pg, :, off] = v.reshape(rows, kv, vdim).to(s["values"].dtype)
    # every sequence's keys and values one behind the other, its rows side by side
    longest, table = c["new"], s["table"].long()
    keys = s["keys"][table].float().transpose(2, 3).reshape(len(count), -1, kv, 2, dim)
    values = s["values"][table].float().transpose(2, 3).reshape(len(count), -1, kv, vdim)
    queries = torch.zeros(len(count), longest, heads, 2, dim, device="cuda")
    queries[seq, place] = q.reshape(rows, heads, 2, dim)
    queries = queries.reshape(len(count), longest, kv, rep, 2, dim).permute(0, 2, 4, 3, 1, 5).reshape(len(count), kv, 2, rep * longest, dim)
    scores = (queries @ keys.permute(0, 2, 3, 4, 1)).mul_(dim ** -0.5)
    if c["softcap"]:
        scores = scores.div_(c["softcap"]).tanh_().mul_(c["softcap"])
    at, key = past[:, None] + torch.arange(longest, device="cuda"), torch.arange(keys.shape[1], device="cuda")
    hidden = key > at[..., None]
    if c["window"]:
        hidden |= key <= at[..., None] - c["window"]
    scores = scores.view(len(count), kv, 2, rep, longest, -1).masked_fill_(hidden[:, None, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    if c["sink"]:
        top = top.clamp_min_(0.0)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    if c["sink"]:
        total = total + (-top).exp()
    total[:, :, 1] /= -s["lambda"].view(kv, rep, 1, 1)
    weights = weights.div_(total)
    out = weights.sum(2).view(len(count), kv, rep * longest, -1) @ values.transpose(1, 2)
    out = out * torch.rsqrt(out.square().mean(-1, keepdim=True) + HEAD_EPS) * s["gain"]
    out = out.view(len(count), heads, longest, vdim)[seq, :, place]
    return {"out": out.reshape(rows, heads * vdim).to(s["proj"].dtype), "keys": s["keys"], "values": s["values"]}


def _plain_rules(s):
    c = s["case"]
    rows, vocab = c["rows"], c["vocab"]
    x, tokens = s["logits"].float(), s["history"].long()
    place = torch.arange(tokens.shape[1], device="cuda")
    held = (place < s["lengths"][:, 1:]).float()
    said = held * (place >= s["lengths"][:, :1])
    seen = torch.zeros(rows, vocab, device="cuda").scatter_add_(1, tokens, held)
    times = torch.zeros(rows, vocab, device="cuda").scatter_add_(1, tokens, said)
    repetition, frequency, presence = (s["penalties"][:, i:i + 1] for i in range(3))
    x = torch.where(seen > 0, torch.where(x > 0, x / repetition, x * repetition), x)
    x = x - times * frequency - (times > 0) * presence
    if c["biases"]:
        x = x.scatter_add(1, s["bias_ids"].long(), s["bias"])
    if c["masks"]:
        bits = (s["masks"][..., None] >> torch.arange(32, device="cuda", dtype=torch.int32) & 1).bool().reshape(c["masks"], -1)[:, :vocab]
        mask_of = s["mask_of"].long()
        x = x.masked_fill(~(bits[mask_of.clamp_min(0)] | (mask_of < 0)[:, None]), -math.inf)
    return x


# ── the same from the definitions, in 64 bits ──
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return _exact_rules(case, s) if case["kind"] == "rules" else _exact_attention(case, s)


def _exact_rules(case, s):
    out = s["logits"].double()
    history, lengths, penalties = (s[k].cpu().numpy() for k in ("history", "lengths", "penalties"))
    for r in range(case["rows"]):
        prompt, total = lengths[r].tolist()
        repetition, frequency, presence = (float(p) for p in penalties[r])
        ids = torch.from_numpy(np.unique(history[r, :total]).astype(np.int64)).cuda()
        out[r, ids] = torch.where(out[r, ids] > 0, out[r, ids] / repetition, out[r, ids] * repetition)
        ids, times = np.unique(history[r, prompt:total], return_counts=True)
        out[r, torch.from_numpy(ids.astype(np.int64)).cuda()] -= torch.from_numpy(times * frequency + presence).cuda()
        if case["biases"]:
            out[r].index_add_(0, s["bias_ids"][r].long(), s["bias"][r].double())
        if case["masks"] and (m := int(s["mask_of"][r])) >= 0:
            allowed = np.unpackbits(s["masks"][m].cpu().numpy().view(np.uint8), bitorder="little")[:case["vocab"]]
            out[r, torch.from_numpy(allowed).cuda() == 0] = -math.inf
    return out


def _exact_attention(case, s):
    pairs = _seen(case)[0] * case["heads"]
    if pairs > 1e9:  # some seconds of 64-bit products
        return None
    heads, kv, dim, vdim, page, dev = case["heads"], case["kv_heads"], case["dim"], case["vdim"], case["page"], "cuda"
    keys, values, x = s["keys"].double(), s["values"].double(), s["proj"].double()
    turns, lam, gain = s["turns"].double().sum(0), s["lambda"].double(), s["gain"].double()
    out, row = torch.empty(x.shape[0], heads, vdim, dtype=torch.float64, device=dev), 0
    for i, (new, past) in enumerate(_lengths(case)):
        angle = 2.0 * math.pi * torch.arange(past, past + new, device=dev, dtype=torch.float64)[:, None] * turns
        mine = x[row:row + new]

        def turned(first, n):
            y = mine[:, first:first + n * dim].reshape(new, n, dim)
            z = torch.complex(y[..., :dim // 2], y[..., dim // 2:]) * torch.polar(torch.ones_like(angle), angle)[:, None]
            y = torch.cat([z.real, z.imag], -1)
            return y / (y.pow(2).mean(-1, keepdim=True) + EPS).sqrt() if case["norm"] else y

        q, k, v = turned(0, heads * 2), turned(heads * 2 * dim, kv * 2).reshape(new, kv, 2 * dim), mine[:, (heads + kv) * 2 * dim:].reshape(new, kv, vdim)
        spots = torch.arange(past + new, device=dev)
        pg, off = s["table"][i].long()[spots // page], spots % page
        keys[pg[past:], :, off[past:]] = k.to(s["keys"].dtype).double()  # as the pool holds them
        values[pg[past:], :, off[past:]] = v
        at = torch.arange(past, past + new, device=dev)[:, None]
        seen = (spots <= at) & (spots > at - case["window"]) if case["window"] else spots <= at
        for h in range(heads):
            g, maps = h // (heads // kv), []
            for m in (0, 1):
                t = q[:, 2 * h + m] @ keys[pg, g, off, m * dim:(m + 1) * dim].T / math.sqrt(dim)
                if case["softcap"]:
                    t = case["softcap"] * torch.tanh(t / case["softcap"])
                t = t.masked_fill(~seen, -math.inf)
                if case["sink"]:
                    t = torch.cat([t, torch.zeros(new, 1, dtype=torch.float64, device=dev)], 1)
                maps.append(torch.softmax(t, 1)[:, :past + new])
            o = (maps[0] - lam[h] * maps[1]) @ values[pg, g, off]
            out[row:row + new, h] = o / (o.pow(2).mean(1, keepdim=True) + HEAD_EPS).sqrt() * gain
        row += new
    return {"out": out.reshape(row, heads * vdim), "keys": keys, "values": values}
