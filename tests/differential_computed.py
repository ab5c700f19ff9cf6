"""The module of one onyxia.DifferentialAttention (or onyxia.PagedKVAttention) whose batch description, page table or angles the module computes itself."""
import numpy as np

from onyxia_b200 import ir
from onyxia_b200.ir import HostTensor
from onyxia_b200.kipizen import turns_per_position


def module(f, dtype, lam, gain, computed=(), maps=2):
    """`f`: differential_util.Form. `computed`: of "seq_info" and "page_table", which come as I64 and are narrowed, "turns", which come as two addends, and "reshaped": a page table with an axis more."""
    b = ir.GraphBuilder()
    N, R, NP, TW = b.sym("num_tokens"), b.sym("num_seqs"), b.sym("num_pages"), b.sym("table_width")
    const = lambda a: b.constant(HostTensor.from_numpy(np.ascontiguousarray(a, np.float32)))  # noqa: E731
    proj = b.input("proj", dtype, [N, f.width])
    keys, values = b.input("pages.keys", dtype, [NP, f.kv_heads, f.page, maps * f.dim]), b.input("pages.values", dtype, [NP, f.kv_heads, f.page, f.vdim])

    def whole(name, shape):
        if name in computed:
            return b.cast(b.input(name, ir.I64, shape), ir.I32)
        return b.input(name, ir.I32, shape)

    seqs = whole("seq_info", [R, 4])
    table = b.reshape(b.input("page_table", ir.I32, [R, 1, TW]), [R, TW]) if "reshaped" in computed else whole("page_table", [R, TW])
    turns = turns_per_position(f.rot_dims, 10000.0, 1.0)
    turns = b.add(const(turns / 2), const(turns / 2)) if "turns" in computed else const(turns)
    q, k, v = f.offsets
    attrs = {"heads": f.heads, "kv_heads": f.kv_heads, "dim": f.dim, "vdim": f.vdim, "q_offset": q, "k_offset": k, "v_offset": v, "rot_dims": f.rot_dims, "window": f.window,
             "scale": float(f.scale), "softcap": float(f.softcap), "norm": f.norm, "epsilon": f.eps, "sink": f.sink}
    outs = [(dtype, [N, f.heads * f.vdim]), (dtype, [NP, f.kv_heads, f.page, maps * f.dim]), (dtype, [NP, f.kv_heads, f.page, f.vdim])]
    b.set_loc("mix", "attention")
    if maps == 2:
        o = b.composite("onyxia.DifferentialAttention", dict(attrs, head_norm=f.head_norm, head_epsilon=f.head_eps), [proj, turns, keys, values, seqs, table, const(lam)] + ([const(gain)] if f.head_norm else []), outs)
    else:
        o = b.composite("onyxia.PagedKVAttention", attrs, [proj, turns, keys, values, seqs, table], outs)
    for name, x in zip(("out", "updated.pages.keys", "updated.pages.values"), o):
        b.output(name, x)
    return b.finish()
