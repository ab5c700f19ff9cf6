"""What a bf16 kernel of differential attention may be off by, from the weights themselves: the formulas in 64 bits, a head at a time, with the share of its error that each (row, head) is due.

A result is off by the rounding of its own bits and by that of the weights: o = o_0 − λ o_1, o_m = Σ_j w_mj v_j, with every exponential off by a rounding δ of its own. Sums are taken of the
rounded exponentials, so that o_m is off by Σ_j w_mj δ_mj (v_j − o_m): a key that takes all weight costs nothing. With independent δ the error of o is to o as

  D = sqrt(Σ_j w_0j² |v_j − o_0|² + λ² Σ_j w_1j² |v_j − o_1|²) / |o|

times a rounding. A rounding to bf16 is half a step of 2^-7 at most, and where mantissas are spread evenly over their octave, as logarithms, sqrt(mean square) of the error relative to the
value is 2^-7 / sqrt(12) · sqrt(3 / (8 ln 2)) = 1.66e-3. Queries enter as the sum of two bf16 (2^-17: nothing beside it), keys as the pool holds them.
"""
import math

import numpy as np

from onyxia_b200.kipizen import turns_per_position

ROUNDING = 2.0 ** -7 / math.sqrt(12.0) * math.sqrt(3.0 / (8.0 * math.log(2.0)))


def exact(f, s, stored):
    """(results [rows, heads, vdim], D [rows, heads]) for `Form` f and `Step` s; rows of no sequence are NaN."""
    x, keys, values = s.proj.astype(np.float64), s.keys.astype(np.float64), s.values.astype(np.float64)
    turns = turns_per_position(f.rot_dims, 10000.0, 1.0).astype(np.float64).sum(0)
    q0, k0, v0 = f.offsets
    half, rep = f.rot_dims // 2, f.heads // f.kv_heads
    out, due = np.full((len(x), f.heads, f.vdim), np.nan), np.full((len(x), f.heads), np.nan)

    def turned(y, pos):
        z = y.copy()
        if half:
            e = np.exp(2j * math.pi * pos[:, None] * turns)[:, None, None] * (y[..., :half] + 1j * y[..., half:2 * half])
            z[..., :half], z[..., half:2 * half] = e.real, e.imag
        return z / np.sqrt((z ** 2).mean(-1, keepdims=True) + f.eps) if f.norm else z

    for i, (row, n, past, _) in enumerate(s.seqs):
        if n == 0:
            continue
        mine, new, spots = x[row:row + n], np.arange(past, past + n), np.arange(past + n)
        q = turned(mine[:, q0:q0 + f.heads * 2 * f.dim].reshape(n, f.heads, 2, f.dim), new.astype(np.float64))
        k = turned(mine[:, k0:k0 + f.kv_heads * 2 * f.dim].reshape(n, f.kv_heads, 2, f.dim), new.astype(np.float64))
        keys[s.table[i, new // f.page], :, new % f.page] = stored(k).astype(np.float64).reshape(n, f.kv_heads, -1)
        values[s.table[i, new // f.page], :, new % f.page] = mine[:, v0:v0 + f.kv_heads * f.vdim].reshape(n, f.kv_heads, f.vdim)
        pg, off = s.table[i, spots // f.page], spots % f.page
        hidden = spots > new[:, None]
        if f.window:
            hidden |= spots <= new[:, None] - f.window
        for h in range(f.heads):
            o, lost, lam, v = np.zeros((n, f.vdim)), np.zeros(n), float(s.lam[h]), values[pg, h // rep, off]
            for m, factor in ((0, 1.0), (1, -lam)):
                t = q[:, h, m] @ keys[pg, h // rep, off, m * f.dim:(m + 1) * f.dim].T * f.scale
                if f.softcap:
                    t = f.softcap * np.tanh(t / f.softcap)
                t[hidden] = -np.inf
                top = t.max(1, keepdims=True)
                if f.sink:
                    top = np.maximum(top, 0.0)
                e = np.exp(t - top)
                w = e / (e.sum(1, keepdims=True) + (np.exp(-top) if f.sink else 0.0))
                o_m, w2 = w @ v, w * w
                o += factor * o_m
                lost += factor ** 2 * (w2 @ (v * v).sum(1) - 2.0 * (o_m * (w2 @ v)).sum(1) + (o_m * o_m).sum(1) * w2.sum(1))
            due[row:row + n, h] = np.sqrt(np.maximum(lost, 0.0) / (o * o).sum(1))
            out[row:row + n, h] = o / np.sqrt((o * o).mean(1, keepdims=True) + f.head_eps) * s.gain if f.head_norm else o
    return out, due


def share(f, s, got, stored, two_parts=False):
    """Error of all results together as a share of what they are due: sqrt(mean of (error / result)²) over sqrt(mean of ROUNDING² (1 + D²)), over (row, head). With weights in two bf16 (2^-17)
    results are due their own rounding alone."""
    want, due = exact(f, s, stored)
    live = ~np.isnan(due[:, 0])
    got, want, due = got.reshape(want.shape)[live].astype(np.float64), want[live], due[live]
    assert np.isfinite(got).all()
    off = ((got - want) ** 2).mean(-1) / (want ** 2).mean(-1)
    due = 0.0 * due if two_parts else due
    return float(np.sqrt(off.mean() / (ROUNDING ** 2 * (1.0 + due ** 2)).mean()))
