"""Rotary positions, appending to a paged cache and attention over it, stated in 64 bits value by value; and the steps that the tests run."""
import math

import numpy as np
import torch

F64 = torch.float64
TYPES = {"f16": torch.float16, "f32": torch.float32, "bf16": torch.bfloat16}
NO_PAGE = 0xFFFFFFFF


def half_step(dtype):
    """A rounding is off by at most half a step, relative to the value."""
    return torch.finfo(TYPES[dtype]).eps / 2


def padded(dim):
    return next(p for p in (32, 64, 128, 192, 256) if dim <= p)


def turn(x, positions, frequencies, amplitude, rot, first, halves):
    """x [rows, heads, dim] in 64 bits; (turned, what the errors of a pair are relative to)."""
    y, size = x.to(F64).clone(), torch.zeros(x.shape, dtype=F64)
    angle = torch.as_tensor(np.asarray(positions, np.float64))[:, None] * torch.as_tensor(np.asarray(frequencies, np.float64))[None, :rot // 2]
    c, s = angle.cos()[:, None] * amplitude, angle.sin()[:, None] * amplitude
    i = torch.arange(rot // 2)
    a, b = (first + i, first + i + rot // 2) if halves else (first + 2 * i, first + 2 * i + 1)
    u, v = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = u * c - v * s, v * c + u * s
    size[..., a] = size[..., b] = (u.abs() + v.abs()) * abs(amplitude) * (1 + angle.abs()[:, None] * 2.0 ** -31)
    return y, size


def turn_tolerance(want, size, dtype):
    """One rounding of the result, and of what it is made of: the fraction of a turn in 32 bits (an angle off by pi 2^-25), sine and cosine
    (2 ulp: 2^-22 of 1 at most), the amplitude and the two products (2^-24 each): together below 2^-21 of |a| + |b|.  Far positions: the product
    with the frequency and the division into turns, in 64 bits, 2^-52 of the angle (`size` has it).  f16 has a smallest step."""
    return half_step(dtype) * want.abs() + size * 2.0 ** -21 + (2.0 ** -25 if dtype == "f16" else 0)


class Step:
    """Sequences given as (rows, positions with them), pages dealt out in a shuffled order."""

    def __init__(self, sequences, page, seed=0, spare=3, table_extra=1):
        self.sequences, self.page = list(sequences), page
        rng = np.random.default_rng(seed)
        need = [max(-(-length // page), 0) for _, length in self.sequences]
        self.pages = sum(need) + spare
        order = rng.permutation(self.pages).astype(np.uint32)
        self.table = np.full((len(need), max(need + [0]) + table_extra), NO_PAGE, np.uint32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.starts = np.concatenate([[0], np.cumsum([n for n, _ in self.sequences])]).astype(np.uint32)
        self.lengths = np.asarray([length for _, length in self.sequences], np.uint32)
        self.rows = int(self.starts[-1])
        self.max_rows = max([n for n, _ in self.sequences] + [1])
        self.max_length = max([length for _, length in self.sequences] + [1])

    def places(self):
        """(row, sequence, position, page or -1, slot) of every row that stands somewhere."""
        for s, (n, length) in enumerate(self.sequences):
            for i in range(n):
                p = length - n + i
                if p < 0:
                    continue
                b = p // self.page
                pg = int(self.table[s, b]) if b < self.table.shape[1] else NO_PAGE
                yield int(self.starts[s]) + i, s, p, pg if pg < self.pages else -1, p % self.page


def appended(step, k, v, keys, values, q, frequencies, amplitude, rot, first, halves):
    """(keys, values, q_output) after an append, in 64 bits, with NaN where q_output is left alone; sizes for the tolerances beside them."""
    keys, values = keys.to(F64).clone(), values.to(F64).clone()
    ksize, qout, qsize = torch.zeros_like(keys), None, None
    dim = k.shape[2]
    places = list(step.places())
    rows, at = [p[0] for p in places], [p[2] for p in places]
    tk, sk = turn(k[rows], at, frequencies, amplitude, rot, first, halves)
    for j, (row, _, _, pg, slot) in enumerate(places):
        if pg < 0:
            continue
        keys[pg, :, slot], values[pg, :, slot], ksize[pg, :, slot] = 0.0, 0.0, 0.0
        keys[pg, :, slot, :dim], values[pg, :, slot, :dim], ksize[pg, :, slot, :dim] = tk[j], v[row].to(F64), sk[j]
    if q is not None:
        qout, qsize = torch.full(q.shape, math.nan, dtype=F64), torch.zeros(q.shape, dtype=F64)
        tq, sq = turn(q[rows], at, frequencies, amplitude, rot, first, halves)
        qout[rows], qsize[rows] = tq, sq
    return keys, values, qout, ksize, qsize


def attended(step, q, keys, values, scale, window=0, sink=None, max_length=None, max_rows=None):
    """(output, tolerance without its own rounding) of attention in 64 bits; rows that are left alone are NaN.

    A score's error is that of a sum of dim products in 32 bits, (dim + 8) 2^-24 of the products' absolute sum, and of its scaling and the
    difference to the maximum, 2^-22 of the largest score; a weight is off by that, 2^-21 of itself for the power of two, and one rounding to
    the type where that has 16 bits; the sums of n weights and products by n 2^-24.  Both sums: twice."""
    R, H, d = q.shape
    G, page = keys.shape[1], step.page
    out, tol = torch.full(q.shape, math.nan, dtype=F64), torch.zeros(q.shape, dtype=F64)
    cap = min(step.table.shape[1] * page, step.max_length if max_length is None else max_length)
    rounding = 0.0 if q.dtype == torch.float32 else torch.finfo(q.dtype).eps / 2
    for s, (n, length) in enumerate(step.sequences):
        if n == 0:
            continue
        at = torch.arange(min(length, cap))
        pg = torch.as_tensor(step.table[s].astype(np.int64))[at // page]
        there = pg < step.pages
        at, pg = at[there], pg[there]
        k, v = (x[pg, :, at % page, :d].to(F64) for x in (keys, values))          # [positions, kv heads, dim]
        for i in range(min(n, step.max_rows if max_rows is None else max_rows)):
            p, row = length - n + i, int(step.starts[s]) + i
            ok = at <= p
            if window:
                ok &= at > p - window
            if not bool(ok.any()):
                out[row] = 0.0
                continue
            kk, vv = (x[ok].repeat_interleave(H // G, 1) for x in (k, v))
            qq = q[row].to(F64)
            z = torch.einsum("hd,phd->hp", qq, kk) * scale
            size = torch.einsum("hd,phd->hp", qq.abs(), kk.abs()).amax(1) * abs(scale)
            top = z.amax(1, keepdim=True)
            if sink is not None:
                top = torch.maximum(top, sink.to(F64)[:, None])
            w = torch.exp(z - top)
            total = w.sum(1, keepdim=True) + (0 if sink is None else torch.exp(sink.to(F64)[:, None] - top))
            w = w / total
            out[row] = torch.einsum("hp,phd->hd", w, vv)
            off = (d + 8) * 2.0 ** -24 * size + 2.0 ** -22 * torch.maximum(z.abs().amax(1), top[:, 0].abs()) + 2.0 ** -21 + rounding + len(z[0]) * 2.0 ** -24
            tol[row] = torch.einsum("hp,phd->hd", w, vv.abs()) * 2 * off[:, None]
    return out, tol


def told_apart(step, q, keys, values, scale, dtype, **more):
    """Of outputs that are wrong in some way, the share of values that attention's tolerance tells from the right ones: zeros, negated ones, those of the pages one
    further in the table, those of keys one slot further."""
    want, tol = attended(step, q, keys, values, scale, **more)
    tol = half_step(dtype) * want.abs() + tol + (2.0 ** -25 if dtype == "f16" else 0)
    seen = tol > 0
    other = Step.__new__(Step)
    other.__dict__.update(step.__dict__)
    other.table = np.stack([np.concatenate([np.roll(row[row != NO_PAGE], 1), row[row == NO_PAGE]]) for row in step.table]).astype(np.uint32)
    wrong = {"zeros": torch.zeros_like(want), "negated": -want, "pages": attended(other, q, keys, values, scale, **more)[0],
             "slots": attended(step, q, keys.roll(1, 2), values, scale, **more)[0]}
    return {name: float(((w - want).abs() > tol)[seen].double().mean()) for name, w in wrong.items()}
