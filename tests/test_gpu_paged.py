"""Rotary positions, appending to a paged cache and attention over it against their statements in 64 bits (paged_models.py)."""
import math

import numpy as np
import pytest
import torch

from paged_models import F64, NO_PAGE, TYPES, Step, appended, attended, half_step, padded, told_apart, turn, turn_tolerance

pytestmark = pytest.mark.gpu
BITS = {"f16": torch.int16, "bf16": torch.int16, "f32": torch.int32}


def code(pkg, dtype):
    return {"f16": pkg.F16, "f32": pkg.F32, "bf16": pkg.BF16}[dtype]


def raw(t):
    return t.contiguous().view(torch.uint8).numpy().reshape(-1)


class Device:
    def __init__(self, pkg, gpu):
        self.pkg, (self.ctx, self.K) = pkg, gpu

    def up(self, t, lead=0):
        """A buffer of t's values; `lead` bytes from the start of its memory."""
        if isinstance(t, np.ndarray):
            t = torch.from_numpy(t.view(np.int32) if t.dtype == np.uint32 else t)
        b = raw(t)
        whole = self.pkg.Buffer.from_slice(self.ctx, np.concatenate([np.zeros(lead, np.uint8), b, np.zeros(16 if b.size == 0 else 0, np.uint8)]))
        return whole.view(lead, max(b.size, 16) if b.size == 0 else b.size) if lead else whole

    def down(self, b, shape, dtype):
        n = math.prod(shape) * (4 if dtype == "f32" else 2)
        return torch.from_numpy(b.as_array(np.uint8, n).copy()).view(TYPES[dtype]).reshape(shape)

    def batch(self):
        return self.pkg.CommandBatch(self.ctx)


@pytest.fixture(scope="module")
def dev(pkg, gpu):
    return Device(pkg, gpu)


def normal(seed, *shape, dtype="f32"):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(TYPES[dtype])


def close(got, want, tol, what=""):
    off = (got.to(F64) - want).abs()
    bad = ~(off <= tol) & ~(got.to(F64).isnan() & want.isnan()) & ~(got.to(F64) == want)
    assert not bool(bad.any()), (what, int(bad.sum()), float((off / tol.clamp_min(1e-300))[bad].max()), bad.nonzero()[:3].tolist())


def same_bits(a, b, dtype):
    return bool((a.contiguous().view(BITS[dtype]) == b.contiguous().view(BITS[dtype])).all())


# ---- rotary positions ---------------------------------------------------------------------------------------------------------
ROTARY = [  # rows, heads, dim, rot, first, halves, margin in front, behind, in place
    (1, 32, 128, 128, 0, True, 0, 0, False), (3, 4, 64, 64, 0, False, 0, 0, True), (5, 2, 80, 50, 30, False, 16, 8, False), (7, 3, 33, 10, 5, True, 1, 2, True),
    (2, 1, 256, 64, 192, True, 0, 64, True), (4, 5, 96, 32, 0, True, 8, 0, False), (1, 1, 2, 2, 0, True, 0, 0, False), (9, 7, 40, 0, 0, False, 3, 0, False),
    (3, 2, 1024, 1024, 0, True, 0, 0, True), (2, 3, 1023, 1022, 1, False, 0, 1, False), (4099, 2, 64, 32, 32, True, 0, 0, True), (9001, 1, 48, 48, 0, False, 0, 0, False),
    (8200, 3, 20, 12, 4, True, 4, 4, False),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,heads,dim,rot,first,halves,front,behind,inplace", ROTARY)
def test_rotary_rows(dev, dtype, rows, heads, dim, rot, first, halves, front, behind, inplace):
    pkg, K = dev.pkg, dev.K
    ld, size = heads * dim + front + behind, 4 if dtype == "f32" else 2
    x = normal(rows + dim, rows, ld, dtype=dtype)
    f = K.rotary_frequencies(max(rot, 2), 1e4)[0]
    at = np.random.default_rng(rows).integers(0, 1 << 17, rows).astype(np.uint32)
    at[0] = 0xFFFFFFFF if rows > 2 else at[0]
    amplitude = 1.25 if dim % 3 else 1.0
    bx, out_ld = dev.up(x), ld if inplace else heads * dim + 3 * (dim % 2)
    marked = torch.full((rows, out_ld), 7.0).to(TYPES[dtype])
    out = bx if inplace else dev.up(marked)
    src = bx.view(front * size, bx.length() - front * size)
    K.rotary_rows_into(dev.batch(), src, src if inplace else out, code(pkg, dtype), dev.up(at), dev.up(f), amplitude, rows, heads, dim, rot, first,
                       pkg.ROTARY_HALVES if halves else pkg.ROTARY_PAIRS, ld, out_ld)
    got = dev.down(out, (rows, out_ld), dtype)
    lo = front if inplace else 0
    beside = torch.cat([got[:, :lo], got[:, lo + heads * dim:]], 1)
    was = x if inplace else marked
    assert same_bits(beside, torch.cat([was[:, :lo], was[:, lo + heads * dim:]], 1), dtype)
    y = x[:, front:front + heads * dim].reshape(rows, heads, dim)
    want, sizes = turn(y, at, f, float(np.float32(amplitude)), rot, first, halves)
    got = got[:, lo:lo + heads * dim].reshape(rows, heads, dim)
    keep = torch.cat([torch.arange(first), torch.arange(first + rot, dim)])
    assert same_bits(got[..., keep], y[..., keep], dtype)
    close(got, want, turn_tolerance(want, sizes, dtype))


def test_rotary_keeps_special_values_outside_the_turned_part(dev):
    x = torch.tensor([[math.nan, math.inf, 1.0, 2.0, -math.inf, -0.0, 3.0, math.nan]]).to(torch.float16)
    b, f = dev.up(x), dev.up(np.ones(1, np.float32))
    dev.K.rotary_rows_into(dev.batch(), b, b, dev.pkg.F16, dev.up(np.zeros(1, np.uint32)), f, 1.0, 1, 1, 8, 2, 2, dev.pkg.ROTARY_PAIRS, 8, 8)
    assert same_bits(dev.down(b, (1, 8), "f16"), x, "f16")


# ---- appending --------------------------------------------------------------------------------------------------------------
APPEND = [  # sequences (rows, length), page, heads, kv heads, dim, rot, first, halves
    ([(1, 1)], 16, 4, 1, 128, 128, 0, True),
    ([(1, 33), (1, 16), (1, 17), (0, 5), (1, 1)], 16, 8, 2, 128, 128, 0, True),
    ([(40, 40), (0, 0), (17, 100), (1, 64)], 32, 6, 3, 80, 50, 30, False),
    ([(5, 3), (3, 3), (2, 0), (70, 71)], 16, 2, 2, 33, 10, 5, True),          # more rows than positions
    ([(300, 700)], 64, 0, 4, 64, 0, 0, False),
    ([(2, 2)] * 70 + [(0, 9)] * 70 + [(3, 40)] * 5, 16, 4, 4, 64, 64, 0, True),
    ([(4200, 4300), (1, 5)], 128, 2, 1, 256, 64, 192, True),
    ([(9, 1030)], 1024, 3, 1, 192, 100, 92, False),
]


def run_append(dev, step, dtype, heads, G, dim, rot, first, halves, seed, inplace=False, keys=None, values=None, stacked=True, starts=None, lengths=None, table=None, rows=None):
    """-> (inputs, results): the pools before, q, k, v; the pools and q after."""
    pkg, K = dev.pkg, dev.K
    rows = step.rows + 2 if rows is None else rows                # two rows of no sequence
    D, size = padded(dim), 4 if dtype == "f32" else 2
    shape = (step.pages, G, step.page, D)
    keys = normal(seed, *shape, dtype=dtype) if keys is None else keys
    values = normal(seed + 1, *shape, dtype=dtype) if values is None else values
    qkv = normal(seed + 2, rows, (heads + 2 * G) * dim, dtype=dtype)
    q, k, v = (x.reshape(rows, -1, dim) for x in qkv.split([heads * dim, G * dim, G * dim], 1))
    f = K.rotary_frequencies(max(rot, 2), 1e4)[0]
    bk, bv = dev.up(keys), dev.up(values)
    ld = qkv.shape[1]
    whole = dev.up(qkv)
    parts = [whole.view(o * dim * size, whole.length() - o * dim * size) for o in (0, heads, heads + G)]
    marked = torch.full((rows, heads * dim), 7.0).to(TYPES[dtype])
    out = parts[0] if inplace else dev.up(marked)
    K.paged_append_into(dev.batch(), parts[1], parts[2], code(pkg, dtype), bk, bv, dev.up(step.table if table is None else table),
                        dev.up(step.starts if starts is None else starts), dev.up(step.lengths if lengths is None else lengths), rows, len(step.sequences), G, dim, step.pages,
                        step.page, step.table.shape[1], ld, ld, dev.up(f) if rot else None, 1.1, rot, first, pkg.ROTARY_HALVES if halves else pkg.ROTARY_PAIRS,
                        parts[0] if heads else None, out if heads else None, heads, ld, ld if inplace else heads * dim)
    got_q = None
    if heads:
        got_q = dev.down(whole, (rows, ld), dtype)[:, :heads * dim].reshape(rows, heads, dim) if inplace else dev.down(out, (rows, heads, dim), dtype)
        if inplace:
            assert same_bits(dev.down(whole, (rows, ld), dtype)[:, heads * dim:], qkv[:, heads * dim:], dtype)
    return (keys, values, q if heads else None, k, v, f, q if inplace else marked.reshape(rows, heads, dim)), (dev.down(bk, shape, dtype), dev.down(bv, shape, dtype), got_q)


def check_append(step, dtype, rot, first, halves, before, after):
    keys, values, q, k, v, f, qwas = before
    wk, wv, wq, sk, sq = appended(step, k, v, keys, values, q, f, float(np.float32(1.1)), rot, first, halves)
    assert bool((after[1].to(F64) == wv).all())                    # values, and every slot that no row went to, as they were
    touched = wk != keys.to(F64)
    assert bool((after[0].to(F64) == keys.to(F64))[~touched & (sk == 0)].all())
    close(after[0], wk, turn_tolerance(wk, sk, dtype), "keys")
    if q is not None:
        left = wq.isnan()
        assert same_bits(after[2][left], qwas[left], dtype)
        close(after[2][~left], wq[~left], turn_tolerance(wq, sq, dtype)[~left], "queries")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append(dev, dtype, case):
    seqs, page, heads, G, dim, rot, first, halves = APPEND[case]
    step = Step(seqs, page, seed=case)
    check_append(step, dtype, rot, first, halves, *run_append(dev, step, dtype, heads, G, dim, rot, first, halves, case, inplace=case % 2 == 1 and heads > 0))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_append_drops_what_has_no_page(dev, dtype):
    step = Step([(20, 40), (3, 30), (2, 16)], 16, seed=3, table_extra=0)
    step.table[0, 1] = step.pages                                  # a page that the pool does not have
    step.table[1, 1] = NO_PAGE
    check_append(step, dtype, 64, 0, True, *run_append(dev, step, dtype, 2, 1, 64, 64, 0, True, 5))
    step = Step([(20, 40), (3, 30)], 16, seed=4)
    short = np.ascontiguousarray(step.table[:, :2])                # position 32 and on of the first sequence are not in the table
    step.table = short
    check_append(step, dtype, 64, 0, True, *run_append(dev, step, dtype, 2, 1, 64, 64, 0, True, 6))


def test_append_of_a_length_beyond_every_table(dev):
    step = Step([(3, 40), (4, 20)], 16, seed=4)
    step.sequences[0] = (3, 0xFFFFFFFF)
    step.lengths[0] = 0xFFFFFFFF
    check_append(step, "bf16", 64, 0, True, *run_append(dev, step, "bf16", 2, 1, 64, 64, 0, True, 6))


def test_append_of_a_sequence_that_ends_behind_the_rows_leaves_everything(dev):
    step = Step([(4, 10), (6, 10)], 16, seed=5)
    before, after = run_append(dev, step, "bf16", 2, 1, 64, 64, 0, True, 7, rows=9)     # row 9 is not there: the second sequence has none
    step.sequences[1] = (0, 10)
    step.starts[2] = step.starts[1]
    check_append(step, "bf16", 64, 0, True, before, after)


# ---- attention ----------------------------------------------------------------------------------------------------------------
def run_attention(dev, step, dtype, heads, G, dim, window=0, sink=False, seed=0, scale=None, q_ld=0, lead=0, out_ld=0, max_length=None, max_rows=None, keys=None, values=None,
                  rows=None, spread=1.0):
    pkg, K = dev.pkg, dev.K
    rows = step.rows + 2 if rows is None else rows
    D, scale = padded(dim), dim ** -0.5 if scale is None else scale
    shape = (step.pages, G, step.page, D)
    keys = (normal(seed, *shape) * spread).to(TYPES[dtype]) if keys is None else keys
    values = normal(seed + 1, *shape, dtype=dtype) if values is None else values
    keys[..., dim:], values[..., dim:] = 0, 0                      # as an append leaves them
    q_ld, out_ld = q_ld or heads * dim, out_ld or heads * dim
    q = normal(seed + 2, rows, q_ld, dtype=dtype)
    s = normal(seed + 3, heads) if sink else None
    marked = torch.full((rows, out_ld), 7.0).to(TYPES[dtype])
    out = dev.up(marked, lead)
    ml, mr = step.max_length if max_length is None else max_length, step.max_rows if max_rows is None else max_rows
    need = K.paged_attention_workspace_bytes(rows, len(step.sequences), mr, ml, heads, G, dim)
    whole, mark = pkg.Buffer.empty(dev.ctx, need + 256), np.arange(256, dtype=np.uint8)
    work, behind = whole.view(0, max(need, 16)), whole.view(need, 256)
    dev.batch().write(behind, mark)
    K.paged_attention_into(dev.batch(), dev.up(q, lead), dev.up(keys), dev.up(values), out, code(pkg, dtype), dev.up(step.table), dev.up(step.starts), dev.up(step.lengths), rows,
                           len(step.sequences), mr, ml, heads, G, dim, step.pages, step.page, step.table.shape[1], q_ld, out_ld, scale, window,
                           dev.up(s) if sink else None, work if need else None)
    got = dev.down(out, (rows, out_ld), dtype)
    assert same_bits(got[:, heads * dim:], marked[:, heads * dim:], dtype)
    assert bool((behind.as_array(np.uint8, 256) == mark).all())
    got = got[:, :heads * dim].reshape(rows, heads, dim)
    q = q[:, :heads * dim].reshape(rows, heads, dim)
    want, tol = attended(step, q, keys, values, float(np.float32(scale)), window, s, max_length, max_rows)
    left = want.isnan().all(2).all(1)
    left[int(step.starts[-1]):] = True
    assert same_bits(got[left], marked[left][:, :heads * dim].reshape(-1, heads, dim), dtype)
    close(got[~left], want[~left], (half_step(dtype) * want.abs() + tol + (2.0 ** -25 if dtype == "f16" else 0))[~left], (step.sequences[:4], window))
    return got, want


ATTENTION = [  # sequences (rows, length), page, heads, kv heads, dim, window, sink
    ([(1, 1)], 16, 4, 1, 128, 0, False),
    ([(1, 1), (1, 2), (1, 15), (1, 16), (1, 17), (1, 31), (1, 32), (1, 33)], 16, 8, 2, 64, 0, False),
    ([(1, 300), (1, 4), (0, 50), (1, 129)], 32, 8, 8, 32, 0, True),                  # a head a group
    ([(40, 40), (17, 100), (1, 64), (5, 5)], 16, 6, 2, 80, 0, False),
    ([(7, 200), (1, 1000), (33, 34)], 64, 5, 1, 33, 50, True),
    ([(1, 2100)], 16, 24, 1, 128, 0, False),                                         # more heads than a tile has rows
    ([(3, 1500), (1, 900)], 128, 16, 4, 256, 0, False),
    ([(70, 70)], 16, 3, 3, 192, 1, False),                                           # a row sees itself
    ([(130, 515)], 1024, 4, 2, 160, 17, False),
    ([(1, 9)] * 70 + [(0, 3)] * 3 + [(2, 77)] * 67, 16, 4, 2, 64, 0, False),
    ([(5, 3), (3, 3), (2, 0), (1, 1)], 16, 2, 2, 128, 0, True),                      # rows that stand nowhere see nothing
    ([(260, 1000), (1, 700), (300, 300)], 32, 8, 1, 128, 0, False),
    ([(129, 4000)], 64, 4, 4, 64, 1000, False),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_attention(dev, dtype, case):
    seqs, page, heads, G, dim, window, sink = ATTENTION[case]
    run_attention(dev, Step(seqs, page, seed=case), dtype, heads, G, dim, window, sink, seed=case, spread=1.0 + 2.0 * (case % 2))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,G,dim,window", [(32, 8, 64, 0), (32, 8, 128, 0), (16, 8, 32, 300), (32, 8, 192, 0), (16, 8, 250, 0)])
def test_attention_of_more_tiles_than_the_chip_has_units(dev, dtype, heads, G, dim, window):
    run_attention(dev, Step([(640, 820), (90, 90), (1, 300), (37, 512)], 16, seed=dim), dtype, heads, G, dim, window, seed=dim)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 128, 192, 256])
@pytest.mark.parametrize("rows,window,sink", [(1, 0, True), (20, 0, False), (20, 2900, True)])
def test_attention_over_long_caches_in_many_parts(dev, dtype, dim, rows, window, sink):
    run_attention(dev, Step([(rows, 6000), (1, 40), (rows, 2000)], 64, seed=dim), dtype, 8, 2, dim, window, sink, seed=dim, spread=3.0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_of_many_tokens_over_long_caches(dev, dtype):
    """More than eight parts of rows that fill the chip; the sequences hold the same pages, to different lengths."""
    lengths = [17000 - 13 * i for i in range(40)]
    step = Step([(1, n) for n in lengths], 128, seed=1)
    own = step.table[0].copy()
    step.table[:] = own
    rank = {int(p): i for i, p in enumerate(sorted(int(p) for p in own if p != NO_PAGE))}
    step.pages = len(rank)
    step.table = np.vectorize(lambda p: rank.get(int(p), NO_PAGE))(step.table).astype(np.uint32)
    run_attention(dev, step, dtype, 8, 8, 32, seed=4)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 40])
def test_attention_of_many_small_weights_beside_a_large_one(dev, dtype, rows):
    """One position with nearly all the weight, as a sequence's first often has, and thousands with 1e-5 of it each: together they weigh as much as it does when
    there are enough of them, and below f16's normal numbers all would be off the same way.

    A weight 2^-16.6 of the largest is rounded to a step of it, also where that has 16 bits: half_step of it, which the tolerance has."""
    length, dim, G = 20000, 64, 2
    step = Step([(rows, length)], 128, seed=3)
    shape = (step.pages, G, 128, 64)
    keys, values = torch.zeros(shape, dtype=TYPES[dtype]), normal(4, *shape, dtype=dtype).abs()
    keys[..., 0] = -1.0
    keys[int(step.table[0, 0]), :, 0, 0] = 10.5
    values[int(step.table[0, 0]), :, 0] = -1.0
    pkg, K = dev.pkg, dev.K
    q = torch.zeros(rows, 4, dim, dtype=TYPES[dtype])
    q[..., 0] = 1.0
    out = pkg.Buffer.empty(dev.ctx, q.numel() * q.element_size())
    need = K.paged_attention_workspace_bytes(rows, 1, rows, length, 4, G, dim)
    K.paged_attention_into(dev.batch(), dev.up(q), dev.up(keys), dev.up(values), out, code(pkg, dtype), dev.up(step.table), dev.up(step.starts), dev.up(step.lengths), rows, 1, rows,
                           length, 4, G, dim, step.pages, 128, step.table.shape[1], 4 * dim, 4 * dim, 1.0, 0, None, pkg.Buffer.empty(dev.ctx, max(need, 16)))
    want, tol = attended(step, q, keys, values, 1.0)
    assert 0.1 < float(1 / (1 + (length - rows) * math.exp(-11.5))) < 0.9
    close(dev.down(out, q.shape, dtype), want, half_step(dtype) * want.abs() + tol + (2.0 ** -25 if dtype == "f16" else 0))


def test_attention_of_a_thousand_sequences(dev):
    run_attention(dev, Step([(i % 2, 1 + i % 37) for i in range(1000)] + [(3, 40)], 16, seed=1), "bf16", 4, 2, 64, seed=3)
    run_attention(dev, Step([(i % 3, 2 + i % 37) for i in range(300)] + [(60, 200)], 16, seed=1), "f16", 4, 2, 64, seed=3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 70])
def test_attention_of_lengths_beyond_everything(dev, dtype, rows):
    """A length that no table reaches: the row sees what the table has."""
    step = Step([(rows, 200), (1, 50)], 16, seed=3, table_extra=0)
    step.sequences[0] = (rows, 0xFFFFFFFF)
    step.lengths[0], step.max_length = 0xFFFFFFFF, 1 << 20
    run_attention(dev, step, dtype, 4, 2, 64, seed=2)
    step = Step([(rows, 200), (1, 50)], 16, seed=3)
    step.sequences[0] = (rows, 0xFFFFFFFF)
    step.lengths[0], step.max_length = 0xFFFFFFFF, 170
    run_attention(dev, step, dtype, 4, 2, 64, window=1 << 31, seed=2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,lead,pad", [(64, 4, 0), (80, 0, 3), (50, 2, 1), (128, 0, 8)])
def test_attention_of_rows_at_odd_places(dev, dtype, dim, lead, pad):
    lead = lead if dtype != "f32" else lead // 4 * 4
    run_attention(dev, Step([(19, 60), (1, 400)], 16, seed=1), dtype, 4, 2, dim, seed=dim, q_ld=4 * dim + pad, out_ld=4 * dim + 2 * pad, lead=lead)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 90])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_attention_scales(dev, dtype, rows, scale):
    run_attention(dev, Step([(rows, 350)], 16, seed=2), dtype, 4, 2, 64, scale=scale, seed=9)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 60])
@pytest.mark.parametrize("window,length", [(0, 333), (100, 333), (0, 3300), (2000, 3300)])
def test_attention_does_not_see_what_is_masked(dev, dtype, rows, window, length):
    """NaN and infinities in slots behind a sequence's end, in front of its window, on pages of nobody -- and at positions that some rows see
    and others do not, where only the rows that see them may have them."""
    step = Step([(rows, length), (rows, 64), (1, 30)], 32, seed=6)
    G, dim = 2, 128
    shape = (step.pages, G, step.page, 128)
    keys, values = normal(1, *shape, dtype=dtype), normal(2, *shape, dtype=dtype)
    mine = torch.zeros(shape[0], shape[2], dtype=torch.bool)
    for s, (n, end) in enumerate(step.sequences):
        for p in range(max(0, end - n + 1 - window) if window else 0, end):
            mine[int(step.table[s, p // 32]), p % 32] = True
    for x, bad in ((keys, math.nan), (values, math.nan)):
        x.permute(0, 2, 1, 3)[~mine] = bad
    last = int(step.table[0, (length - 1) // 32]), (length - 1) % 32                 # the first sequence's last position: its last row alone sees it
    values[last[0], 0, last[1], 3] = math.inf
    values[last[0], 1, last[1], 5] = math.nan
    keys[int(step.table[1, 63 // 32]), 0, 63 % 32] = math.nan
    got, want = run_attention(dev, step, dtype, 4, G, dim, window, seed=8, keys=keys, values=values)
    r = int(step.starts[1]) - 1
    assert got[r, 0, 3] == math.inf and got[r, 2, 5].isnan() and got[r, 0, 5].isfinite()
    assert bool(got[:r].isfinite().all()) and bool(got[int(step.starts[2]) - 1, :2].isnan().all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 50])
def test_attention_of_pages_that_are_not_there(dev, dtype, rows):
    """A page index that the pool does not have, positions that the table does not reach, lengths and rows beyond the bounds."""
    step = Step([(rows, 200), (rows, 150), (rows, 300)], 16, seed=7)
    step.table[0, 3], step.table[0, 12], step.table[1, 0], step.table[2, :] = step.pages, NO_PAGE, 0xFFFFFFF0, NO_PAGE
    run_attention(dev, step, dtype, 4, 2, 64, seed=3)
    step = Step([(rows, 200), (rows, 90)], 16, seed=8)
    step.table = np.ascontiguousarray(step.table[:, :7])
    run_attention(dev, step, dtype, 4, 2, 64, seed=4)
    run_attention(dev, Step([(rows, 200), (rows, 90)], 16, seed=8), dtype, 4, 2, 64, seed=5, max_length=120)
    run_attention(dev, Step([(rows, 200), (3, 90)], 16, seed=8), dtype, 4, 2, 64, seed=6, max_rows=1)
    run_attention(dev, Step([(rows, 200), (3, 90)], 16, seed=8), dtype, 4, 2, 64, seed=6, max_length=0)


def test_attention_of_shared_pages_and_one_sequence_twice(dev):
    step = Step([(1, 100), (1, 100), (20, 120)], 16, seed=9)
    step.table[1] = step.table[0]
    step.table[2, :6] = step.table[0, :6]
    run_attention(dev, step, "bf16", 8, 2, 128, seed=10)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_of_sequences_with_and_without_a_common_beginning(dev, dtype, dim):
    """Caches that may be long, whose sequences share all, some or none of their pages with the ones beside them."""
    step = Step([(1, 3000), (1, 3000), (2, 2900), (0, 500), (1, 2600), (1, 40), (1, 0), (1, 1300)], 32, seed=dim)
    step.table[1, :60] = step.table[0, :60]
    step.table[2, :] = step.table[1, :]
    step.table[3, :] = step.table[4, :]
    step.table[4, 7] = NO_PAGE
    run_attention(dev, step, dtype, 8, 2, dim, seed=dim, max_length=40000)
    run_attention(dev, step, dtype, 8, 2, dim, 700, True, seed=dim + 1, max_length=40000)


BOUNDS = [  # sequences (rows, length), page, heads, kv heads, dim, window
    ([(1, 9000)] + [(1, 30 + i) for i in range(70)], 64, 8, 2, 64, 0),               # one long among many short ones
    ([(1, 700)] * 3, 16, 4, 4, 128, 0),
    ([(60, 5000), (60, 60), (1, 2000), (3, 3)], 32, 8, 2, 64, 0),
    ([(200, 200)] * 20 + [(130, 3000)], 32, 8, 8, 32, 0),                             # tiles that fill the chip
    ([(5, 4000)] * 9, 64, 6, 2, 192, 1500),
    ([(1, 40)] * 300, 16, 16, 16, 32, 0),                                             # more units than workgroups are wanted
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(BOUNDS)))
@pytest.mark.parametrize("bound", [1, 9, 300])
def test_attention_of_a_call_for_longer_sequences(dev, dtype, case, bound):
    """How sequences are cut goes by what they have, not by what the call allows."""
    seqs, page, heads, G, dim, window = BOUNDS[case]
    step = Step(seqs, page, seed=case)
    run_attention(dev, step, dtype, heads, G, dim, window, sink=case % 2 == 1, seed=case, max_length=step.max_length * bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 60])
def test_attention_of_starts_that_do_not_ascend(dev, dtype, rows):
    """What such a step computes is not said, but it stays inside its buffers: more tiles and parts than the rows can have are left out."""
    pkg, K = dev.pkg, dev.K
    n, G, D, page, length = 40, 2, 64, 64, 6000
    step = Step([(rows, length)], page, seed=rows)
    table, lengths = np.repeat(step.table, n, 0), np.full(n, length, np.uint32)
    starts = np.zeros(n + 1, np.uint32)
    starts[1::2] = rows                                            # every other sequence has all the rows
    keys, values = (dev.up(normal(i, step.pages, G, page, D, dtype=dtype)) for i in range(2))
    q, marked = normal(2, rows, 8 * D, dtype=dtype), torch.full((rows + 1, 8 * D), 7.0).to(TYPES[dtype])
    need = K.paged_attention_workspace_bytes(rows, n, rows, length, 8, G, D)
    whole, mark, out = pkg.Buffer.empty(dev.ctx, need + 256), np.arange(256, dtype=np.uint8), dev.up(marked)
    dev.batch().write(whole.view(need, 256), mark)
    K.paged_attention_into(dev.batch(), dev.up(q), keys, values, out, code(pkg, dtype), dev.up(table), dev.up(starts), dev.up(lengths), rows, n, rows, length, 8, G, D,
                           step.pages, page, table.shape[1], 8 * D, 8 * D, 0.1, 0, None, whole.view(0, need))
    got = dev.down(out, (rows + 1, 8 * D), dtype)
    assert same_bits(got[rows:], marked[rows:], dtype)
    assert bool((whole.view(need, 256).as_array(np.uint8, 256) == mark).all())


def test_attention_of_no_sequence_and_of_one_that_ends_behind_the_rows(dev):
    step = Step([(0, 10), (0, 0)], 16, seed=1)
    run_attention(dev, step, "bf16", 4, 2, 64, rows=3)
    step = Step([(4, 10), (6, 10)], 16, seed=5)
    starts = step.starts.copy()
    step.sequences[1], step.starts[2] = (0, 10), step.starts[1]
    good = step.starts
    step.starts = starts
    try:
        run_attention(dev, step, "bf16", 2, 1, 64, rows=9, seed=2)
    finally:
        step.starts = good


def test_pools_larger_than_32_bits_reach(dev):
    """Pages whose values stand beyond 2^32 values, a table whose last pages are the pool's."""
    pkg, K = dev.pkg, dev.K
    G, dim, page = 8, 256, 128
    pages = (1 << 32) // (G * dim * page) + 8
    keys, values = (pkg.Buffer.empty(dev.ctx, pages * G * page * dim * 2) for _ in range(2))
    step = Step([(200, 200), (1, 90)], page, seed=1)
    step.table = np.where(step.table == NO_PAGE, NO_PAGE, pages - 1 - step.table).astype(np.uint32)
    own = sorted(int(p) for p in step.table.reshape(-1) if p != NO_PAGE)
    k, v, q = (normal(i, step.rows, n, dim, dtype="bf16") for i, n in ((1, G), (2, G), (3, 2 * G)))
    f = K.rotary_frequencies(dim, 1e4)[0]
    bq, out = dev.up(q), pkg.Buffer.empty(dev.ctx, q.numel() * 2)
    plan = [dev.up(x) for x in (step.table, step.starts, step.lengths)]
    for n in (1, 0):                                                # the second sequence's earlier positions, then the step
        first = Step([(0, 200), (89, 89)], page) if n else step
        kk, vv = (normal(4 + i, 89, G, dim, dtype="bf16") for i in range(2)) if n else (k, v)
        K.paged_append_into(dev.batch(), dev.up(kk), dev.up(vv), pkg.BF16, keys, values, plan[0], dev.up(first.starts), dev.up(first.lengths), first.rows, 2, G, dim, pages, page,
                            step.table.shape[1], G * dim, G * dim, dev.up(f), 1.0, dim, 0, pkg.ROTARY_HALVES, None if n else bq, None if n else bq, 0 if n else 2 * G, 2 * G * dim,
                            2 * G * dim)
    need = K.paged_attention_workspace_bytes(step.rows, 2, 200, 200, 2 * G, G, dim)
    K.paged_attention_into(dev.batch(), bq, keys, values, out, pkg.BF16, *plan, step.rows, 2, 200, 200, 2 * G, G, dim, pages, page, step.table.shape[1], 2 * G * dim, 2 * G * dim,
                           1 / 16, 0, None, pkg.Buffer.empty(dev.ctx, need) if need else None)
    n = G * page * dim * 2
    pool = [torch.stack([dev.down(b.view(p * n, n), (G, page, dim), "bf16") for p in own]) for b in (keys, values)]
    step.pages, step.table = len(own), np.where(step.table == NO_PAGE, NO_PAGE, step.table - np.uint32(own[0])).astype(np.uint32)
    remap = {p - own[0]: i for i, p in enumerate(own)}
    step.table = np.vectorize(lambda p: remap.get(int(p), NO_PAGE))(step.table).astype(np.uint32)
    want, sizes = turn(k[:200], np.arange(200), f, 1.0, dim, 0, True)
    at = torch.arange(200)
    stored = pool[0][torch.as_tensor(step.table[0].astype(np.int64))[at // page], :, at % page]
    close(stored, want, turn_tolerance(want, sizes, "bf16"), "keys")
    got_q = dev.down(bq, q.shape, "bf16")
    want, tol = attended(step, got_q, *pool, 1 / 16)
    close(dev.down(out, q.shape, "bf16"), want, half_step("bf16") * want.abs() + tol)


# ---- as they are used ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
def test_sequences_that_come_and_go_through_the_cache(dev, dtype):
    """Prompts in chunks, tokens beside them, a sequence that shares another's beginning, one that ends and whose pages serve the next: every
    step's outputs against attention over all that the sequence was given, turned in 64 bits from the start."""
    from local_ai_amd import kv_cache as kv
    pkg, K = dev.pkg, dev.K
    H, G, dim, page, S = 8, 2, 64, 16, 3
    tables = kv.PageTables(14, page, S, 160)
    cache = kv.PagedKvCache(dev.ctx, K, G, dim, 14, page, code(pkg, dtype))
    step = kv.PagedStep(dev.ctx, tables, 90, 64, 160)
    f, _ = K.rotary_frequencies(dim, 1e4)
    rotary = kv.Rotary(dev.up(f), dim)
    work = pkg.Buffer.empty(dev.ctx, max(cache.workspace_bytes(K, step, H), 16))
    told = [[] for _ in range(S)]                                   # (k, v) of every position
    size = 4 if dtype == "f32" else 2

    def run(counts, seed):
        lengths = [len(t) + n for t, n in zip(told, counts)]
        for s, (n, length) in enumerate(zip(counts, lengths)):
            if n:
                tables.reserve(s, length)
        x = normal(seed, 90, (H + 2 * G) * dim, dtype=dtype)
        qkv, out, batch = dev.up(x), pkg.Buffer.empty(dev.ctx, 90 * H * dim * size), dev.batch()
        step.write(batch, counts, lengths)
        q, k, v = (qkv.view(o * dim * size, qkv.length() - o * dim * size) for o in (0, H, H + G))
        ld = x.shape[1]
        cache.append_into(batch, K, step, k, v, ld, ld, rotary, q, q, H, ld, ld)
        cache.attention_into(batch, K, step, q, out, H, dim ** -0.5, work, q_ld=ld)
        batch.commit_and_wait()
        got, row = dev.down(out, (90, H, dim), dtype), 0
        heads = x.reshape(90, H + 2 * G, dim)
        for s, n in enumerate(counts):
            told[s] += [(heads[row + i, H:H + G], heads[row + i, H + G:]) for i in range(n)]
            if n == 0:
                continue
            length = len(told[s])
            ks, vs = (torch.stack([t[i] for t in told[s]]) for i in range(2))
            kt, _ = turn(ks, np.arange(length), f, 1.0, dim, 0, True)
            qt, _ = turn(heads[row:row + n, :H], np.arange(length - n, length), f, 1.0, dim, 0, True)
            kt, qt = kt.to(TYPES[dtype]), qt.to(TYPES[dtype])
            one = Step([(n, length)], page, seed=1)
            pool = torch.zeros(2, one.pages, G, page, dim, dtype=TYPES[dtype])
            at = torch.arange(length)
            pg = torch.as_tensor(one.table[0].astype(np.int64))[at // page]
            pool[0, pg, :, at % page], pool[1, pg, :, at % page] = kt, vs
            want, tol = attended(one, qt, pool[0], pool[1], dim ** -0.5)
            # a turned value may fall to either side where it is rounded: a step of q and of k in every score, twice half a step each, relative to
            # the products' absolute sum, which the tolerance of a score has (dim + 8) 2^-24 of
            tol = tol * (1 + (4 * half_step(dtype) / ((dim + 8) * 2.0 ** -24) if dtype != "f32" else 2))
            close(got[row:row + n], want, half_step(dtype) * want.abs() + tol, (s, n))
            row += n

    run([40, 0, 0], 1)
    run([24, 64, 0], 2)
    run([1, 1, 0], 3)
    shared = tables.share(0, 2, len(told[0]))
    assert shared == 64
    told[2] = told[0][:shared]
    run([1, 1, 5], 4)
    run([0, 1, 1], 5)
    tables.release(1)
    told[1] = []
    run([1, 33, 1], 6)
    tables.release(0)
    told[0] = []
    run([17, 1, 20], 7)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 40])
def test_a_recorded_step_follows_its_plan(dev, dtype, rows):
    """Append and attention recorded once for the largest lengths and replayed as the sequences grow, two graphs over one workspace in turn, with
    work of its own between them: every replay as the calls made one by one."""
    pkg, K = dev.pkg, dev.K
    H, G, dim, page, size = 8, 2, 128, 16, 4 if dtype == "f32" else 2
    step = Step([(rows, 1500), (rows, 700)], page, seed=2)
    n, ld = step.rows, (H + 2 * G) * dim
    f = dev.up(K.rotary_frequencies(dim, 1e4)[0])
    shape = (step.pages, G, page, dim)
    need = K.paged_attention_workspace_bytes(n, 2, rows, 1500, H, G, dim)
    work = pkg.Buffer.empty(dev.ctx, max(need, 16))

    class Stream:
        def __init__(self, seed):
            self.pools = [dev.up(normal(seed + i, *shape, dtype=dtype)) for i in range(2)]
            self.twin = [dev.up(normal(seed + i, *shape, dtype=dtype)) for i in range(2)]
            self.qkv, self.lengths = pkg.Buffer.empty(dev.ctx, n * ld * size), pkg.Buffer.empty(dev.ctx, 8)
            self.table, self.starts = dev.up(step.table), dev.up(step.starts)
            self.out, self.other = (pkg.Buffer.empty(dev.ctx, n * H * dim * size) for _ in range(2))

        def encode(self, batch, pools, out):
            q, k, v = (self.qkv.view(o * dim * size, self.qkv.length() - o * dim * size) for o in (0, H, H + G))
            K.paged_append_into(batch, k, v, code(pkg, dtype), *pools, self.table, self.starts, self.lengths, n, 2, G, dim, step.pages, page, step.table.shape[1], ld, ld, f, 1.0, dim,
                                0, pkg.ROTARY_HALVES, q, out, H, ld, H * dim)
            K.paged_attention_into(batch, out, *pools, self.other, code(pkg, dtype), self.table, self.starts, self.lengths, n, 2, rows, 1500, H, G, dim, step.pages, page,
                                   step.table.shape[1], H * dim, H * dim, dim ** -0.5, 0, None, work if need else None)

        def feed(self, seed, lengths):
            self.qkv.copy_from_bytes(raw(normal(seed, n, ld, dtype=dtype)))
            self.lengths.copy_from_bytes(np.asarray(lengths, np.uint32))

    streams, graphs = [Stream(10), Stream(20)], []
    for s in streams:
        s.feed(1, [rows, rows])
        for pools in (s.pools, s.twin):                             # once unrecorded: kernels are set up
            s.encode(dev.batch(), pools, s.out)
        batch = dev.batch()
        batch.begin_capture()
        s.encode(batch, s.pools, s.out)
        graphs.append(batch.end_capture())
    for i, lengths in enumerate([[rows, rows + 3], [500, 200], [1500, 700], [33, 699], [1499, rows]]):
        for j, (s, graph) in enumerate(zip(streams, graphs)):
            s.feed(100 + 10 * i + j, lengths)
            graph.launch()
            dev.batch().commit_and_wait()
            got, turned = (dev.down(b, (n, H, dim), dtype) for b in (s.other, s.out))
            s.encode(dev.batch(), s.twin, s.out)
            dev.batch().commit_and_wait()
            assert same_bits(got, dev.down(s.other, (n, H, dim), dtype), dtype) and same_bits(turned, dev.down(s.out, (n, H, dim), dtype), dtype)
            for a, b in zip(s.pools, s.twin):
                assert same_bits(dev.down(a, shape, dtype), dev.down(b, shape, dtype), dtype)


# ---- values that are seen, however little they weigh ---------------------------------------------------------------------------
def attention_of(dev, step, q, keys, values, dtype, scale, window=0, sink=None, max_length=None):
    pkg, K = dev.pkg, dev.K
    rows, H, dim = q.shape
    G, ml = keys.shape[1], step.max_length if max_length is None else max_length
    out = pkg.Buffer.empty(dev.ctx, q.numel() * q.element_size())
    need = K.paged_attention_workspace_bytes(rows, len(step.sequences), step.max_rows, ml, H, G, dim)
    K.paged_attention_into(dev.batch(), dev.up(q), dev.up(keys), dev.up(values), out, code(pkg, dtype), dev.up(step.table), dev.up(step.starts), dev.up(step.lengths), rows,
                           len(step.sequences), step.max_rows, ml, H, G, dim, step.pages, step.page, step.table.shape[1], H * dim, H * dim, scale, window,
                           None if sink is None else dev.up(sink), pkg.Buffer.empty(dev.ctx, max(need, 16)))
    return dev.down(out, q.shape, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("length,at", [(400, 20), (400, 300), (6000, 20), (6000, 150), (6000, 3000), (6000, 5900)])
@pytest.mark.parametrize("weight", ["key", "sink", "none"])
def test_a_nan_that_a_row_sees_reaches_it(dev, dtype, rows, length, at, weight):
    """A NaN among the values of a position beside which another (or the sink) weighs 2^230 times as much, or whose score is minus infinity as those of all positions near
    it are: 0 times NaN is NaN, whichever wave or part has the position.

    Tolerance: a weight below 2^-126 may be 0, which 6000 of them times values of at most 5 make less than 2^-110 of."""
    G, dim = 2, 64
    step = Step([(rows, length)], 32, seed=length)
    shape = (step.pages, G, 32, dim)
    keys, values = torch.zeros(shape, dtype=TYPES[dtype]), normal(1, *shape, dtype=dtype)

    def place(p):
        return int(step.table[0, p // 32]), p % 32
    sink = torch.full((4,), 160.0) if weight == "sink" else None
    if weight == "key":
        keys[place(5)[0], :, place(5)[1], 0] = 160.0
    if weight == "none":
        keys[..., 0] = -math.inf
        keys[place(5)[0], :, place(5)[1], 0] = 0.0
    values[place(at)[0], 1, place(at)[1], 7] = math.nan
    q = torch.zeros(rows, 4, dim, dtype=TYPES[dtype])
    q[..., 0] = 1.0
    got = attention_of(dev, step, q, keys, values, dtype, 1.0, sink=sink)
    want, tol = attended(step, q, keys, values, 1.0, sink=sink)
    assert bool(want[:, 2:, 7].isnan().all()) and int(want.isnan().sum()) == 2 * rows
    if weight == "none":                                           # (one position has all the weight: 1, exactly)
        tol = torch.zeros_like(tol)
    close(got, want, half_step(dtype) * want.abs() + tol + (2.0 ** -25 if dtype == "f16" else 2.0 ** -110))


def test_what_is_read_may_stand_between_the_rows_of_an_output(dev):
    """One allocation: rows of 64 values, 128 apart, with the frequencies behind the first and the positions behind the second."""
    pkg, K = dev.pkg, dev.K
    rows, ld = 3, 128
    x, f, at = normal(1, rows, 64), K.rotary_frequencies(64, 1e4)[0], np.asarray([7, 100, 3000], np.uint32)
    whole = torch.full((rows, ld), 7.0)
    whole[0, 64:96], whole[1, 64:67] = torch.from_numpy(f), torch.from_numpy(at.view(np.float32))
    b = dev.up(whole)
    K.rotary_rows_into(dev.batch(), dev.up(x), b, pkg.F32, b.view(4 * (ld + 64), 12), b.view(4 * 64, 128), 1.0, rows, 1, 64, 64, 0, pkg.ROTARY_HALVES, 64, ld)
    got = dev.down(b, (rows, ld), "f32")
    want, sizes = turn(x.reshape(rows, 1, 64), at, f, 1.0, 64, 0, True)
    close(got[:, :64].reshape(rows, 1, 64), want, turn_tolerance(want, sizes, "f32"))
    assert same_bits(got[:, 64:], whole[:, 64:], "f32")


# ---- as they are used, from what is stored ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
def test_a_session_against_what_its_pages_hold(dev, dtype):
    """Prompts in chunks, tokens beside them, a shared beginning, sequences that end and whose pages serve the next.  The turned queries and the pages are read back:
    keys and queries against 64 bits by the tolerance of a turn, outputs against attention over what stands there, by its own."""
    from local_ai_amd import kv_cache as kv
    pkg, K = dev.pkg, dev.K
    H, G, dim, page, S, rows = 8, 2, 64, 16, 3, 90
    tables = kv.PageTables(14, page, S, 160)
    cache = kv.PagedKvCache(dev.ctx, K, G, dim, 14, page, code(pkg, dtype))
    step = kv.PagedStep(dev.ctx, tables, rows, 64, 160)
    f, _ = K.rotary_frequencies(dim, 1e4)
    rotary = kv.Rotary(dev.up(f), dim)
    work = pkg.Buffer.empty(dev.ctx, max(cache.workspace_bytes(K, step, H), 16))
    told = [[] for _ in range(S)]                                   # (k, v) of every position
    size = 4 if dtype == "f32" else 2

    def run(counts, seed):
        lengths = [len(t) + n for t, n in zip(told, counts)]
        for s, (n, length) in enumerate(zip(counts, lengths)):
            if n:
                tables.reserve(s, length)
        x = normal(seed, rows, (H + 2 * G) * dim, dtype=dtype)
        qkv, out, batch = dev.up(x), pkg.Buffer.empty(dev.ctx, rows * H * dim * size), dev.batch()
        step.write(batch, counts, lengths)
        q, k, v = (qkv.view(o * dim * size, qkv.length() - o * dim * size) for o in (0, H, H + G))
        ld = x.shape[1]
        cache.append_into(batch, K, step, k, v, ld, ld, rotary, q, q, H, ld, ld)
        cache.attention_into(batch, K, step, q, out, H, dim ** -0.5, work, q_ld=ld)
        batch.commit_and_wait()
        keys, values = (dev.down(b, (14, G, page, dim), dtype) for b in (cache.keys, cache.values))
        heads = x.reshape(rows, H + 2 * G, dim)
        turned = dev.down(qkv, (rows, H + 2 * G, dim), dtype)[:, :H]
        model = Step([(n, length) for n, length in zip(counts, lengths)], page)
        model.pages, model.table = 14, tables.table.copy()
        places = list(model.places())
        want, sizes = turn(heads[[p[0] for p in places], :H], [p[2] for p in places], f, 1.0, dim, 0, True)
        close(turned[[p[0] for p in places]], want, turn_tolerance(want, sizes, dtype), "queries")
        for s, n in enumerate(counts):
            told[s] += [(heads[int(model.starts[s]) + i, H:H + G], heads[int(model.starts[s]) + i, H + G:]) for i in range(n)]
        for s, length in enumerate(lengths):                        # all positions of all sequences, also of those that take no part
            if length == 0:
                continue
            at = torch.arange(length)
            pg = torch.as_tensor(tables.table[s].astype(np.int64))[at // page]
            ks, vs = (torch.stack([t[i] for t in told[s]]) for i in range(2))
            want, sizes = turn(ks, np.arange(length), f, 1.0, dim, 0, True)
            close(keys[pg, :, at % page], want, turn_tolerance(want, sizes, dtype), "keys")
            assert same_bits(values[pg, :, at % page], vs, dtype)
        keys[~keys.isfinite()], values[~values.isfinite()] = 0, 0    # (slots that nobody has written)
        want, tol = attended(model, turned[:model.rows], keys, values, dim ** -0.5)
        close(dev.down(out, (rows, H, dim), dtype)[:model.rows], want, half_step(dtype) * want.abs() + tol + (2.0 ** -25 if dtype == "f16" else 0), counts)
        apart = told_apart(model, turned[:model.rows], keys, values, dim ** -0.5, dtype)
        assert min(apart[n] for n in ("zeros", "negated")) > 0.9, apart

    run([40, 0, 0], 1)
    run([24, 64, 0], 2)
    run([1, 1, 0], 3)
    shared = tables.share(0, 2, len(told[0]))
    assert shared == 64
    told[2] = told[0][:shared]
    run([1, 1, 5], 4)
    run([0, 1, 1], 5)
    tables.release(1)
    told[1] = []
    run([1, 33, 1], 6)
    tables.release(0)
    told[0] = []
    run([17, 1, 20], 7)


# ---- weights in two terms, and bounds beyond all sums ------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,length", [(1, 65), (4, 65), (1, 600)])
def test_weights_of_few_rows_have_two_terms(dev, dtype, rows, length):
    """One position of weight 1 beside many of a weight that lies between two 16-bit numbers, whose values cancel, so that the output's own rounding hides nothing.

    Rounded once, a weight is off by 0.49 of a step; what is left of it behind two terms is half a step of half a step, half_step^2.  The scores are 0 and ln w, a product
    of one value by the scale: off by 2^-23 |ln w|, 2^-21 for the power of two; the sums of n weights and products n 2^-24 each; each of numerator and denominator."""
    G, dim, H = 2, 64, 8 // rows
    eps, half = torch.finfo(TYPES[dtype]).eps, half_step(dtype)
    w = 0.5 * (1 + 0.49 * eps)
    scale = float(np.float32(-math.log(w)))
    step = Step([(rows, length)], 32, seed=length)
    shape = (step.pages, G, 32, dim)
    keys, values = torch.zeros(shape, dtype=TYPES[dtype]), torch.ones(shape, dtype=TYPES[dtype])
    keys[..., 0] = -1.0
    first = int(step.table[0, 0])
    keys[first, :, 0, 0] = 0.0
    values[first, :, 0] = -w * (length - 1)
    q = torch.zeros(rows, H, dim, dtype=TYPES[dtype])
    q[..., 0] = 1.0
    want, _ = attended(step, q, keys, values, scale)
    n = torch.arange(length - rows, length, dtype=F64)[:, None, None]              # positions of weight w that a row sees
    big = values[first, 0, 0, 0].to(F64).abs()
    off = 2.0 ** -23 + 2.0 ** -21 + (n + 1) * 2.0 ** -24 + (half ** 2 if dtype != "f32" else 0)
    tol = half * want.abs() + 2 * off * (n * w + big) / (1 + n * w)
    if dtype != "f32":                                              # one term would not be within it
        once = (n * torch.tensor(w).to(TYPES[dtype]).to(F64) - big) / (1 + n * w)
        assert bool(((once - want).abs() > 2 * tol).all())
    close(attention_of(dev, step, q, keys, values, dtype, scale), want, tol)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,window", [(1, 0), (60, 0), (1, 700)])
@pytest.mark.parametrize("bound", [0x7FFFFFFF, 0xFFFFFFFF])
def test_attention_of_bounds_whose_steps_exceed_32_bits(dev, dtype, rows, window, bound):
    """A call for lengths up to what a word holds, with so many tiles that what all have to do is summed in larger units."""
    step = Step([(rows, 3000)] + [(rows, 60 + i) for i in range(70)] + [(1, 1500)], 64, seed=rows)
    run_attention(dev, step, dtype, 8, 2, 64, window, seed=rows, max_length=bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("length,max_length", [(100, 100), (6000, 6000), (300, 100000)])
def test_positions_of_scores_of_minus_infinity_weigh_nothing(dev, dtype, rows, length, max_length):
    """As what is masked; a row whose positions are all so becomes zero, as one that sees nothing."""
    step = Step([(rows, length), (1, 50)], 32, seed=length)
    shape = (step.pages, 2, 32, 64)
    keys, values = normal(1, *shape, dtype=dtype), normal(2, *shape, dtype=dtype)
    keys[..., 0] = 0.0
    first = torch.from_numpy(step.table[0][step.table[0] != NO_PAGE].astype(np.int64))
    keys[first, 1, :, 0] = -math.inf                               # all of the first sequence for one kv head, some positions for the other
    keys[first, 0, ::3, 0] = -math.inf
    q = normal(3, step.rows, 4, 64, dtype=dtype)
    q[..., 0] = 1.0
    got = attention_of(dev, step, q, keys, values, dtype, 0.125, max_length=max_length)
    assert bool((got[:rows, 2:] == 0).all())
    # the same without those positions: keys that score -2^9 there, whose weights 64 bits hold and 32 do not
    low = keys.clone()
    low[first, :, :, 0] = torch.where(keys[first, :, :, 0].isinf(), torch.tensor(-4096.0).to(TYPES[dtype]), keys[first, :, :, 0])
    want, _ = attended(step, q, low, values, 0.125)
    keys[first, :, :, 0] = torch.where(keys[first, :, :, 0].isinf(), torch.tensor(0.0).to(TYPES[dtype]), keys[first, :, :, 0])
    _, tol = attended(step, q, keys, values, 0.125)
    tol = half_step(dtype) * want.abs() + 2 * tol + (2.0 ** -25 if dtype == "f16" else 0)
    close(got[:rows, :2], want[:rows, :2], tol[:rows, :2])
    close(got[rows:], want[rows:], tol[rows:])
