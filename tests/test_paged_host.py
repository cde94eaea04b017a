"""Host side of rotary positions and paged caches: frequencies, page tables, workspaces and every refusal.  No GPU work: the entry points
refuse before they touch a device, so the buffers here are handles over no memory."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from paged_models import TYPES, Step, padded, told_apart


# ---- frequencies ------------------------------------------------------------------------------------------------------------
def by_parts(rot, base, factor, original, fast, slow):
    def index(turns):
        return rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
    lo, hi = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), rot - 1)
    i = np.arange(rot // 2)
    f = base ** (-2.0 * i / rot)
    ramp = np.clip((i - lo) / (max(hi - lo, 0.001)), 0, 1)
    return f * (1 - ramp) + f / factor * ramp


@pytest.mark.parametrize("rot,base", [(2, 1e4), (50, 1e4), (128, 1e6), (256, 5e5)])
def test_frequencies_follow_their_formulas(pkg, rot, base):
    K = pkg.Kernels
    f, a = K.rotary_frequencies(rot, base)
    want = base ** (-2.0 * np.arange(rot // 2) / rot)
    assert a == 1.0 and f.dtype == np.float32 and np.allclose(f, want, rtol=2.0 ** -23, atol=0)
    f, a = K.rotary_frequencies(rot, base, pkg.ROTARY_LINEAR, 8.0)
    assert a == 1.0 and np.allclose(f, want / 8, rtol=2.0 ** -23, atol=0)
    f, a = K.rotary_frequencies(rot, base, pkg.ROTARY_BY_PARTS, 4.0, 4096.0, 32.0, 1.0)
    assert a == np.float32(0.1 * math.log(4.0) + 1.0) and np.allclose(f, by_parts(rot, base, 4.0, 4096.0, 32.0, 1.0), rtol=2.0 ** -22, atol=0)
    assert np.isclose(f[0], 1.0) and np.all(f <= want.astype(np.float32) * (1 + 2.0 ** -22)) and np.all(f >= want / 4 * (1 - 2.0 ** -22))


@pytest.mark.parametrize("args", [(0, 1e4), (3, 1e4), (4098, 1e4), (64, 1.0), (64, math.nan), (64, math.inf), (64, 1e4, 3), (64, 1e4, 1, 0.5), (64, 1e4, 1, math.nan),
                                  (64, 1e4, 2, 4.0, 0.0), (64, 1e4, 2, 4.0, 4096.0, 1.0, 1.0), (64, 1e4, 2, 4.0, 4096.0, 32.0, 0.0),
                                  (64, 1e4, 2, 4.0, math.inf)])
def test_frequencies_that_are_refused(pkg, args):
    with pytest.raises(pkg.InvalidArgument):
        pkg.Kernels.rotary_frequencies(*args)


# ---- page tables --------------------------------------------------------------------------------------------------------------
def test_tables_deal_out_and_take_back_pages(pkg):
    from local_ai_amd.kv_cache import PageTables
    t = PageTables(10, 16, 3, 100)
    assert t.table.shape == (3, 7) and np.all(t.table == t.NO_PAGE)
    t.reserve(0, 1)
    t.reserve(0, 16)
    assert t.held[0] == 1
    t.reserve(0, 17)
    t.reserve(1, 100)
    assert t.held == [2, 7, 0] and len(t.free) == 1
    used = np.concatenate([t.table[0, :2], t.table[1]])
    assert len(set(used.tolist())) == 9 and used.max() < 10
    with pytest.raises(pkg.InvalidArgument):
        t.reserve(2, 17)
    assert t.held[2] == 0 and len(t.free) == 1          # nothing of it is kept
    with pytest.raises(pkg.InvalidArgument):
        t.reserve(0, 113)
    t.release(1)
    t.reserve(2, 100)
    t.reserve(2, 5)                                      # never fewer
    assert t.held == [2, 0, 7] and np.all(t.table[1] == t.NO_PAGE)


def test_shared_pages_go_back_with_their_last_holder(pkg):
    from local_ai_amd.kv_cache import PageTables
    t = PageTables(8, 16, 3, 64)
    t.reserve(0, 40)
    assert t.share(0, 1, 40) == 32 and t.held[1] == 2 and np.array_equal(t.table[0, :2], t.table[1, :2])
    t.reserve(1, 40)
    assert t.table[1, 2] != t.table[0, 2]
    with pytest.raises(pkg.InvalidArgument):
        t.share(0, 1, 16)
    assert t.share(1, 2, 15) == 0
    first = set(t.table[0, :2].tolist())
    t.release(0)
    assert not first & set(t.free) and len(t.free) == 5
    t.release(1)
    assert first <= set(t.free) and len(t.free) == 8 and not t.holders.any()
    for page in (0, 8, 24, 2048):
        with pytest.raises(pkg.InvalidArgument):
            PageTables(8, page, 1, 64)


def test_steps_that_are_refused(pkg, monkeypatch):
    from local_ai_amd import kv_cache
    written = []

    class Fake:
        @staticmethod
        def empty(ctx, n):
            return n

    class Batch:
        def write(self, dst, src):
            written.append((dst, np.array(src)))
    monkeypatch.setattr(kv_cache, "Buffer", Fake)
    t = kv_cache.PageTables(8, 16, 3, 64)
    t.reserve(0, 33)
    t.reserve(2, 16)
    s = kv_cache.PagedStep(None, t, rows=6, max_rows=4, max_length=40)
    s.write(Batch(), [4, 0, 2], [33, 0, 16])
    assert [w[1].tolist() for w in written[1:]] == [[0, 4, 4, 6], [33, 0, 16]] and np.array_equal(written[0][1], t.table)
    for counts, lengths in (([4, 0], [33, 0]), ([5, 0, 0], [33, 0, 0]), ([1, 1, 0], [33, 1, 0]), ([1, 0, 0], [49, 0, 0]), ([3, 0, 0], [2, 0, 0]),
                            ([4, 0, 3], [33, 0, 16]), ([-1, 0, 0], [33, 0, 0])):
        with pytest.raises(pkg.InvalidArgument):
            s.write(Batch(), counts, lengths)
    t.reserve(0, 48)
    with pytest.raises(pkg.InvalidArgument):
        s.write(Batch(), [1, 0, 0], [41, 0, 0])


# ---- workspaces -----------------------------------------------------------------------------------------------------------------
def test_padded_heads_and_workspaces(pkg):
    lib = pkg.lib()
    for d in (1, 31, 32, 33, 64, 65, 100, 128, 129, 192, 193, 256):
        assert lib.lh_paged_padded_dim(d) == padded(d)
    f = lib.lh_paged_attention_workspace_bytes
    assert f(1, 1, 1, 64, 8, 2, 128) == 0                     # too short to be cut
    assert f(1, 1, 1, 32768, 8, 2, 128) > 0
    assert f(1, 1, 1, 32768, 8, 3, 128) == 0 and f(0, 1, 1, 99, 8, 2, 128) == 0 and f(1, 1, 1, 32768, 8, 0, 128) == 0


# ---- refusals --------------------------------------------------------------------------------------------------------------------
class BufferHandle(C.Structure):          # lh_buffer of csrc/common.hpp
    _fields_ = [("ctx", C.c_void_p), ("ptr", C.c_void_p), ("len", C.c_size_t), ("owns", C.c_bool), ("slack", C.c_size_t), ("host", C.c_void_p)]


class BatchHandle(C.Structure):
    _fields_ = [("ctx", C.c_void_p), ("dispatch_count", C.c_uint32)]


def buf(at, nbytes):
    return BufferHandle(None, at, nbytes, False, 0, None)


GB = 1 << 30


class Call:
    """Arguments of a call that would be taken, by name and in order; `refused` changes some of them."""

    def __init__(self, pkg, name, **args):
        self.pkg, self.f, self.args = pkg, getattr(pkg.lib(), name), args

    def status(self, **changed):
        assert set(changed) <= set(self.args)
        batch = BatchHandle(None, 0)
        vals = [None if changed.get("batch", 0) is None else C.byref(batch)] if "batch" in self.args else []
        for name, v in {**self.args, **changed}.items():
            if name == "batch":
                continue
            vals.append(C.byref(v) if isinstance(v, BufferHandle) else C.c_float(v) if isinstance(v, float) else None if v is None else C.c_uint32(v))
        rc = self.f(*vals)
        assert batch.dispatch_count == 0
        return rc

    def refused(self, **changed):
        assert self.status(**changed) == self.pkg.InvalidArgument.code, changed
        assert self.pkg.lib().lh_last_error().decode().startswith("Invalid argument: ")


def test_prototypes_are_the_headers(pkg):
    import os
    import re
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "local_hip.h")).read(), flags=re.S)
    for name, kinds in pkg._PROTOTYPES.items():
        args, = re.findall(rf"\b{name}\(([^)]*)\)", text)
        want = "".join("p" if "*" in a else "f" if "float" in a else "u" for a in args.split(","))
        assert kinds == want, name


def test_whole_numbers_of_numpy_are_taken(pkg):
    class Handle:
        def __init__(self, h):
            self._h = C.cast(C.pointer(h), C.c_void_p)
    b, x = Handle(BatchHandle(None, 0)), Handle(buf(GB, 1 << 20))
    K = pkg.Kernels.__new__(pkg.Kernels)
    K._l = pkg.lib()
    for u, f in ((np.int64, np.float32), (np.uint32, float), (int, np.float64)):
        K.rotary_rows_into(b, x, x, u(2), x, x, f(1.0), u(0), u(4), u(64), u(64), u(0), u(1), u(256), u(256))
        with pytest.raises(pkg.InvalidArgument, match="dtype 9"):
            K.rotary_rows_into(b, x, x, u(9), x, x, f(1.0), u(0), u(4), u(64), u(64), u(0), u(1), u(256), u(256))


def test_rotary_refusals(pkg):
    c = Call(pkg, "lh_rotary_rows_into", batch=True, input=buf(GB, 10 * 512 * 2), output=buf(2 * GB, 10 * 512 * 2), dtype=2, positions=buf(3 * GB, 40), frequencies=buf(4 * GB, 256),
             amplitude=1.0, rows=10, heads=4, dim=128, rot=128, first=0, pairing=1, input_ld=512, output_ld=512)
    assert c.status(rows=0) == 0 and c.status(heads=0) == 0
    for changed in (dict(batch=None), dict(dtype=3), dict(dtype=1), dict(rot=127), dict(rot=130), dict(rot=64, first=65), dict(first=2), dict(pairing=2), dict(dim=0), dict(dim=2048),
                    dict(input=None), dict(output=None), dict(positions=None), dict(frequencies=None), dict(rows=11), dict(heads=5), dict(input_ld=511), dict(output_ld=500),
                    dict(input_ld=513), dict(positions=buf(3 * GB, 39)), dict(frequencies=buf(4 * GB, 255)), dict(input=buf(GB + 1, 10 * 512 * 2)),
                    dict(heads=1 << 20), dict(output=buf(GB + 2, 10 * 512 * 2)), dict(output=buf(GB + 1024, 10 * 512 * 2)),
                    dict(positions=buf(3 * GB + 2, 40)), dict(frequencies=buf(4 * GB + 1, 256)), dict(first=0xFFFFFFFE)):
        c.refused(**changed)
    # the same rows at another distance; rows of one distance side by side are taken (checked on the device)
    c.refused(output=buf(GB, 10 * 600 * 2), output_ld=600)


def append_call(pkg, **more):
    pool = 7 * 2 * 16 * 128 * 2
    a = dict(batch=True, k=buf(GB, 6 * 1024 * 2), v=buf(2 * GB, 6 * 1024 * 2), dtype=2, keys=buf(3 * GB, pool), values=buf(4 * GB, pool), table=buf(5 * GB, 3 * 4 * 4),
             starts=buf(6 * GB, 16), lengths=buf(7 * GB, 12), rows=6, sequences=3, kv_heads=2, dim=100, pages=7, page=16, table_ld=4, k_ld=1024, v_ld=1024,
             frequencies=buf(8 * GB, 200), amplitude=1.0, rot=100, first=0, pairing=0, q=buf(9 * GB, 6 * 800 * 2), q_output=buf(10 * GB, 6 * 800 * 2), heads=8, q_ld=800, q_output_ld=800)
    return Call(pkg, "lh_paged_append_into", **{**a, **more})


def test_append_refusals(pkg):
    c = append_call(pkg)
    assert c.status(rows=0) == 0
    pool = 7 * 2 * 16 * 128 * 2
    for changed in (dict(batch=None), dict(dtype=4), dict(dtype=1), dict(k=None), dict(v=None), dict(keys=None), dict(values=None), dict(table=None), dict(starts=None),
                    dict(lengths=None), dict(rows=7), dict(sequences=0), dict(sequences=4), dict(kv_heads=0), dict(kv_heads=3), dict(dim=0), dict(dim=257), dict(dim=129),
                    dict(pages=0), dict(pages=8), dict(page=8), dict(page=24), dict(page=32), dict(page=2048), dict(table_ld=0), dict(table_ld=5), dict(k_ld=199), dict(v_ld=199),
                    dict(k_ld=1300), dict(frequencies=None), dict(rot=101), dict(rot=102), dict(first=2), dict(pairing=2), dict(q=None), dict(q_output=None), dict(heads=0),
                    dict(q=None, q_output=None), dict(heads=9), dict(q_ld=799), dict(q_output_ld=900), dict(keys=buf(3 * GB + 8, pool)), dict(values=buf(3 * GB, pool)),
                    dict(values=buf(3 * GB + pool - 16, pool)), dict(k=buf(3 * GB + 64, 6 * 1024 * 2)), dict(v=buf(4 * GB - 16, 6 * 1024 * 2)), dict(q=buf(3 * GB, 6 * 800 * 2)),
                    dict(q_output=buf(4 * GB + pool - 2, 6 * 800 * 2)), dict(q_output=buf(9 * GB + 2, 6 * 800 * 2)), dict(q_output=buf(GB + 398, 6 * 1024 * 2), q_output_ld=1024),
                    dict(q_output=buf(2 * GB, 6 * 800 * 2)), dict(k=buf(GB + 1, 6 * 1024 * 2)), dict(table=buf(5 * GB + 2, 48)), dict(starts=buf(6 * GB + 1, 16)),
                    dict(table_ld=1 << 28, page=1024), dict(sequences=1 << 21)):
        c.refused(**changed)
    append_call(pkg, q=None, q_output=None, heads=0).refused(q=buf(9 * GB, 6 * 800 * 2))


def test_attention_refusals(pkg):
    pool = 2000 * 2 * 16 * 128 * 2
    need = pkg.lib().lh_paged_attention_workspace_bytes(6, 3, 4, 16000, 8, 2, 100)
    assert need > 0
    c = Call(pkg, "lh_paged_attention_into", batch=True, q=buf(GB, 6 * 800 * 2), keys=buf(3 * GB, pool), values=buf(4 * GB, pool), output=buf(2 * GB, 6 * 800 * 2), dtype=2,
             table=buf(5 * GB, 3 * 1000 * 4), starts=buf(6 * GB, 16), lengths=buf(7 * GB, 12), rows=6, sequences=3, max_rows=4, max_length=16000, heads=8, kv_heads=2, dim=100,
             pages=2000, page=16, table_ld=1000, q_ld=800, output_ld=800, scale=0.1, window=0, sink=buf(8 * GB, 32), workspace=buf(9 * GB, need))
    assert c.status(rows=0) == 0
    for changed in (dict(batch=None), dict(dtype=7), dict(dtype=1), dict(q=None), dict(keys=None), dict(values=None), dict(output=None), dict(table=None), dict(starts=None),
                    dict(lengths=None), dict(rows=7), dict(sequences=4), dict(sequences=0), dict(max_rows=0), dict(max_rows=7), dict(heads=0), dict(heads=7), dict(kv_heads=3), dict(kv_heads=0),
                    dict(dim=0), dict(dim=101), dict(dim=300), dict(pages=2001), dict(page=17), dict(table_ld=1001), dict(q_ld=700), dict(output_ld=799), dict(output_ld=801),
                    dict(scale=math.nan), dict(scale=math.inf), dict(sink=buf(8 * GB, 31)), dict(sink=buf(8 * GB + 2, 32)), dict(workspace=None), dict(workspace=buf(9 * GB, need - 1)),
                    dict(workspace=buf(9 * GB + 4, need)), dict(output=buf(GB, 6 * 800 * 2)), dict(output=buf(GB + 6 * 1600 - 2, 6 * 800 * 2)), dict(keys=buf(3 * GB + 2, pool)),
                    dict(output=buf(4 * GB + pool - 2, 6 * 800 * 2)), dict(workspace=buf(2 * GB + 6 * 1600 - 16, need)), dict(workspace=buf(GB - need + 16, need)),
                    dict(workspace=buf(3 * GB + 16, need))):
        c.refused(**changed)


# ---- what is read may not lie where a call writes ----------------------------------------------------------------------------------
def test_rotary_outputs_over_what_is_read_are_refused(pkg):
    rows, ld = 10, 1024
    c = Call(pkg, "lh_rotary_rows_into", batch=True, input=buf(GB, rows * 512 * 2), output=buf(2 * GB, rows * ld * 2), dtype=2, positions=buf(3 * GB, 40), frequencies=buf(4 * GB, 256),
             amplitude=1.0, rows=rows, heads=4, dim=128, rot=128, first=0, pairing=1, input_ld=512, output_ld=ld)
    for at in (2 * GB, 2 * GB - 36, 2 * GB + 9 * ld * 2 + 1020, 2 * GB + 4 * ld * 2 - 4, 2 * GB + 1000):
        c.refused(positions=buf(at, 40))
        assert "output lies over positions" in pkg.lib().lh_last_error().decode()
    for at in (2 * GB, 2 * GB - 252, 2 * GB + 9 * ld * 2 + 1020, 2 * GB + ld * 2 + 1000, 2 * GB + ld * 2 - 252):
        c.refused(frequencies=buf(at, 256))
        assert "output lies over frequencies" in pkg.lib().lh_last_error().decode()


def test_append_outputs_over_what_is_read_are_refused(pkg):
    pool = 7 * 2 * 16 * 128 * 2
    c = append_call(pkg)
    sizes = {"table": 48, "starts": 16, "lengths": 12, "frequencies": 200}
    for name, n in sizes.items():
        for written, (at, end) in {"keys": (3 * GB, 3 * GB + pool), "values": (4 * GB, 4 * GB + pool), "q_output": (10 * GB, 10 * GB + 6 * 1600)}.items():
            for where in (at - n + 4, at, (at + end) // 2 // 16 * 16, end - 4):
                c.refused(**{name: buf(where, n)})
                assert f"{written} lies over {name}" in pkg.lib().lh_last_error().decode()


def test_attention_outputs_over_what_is_read_are_refused(pkg):
    pool = 2000 * 2 * 16 * 128 * 2
    need = pkg.lib().lh_paged_attention_workspace_bytes(6, 3, 4, 16000, 8, 2, 100)
    c = Call(pkg, "lh_paged_attention_into", batch=True, q=buf(GB, 6 * 800 * 2), keys=buf(3 * GB, pool), values=buf(4 * GB, pool), output=buf(2 * GB, 6 * 800 * 2), dtype=2,
             table=buf(5 * GB, 3 * 1000 * 4), starts=buf(6 * GB, 16), lengths=buf(7 * GB, 12), rows=6, sequences=3, max_rows=4, max_length=16000, heads=8, kv_heads=2, dim=100,
             pages=2000, page=16, table_ld=1000, q_ld=800, output_ld=800, scale=0.1, window=0, sink=buf(8 * GB, 32), workspace=buf(9 * GB, need))
    for name, n in {"table": 12000, "starts": 16, "lengths": 12, "sink": 32}.items():
        for written, (at, end) in {"output": (2 * GB, 2 * GB + 6 * 1600), "workspace": (9 * GB, 9 * GB + need)}.items():
            for where in (at - n + 4, at, (at + end) // 2 // 16 * 16, end - 4):
                c.refused(**{name: buf(where, n)})
                assert f"{written} lies over {name}" in pkg.lib().lh_last_error().decode()


# ---- steps over shared pages ---------------------------------------------------------------------------------------------------------
class Written:
    """Stands for a batch: what was written, no device."""
    def __init__(self):
        self.all = []

    def write(self, dst, src):
        self.all.append(np.array(src))


@pytest.fixture
def no_device(pkg, monkeypatch):
    from local_ai_amd import kv_cache

    class Fake:
        @staticmethod
        def empty(ctx, n):
            return n
    monkeypatch.setattr(kv_cache, "Buffer", Fake)
    return kv_cache


def test_steps_that_append_to_shared_pages_are_refused(pkg, no_device):
    t = no_device.PageTables(12, 16, 3, 96)
    t.reserve(0, 40)
    assert t.share(0, 1, 40) == 32
    t.reserve(1, 60)
    s, b = no_device.PagedStep(None, t, rows=40, max_rows=40, max_length=96), Written()
    for counts, lengths in (([0, 4, 0], [40, 30, 0]),                  # the target, inside what it was given
                            ([0, 1, 0], [0, 32, 0]), ([0, 2, 0], [0, 33, 0]), ([0, 40, 0], [0, 60, 0]),
                            ([1, 0, 0], [20, 0, 0]),                   # the source, whose pages were given away before they were written
                            ([9, 0, 0], [40, 0, 0])):
        with pytest.raises(pkg.InvalidArgument, match="shared"):
            s.write(b, counts, lengths)
        assert not b.all                                              # nothing of it is sent
    s.write(b, [8, 28, 0], [40, 60, 0])                               # both behind what they share
    assert [w.tolist() for w in b.all[1:]] == [[0, 8, 36, 36], [40, 60, 0]]
    s.write(b, [0, 2, 0], [0, 60, 0])
    t.release(0)                                                      # the last holder may write again
    s.write(b, [0, 30, 0], [0, 30, 0])


def test_steps_that_only_attend_may_stand_on_shared_pages(pkg, no_device):
    t = no_device.PageTables(12, 16, 2, 96)
    t.reserve(0, 48)
    assert t.share(0, 1, 48) == 48
    s, b = no_device.PagedStep(None, t, rows=4, max_rows=4, max_length=96), Written()
    cache = no_device.PagedKvCache.__new__(no_device.PagedKvCache)
    cache.kv_heads, cache.dim, cache.dtype, cache.pages, cache.page, cache.keys, cache.values = 1, 64, 2, 12, 16, None, None

    class Kernels:
        calls = 0

        def paged_append_into(self, *a, **k):
            Kernels.calls += 1
    with pytest.raises(pkg.InvalidArgument):
        s.write(b, [0, 1], [48, 48])
    s.write(b, [0, 1], [48, 48], append=False)                        # a given beginning's last row once more, for its logits
    assert b.all[-1].tolist() == [48, 48]
    with pytest.raises(pkg.InvalidArgument, match="append"):
        cache.append_into(None, Kernels(), s, None, None)
    assert Kernels.calls == 0
    t.reserve(1, 49)
    s.write(b, [0, 1], [48, 49])
    cache.append_into(None, Kernels(), s, None, None)
    assert Kernels.calls == 1


def test_shares_of_fewer_than_no_positions_are_refused(pkg, no_device):
    t = no_device.PageTables(12, 16, 3, 96)
    t.reserve(0, 40)
    for positions in (-1, -16, -17, -100):
        with pytest.raises(pkg.InvalidArgument):
            t.share(0, 1, positions)
        with pytest.raises(pkg.InvalidArgument):
            t.reserve(1, positions)
    assert t.held == [3, 0, 0] and np.all(t.table[1] == t.NO_PAGE) and int(t.holders.sum()) == 3 and len(t.free) == 9
    assert t.share(0, 1, 0) == 0
    t.reserve(1, 0)
    assert t.held[1] == 0


def test_steps_of_other_pools_are_refused(pkg, no_device):
    """Tables of another page size, or of more pages than the cache has, would send rows to wrong slots or drop them."""
    class Kernels:
        calls = 0

        def paged_padded_dim(self, dim):
            return padded(dim)

        def paged_append_into(self, *a, **k):
            Kernels.calls += 1
        paged_attention_into = paged_append_into
    K = Kernels()
    for pages, page, right in ((12, 16, True), (12, 32, False), (6, 32, False), (13, 16, False), (11, 16, True)):
        cache = no_device.PagedKvCache(None, K, 2, 64, 12, 16)
        t = no_device.PageTables(pages, page, 2, 64)
        s, before = no_device.PagedStep(None, t, 4, 4, 64), Kernels.calls
        for call in (lambda: cache.append_into(None, K, s, None, None), lambda: cache.attention_into(None, K, s, None, None, 4, 0.1)):
            if right:
                call()
            else:
                with pytest.raises(pkg.InvalidArgument, match="pages"):
                    call()
        assert Kernels.calls - before == (2 if right else 0)


# ---- the tolerance -------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sequences", [[(40, 40)], [(24, 64), (64, 64)], [(1, 65), (1, 65)], [(1, 67), (1, 66), (5, 69)]])
def test_the_tolerance_of_attention_tells_wrong_results(dtype, sequences):
    """The steps of a session of 8 heads of 64 over 2: outputs that are zero, negated, of other pages or other slots are not within it."""
    step, g = Step(sequences, 16, seed=1), torch.Generator().manual_seed(2)
    q = torch.randn(step.rows, 8, 64, generator=g).to(TYPES[dtype])
    keys, values = (torch.randn(step.pages, 2, 16, 64, generator=g).to(TYPES[dtype]) for _ in range(2))
    shares = told_apart(step, q, keys, values, 0.125, dtype)
    assert min(shares.values()) > 0.9, shares


def test_scales_that_are_not_finite_in_powers_of_two_are_refused(pkg):
    """Scores are kept in powers of two: a scale above the largest f32 over log2(e) would be an infinity there, and 0 times it NaN."""
    pool = 2000 * 2 * 16 * 128 * 2
    c = Call(pkg, "lh_paged_attention_into", batch=True, q=buf(GB, 6 * 800 * 2), keys=buf(3 * GB, pool), values=buf(4 * GB, pool), output=buf(2 * GB, 6 * 800 * 2), dtype=2,
             table=buf(5 * GB, 3 * 1000 * 4), starts=buf(6 * GB, 16), lengths=buf(7 * GB, 12), rows=0, sequences=3, max_rows=4, max_length=16000, heads=8, kv_heads=2, dim=100,
             pages=2000, page=16, table_ld=1000, q_ld=800, output_ld=800, scale=0.1, window=0, sink=buf(8 * GB, 32), workspace=None)
    for scale in (3e38, -3e38, 2.36e38):
        c.refused(scale=scale)
    assert c.status(scale=2.35e38) == 0 and c.status(scale=-2.35e38) == 0
