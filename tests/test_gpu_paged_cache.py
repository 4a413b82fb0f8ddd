"""The paged cache: rows written (bf16 and quantised to e4m3), read back, and attended to by one row a sequence, against float64. The cache's own
content is compared place by place; places that no row goes to keep what they held."""
import ctypes as C

import numpy as np
import pytest

import sequences_reference as sr
from gpu_harness import Dev, ptr_add

pytestmark = pytest.mark.gpu
KINDS = ["bf16", "fp8"]


@pytest.fixture(scope="module")
def dev():
    return Dev()


class Cache:
    """A cache on the device with its image on the host. What it starts with is not a number anywhere."""

    def __init__(self, dev, kind, pages, page, kv, hd, table, offset=0):
        self.dev, self.kind, self.pages, self.page, self.kv, self.hd = dev, kind, pages, page, kv, hd
        self.table = np.asarray(table, np.int32)
        shape = (max(pages, 1), kv, page, hd)
        self.fill = 0x7fc0 if kind == "bf16" else 0x7f
        self.k, self.v = (np.full(shape, self.fill, np.uint16 if kind == "bf16" else np.uint8) for _ in "kv")
        self.ks, self.vs = (np.full(shape[:3], 255, np.uint8) for _ in "kv")
        self.offset = offset

        def put(a):
            d = dev.alloc(a.nbytes + 64)
            dev.lib.iris_dev_upload(ptr_add(d, offset), a.ctypes.data, a.nbytes)
            return ptr_add(d, offset)
        self.dk, self.dv, self.dks, self.dvs = put(self.k), put(self.v), put(self.ks), put(self.vs)
        self.dtable = dev.put(self.table)

    def where(self):
        return (self.dk, self.dv) if self.kind == "bf16" else (self.dk, self.dv, self.dks, self.dvs)

    def place(self, g, pos):
        """(page, place) or None"""
        if not 0 <= pos < self.table.shape[1] * self.page:
            return None
        page = int(self.table[g, pos // self.page])
        return (page, pos % self.page) if 0 <= page < self.pages else None

    def length(self, lengths, g):
        return int(min(max(int(lengths[g]), 0), self.table.shape[1] * self.page))

    def rows_of(self, lengths, first, rows):
        """(row, place) of every row that goes somewhere"""
        at = [(g, g + 1) for g in range(rows)] if first is None else sr.spans(first, rows)
        for g, (a, b) in enumerate(at):
            for r in range(a, b):
                where = self.place(g, max(int(lengths[g]), 0) - (b - a) + r - a)
                if where:
                    yield r, where

    def write(self, lengths, k, v, first=None, pad=0, offset=0):
        dev, n, cols = self.dev, len(lengths), self.kv * self.hd
        rows = len(k)

        def put(a):
            b = np.full((rows, cols + pad), 0x7fc0, np.uint16)
            b[:, :cols] = a
            d = dev.alloc(b.nbytes + 64)
            dev.lib.iris_dev_upload(ptr_add(d, 2 * offset), b.ctypes.data, b.nbytes)
            return ptr_add(d, 2 * offset)
        dfirst = dev.put(np.asarray(first, np.int32)) if first is not None else None
        getattr(dev.lib, "iris_dev_cache_write_" + self.kind)(*self.where(), self.pages, self.page, self.dtable, self.table.shape[1],
                                                              dev.put(np.asarray(lengths, np.int32)), put(k), put(v), cols + pad, dfirst, n, rows,
                                                              self.kv, self.hd)
        dev.check()
        shape = (rows, self.kv, self.hd)
        if self.kind == "bf16":
            new = [(self.k, None, k.reshape(shape), None), (self.v, None, v.reshape(shape), None)]
        else:
            new = [(self.k, self.ks, *sr.quantise(sr.bf16_value(k).reshape(shape))), (self.v, self.vs, *sr.quantise(sr.bf16_value(v).reshape(shape)))]
        for pages, scales, rows_, bytes_ in new:
            for r, (page, at) in self.rows_of(lengths, first, rows):
                pages[page, :, at] = rows_[r]
                if scales is not None:
                    scales[page, :, at] = bytes_[r]

    def check(self):
        """The device holds what the host's image says, bit for bit"""
        for d, a in ((self.dk, self.k), (self.dv, self.v), *(((self.dks, self.ks), (self.dvs, self.vs)) if self.kind == "fp8" else ())):
            got = self.dev.get(d, a.shape, a.dtype)
            assert np.array_equal(got, a), f"{(got != a).sum()} of {a.size} differ, first at {np.argwhere(got != a)[0]}"

    def values(self):
        if self.kind == "bf16":
            return sr.bf16_value(self.k).astype(np.float64), sr.bf16_value(self.v).astype(np.float64)
        return (sr.e4m3_value(self.k) * sr.scale_value(self.ks)[..., None], sr.e4m3_value(self.v) * sr.scale_value(self.vs)[..., None])

    def read(self, lengths, rows, first=None, pad=0, offset=0):
        dev, cols = self.dev, self.kv * self.hd
        out0 = np.full((rows * (cols + pad) + 16,), 0x4321, np.uint16)
        dk, dv = dev.put(out0), dev.put(out0)
        dfirst = dev.put(np.asarray(first, np.int32)) if first is not None else None
        getattr(dev.lib, "iris_dev_cache_read_" + self.kind)(ptr_add(dk, 2 * offset), ptr_add(dv, 2 * offset), cols + pad, *self.where(), self.pages, self.page,
                                                             self.dtable, self.table.shape[1], dev.put(np.asarray(lengths, np.int32)), dfirst,
                                                             len(lengths), rows, self.kv, self.hd)
        dev.check()
        kf, vf = self.values()
        for d, whole in ((dk, kf), (dv, vf)):
            want = out0.copy()
            body = want[offset:offset + rows * (cols + pad)].reshape(rows, cols + pad)
            for r, (page, at) in self.rows_of(lengths, first, rows):
                body[r, :cols] = sr.bf16_round(whole[page, :, at].reshape(-1).astype(np.float32))
            got = dev.get(d, out0.shape, np.uint16)
            nan = np.isnan(sr.bf16_value(want))
            assert np.isnan(sr.bf16_value(got[nan])).all() and np.array_equal(got[~nan], want[~nan])

    def attend(self, lengths, q, heads, scale, pad=0, offset=0, kernel=None, workspace=None, compare=True):
        dev, n, cols = self.dev, len(lengths), heads * self.hd
        b = np.full((max(n, 1), cols + pad), 0x7fc0, np.uint16)
        b[:len(q), :cols] = q
        dq = dev.alloc(b.nbytes + 64)
        dev.lib.iris_dev_upload(ptr_add(dq, 2 * offset), b.ctypes.data, b.nbytes)
        out0 = np.full((n * (cols + pad) + 16,), 0x4321, np.uint16)
        do = dev.put(out0)
        getattr(dev.lib, "iris_dev_attention_paged_" + self.kind)(ptr_add(do, 2 * offset), cols + pad, ptr_add(dq, 2 * offset), cols + pad, *self.where(), self.pages,
                                                                  self.page, self.dtable, self.table.shape[1], dev.put(np.asarray(lengths, np.int32)), n,
                                                                  heads, self.kv, self.hd, scale, workspace)
        dev.check()
        if kernel:
            assert dev.dev.last_kernel() == kernel
        got = dev.get(do, out0.shape, np.uint16)
        assert (got[:offset] == 0x4321).all() and (got[offset + n * (cols + pad):] == 0x4321).all()
        got = got[offset:offset + n * (cols + pad)].reshape(n, -1)
        assert (got[:, cols:] == 0x4321).all()
        got = got[:, :cols]
        if compare:
            values = self.values()
            for g in range(n):
                sr.check(sr.bf16_value(got[g]).astype(np.float64).reshape(1, heads, self.hd), self.expected(lengths, g, q[g], heads, scale, values), f"sequence {g}")
        return got

    def expected(self, lengths, g, q, heads, scale, values=None):
        at = [p for p in (self.place(g, i) for i in range(self.length(lengths, g))) if p]
        kf, vf = values or self.values()
        k = np.array([kf[page, :, i] for page, i in at]).reshape(len(at), self.kv, self.hd)
        v = np.array([vf[page, :, i] for page, i in at]).reshape(len(at), self.kv, self.hd)
        o, w, s = sr.softmax_rows(sr.bf16_value(q).astype(np.float64).reshape(1, heads, self.hd), k, v, scale, [len(at)])
        return o, sr.bound(o, w, s, self.hd, True)


def rows(seed, n, cols, spread=1.0):
    return sr.bf16_round(np.random.default_rng(seed).standard_normal((n, cols)).astype(np.float32) * spread)


def filled(dev, kind, lengths, page, kv, hd, seed=1, spare=2, extra_columns=0, spread=1.0, offset=0):
    """A cache of sequences of these lengths in pages of no order, written in one call"""
    per = [-(-n // page) for n in lengths]
    order = np.random.default_rng(seed).permutation(sum(per) + spare)
    table, at = np.full((len(lengths), max(1, max(per, default=0)) + extra_columns), -1), 0
    for g, n in enumerate(per):
        table[g, :n] = order[at:at + n]
        at += n
    c = Cache(dev, kind, len(order), page, kv, hd, table, offset)
    total = sum(lengths)
    if total:
        c.write(lengths, rows(seed, total, kv * hd, spread), rows(seed + 1, total, kv * hd, spread), np.concatenate([[0], np.cumsum(lengths)]))
    return c


LENGTHS = {
    "one": [1], "two pages": [17], "odd": [1, 16, 31, 33, 0, 70], "a page and more": [64, 65, 128], "longer": [700, 3, 0, 129], "many": [(7 * i) % 41 for i in range(130)],
    "all empty": [0, 0], "one long": [5000],
}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [1, 2, 16, 64])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_written_read_back_and_attended_to(dev, lengths, page, kind):
    lengths = LENGTHS[lengths]
    kv, heads, hd = 2, 8, 128
    c = filled(dev, kind, lengths, page, kv, hd)
    c.check()
    c.read(lengths, sum(lengths) + 1, np.concatenate([[0], np.cumsum(lengths)]))
    c.attend(lengths, rows(3, len(lengths), heads * hd), heads, hd ** -0.5)
    dev.free_all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (5, 1), (16, 1), (17, 1), (64, 2), (24, 24), (30, 6)])
def test_groups_of_any_size(dev, heads, kv, kind):
    lengths = [90, 1, 40]
    c = filled(dev, kind, lengths, 16, kv, 128)
    c.attend(lengths, rows(4, 3, heads * 128), heads, 128 ** -0.5)
    dev.free_all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [1, 24, 64, 80, 129, 256, 520])
def test_other_head_sizes(dev, hd, kind):
    lengths = [37, 0, 80]
    c = filled(dev, kind, lengths, 16, 2, hd)
    c.check()
    c.read(lengths, 117, [0, 37, 37, 117])
    c.attend(lengths, rows(5, 3, 4 * hd), 4, hd ** -0.5, kernel="attention_paged_generic")
    dev.free_all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pad,offset", [(0, 1), (5, 0), (4, 4), (8, 8), (1, 3)])
def test_strides_and_alignments(dev, pad, offset, kind):
    lengths, first = [37, 5], [0, 37, 42]
    c = filled(dev, kind, lengths, 8, 2, 128)
    c.write(lengths, rows(6, 42, 256), rows(7, 42, 256), first, pad, offset)
    c.check()
    c.read(lengths, 42, first, pad, offset)
    c.attend(lengths, rows(8, 2, 512), 4, 0.1, pad, offset)
    other = filled(dev, kind, lengths, 8, 2, 128, offset=2 * offset)
    other.check()
    other.read(lengths, 42, first)
    other.attend(lengths, rows(8, 2, 512), 4, 0.1)
    dev.free_all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lengths,kv,hd", [([17001, 30], 1, 128), ([9, 16500], 2, 64), ([2500, 0, 33, 900], 6, 64), ([2100, 40], 3, 128), ([700, 1, 1200], 24, 128),
                                           ([300], 24, 128), ([1500, 801], 5, 256), ([1] * 500, 2, 128)], ids=str)
def test_any_number_of_rows(dev, lengths, kv, hd, kind):
    c = filled(dev, kind, lengths, 32, kv, hd, extra_columns=1)
    c.check()
    first = np.concatenate([[0], np.cumsum(lengths)])
    c.read(lengths, first[-1] + 1, first)
    new = np.minimum(lengths, 77)
    c.write(lengths, rows(9, new.sum(), kv * hd), rows(10, new.sum(), kv * hd), np.concatenate([[0], np.cumsum(new)]))
    c.check()
    c.read(lengths, first[-1], first)
    dev.free_all()


@pytest.mark.parametrize("kind", KINDS)
def test_more_sequences_than_a_wave_looks_at_in_one_go(dev, kind):
    """Empty, short and long ones on both sides of number 256 and 512, among them some that ranges cut several times"""
    lengths = [(13 * i) % 29 for i in range(600)]
    for g, n in ((3, 2500), (255, 1700), (256, 0), (257, 3100), (511, 900), (599, 2000)):
        lengths[g] = n
    c = filled(dev, kind, lengths, 16, 1, 128)
    c.attend(lengths, rows(11, 600, 3 * 128), 3, 128 ** -0.5, kernel="fa_paged_hd128")
    dev.free_all()


@pytest.mark.parametrize("kind", KINDS)
def test_token_by_token(dev, kind):
    """The newest token of each sequence, first_row NULL: as many calls as tokens give the cache that one call gives"""
    kv, hd, heads, page = 2, 128, 4, 4
    lengths = [9, 5, 12]
    whole = filled(dev, kind, lengths, page, kv, hd)
    c = Cache(dev, kind, whole.pages, page, kv, hd, whole.table)
    k, v, first = rows(1, 26, kv * hd), rows(2, 26, kv * hd), [0, 9, 14, 26]
    for t in range(12):
        now = [min(t + 1, n) for n in lengths]
        at = [first[g] + n - 1 for g, n in enumerate(now)]
        c.write(now, k[at], v[at])
        c.attend(now, rows(t, 3, heads * hd), heads, hd ** -0.5)
    for mine, theirs in ((c.k, whole.k), (c.v, whole.v), (c.ks, whole.ks)):
        assert np.array_equal(mine, theirs)
    c.check()
    c.read(lengths, 3)
    dev.free_all()


@pytest.mark.parametrize("kind", KINDS)
def test_lengths_and_pages_that_are_not_there(dev, kind):
    """Page numbers out of range, lengths below zero and past the table, first rows out of order: nothing outside is read or written"""
    kv, hd, page, pages = 2, 128, 8, 6
    table = [[0, -1, 2], [9, 3, -7], [2 ** 31 - 1, -2 ** 31, 6], [4, 5, 1]]
    c = Cache(dev, kind, pages, page, kv, hd, table)
    lengths = [24, 17, 20, 24]
    c.write(lengths, rows(1, 85, kv * hd), rows(2, 85, kv * hd), [0, 24, 41, 61, 85])
    c.check()
    for n in (lengths, [-3, 10, 2 ** 31 - 1, 99], [25, 2 ** 31 - 1, -2 ** 31, 24]):
        c.attend(n, rows(3, 4, 8 * hd), 8, hd ** -0.5)
    for n, first in (([24, 17, 20, 24], [0, 3, 5, 200, 300]), ([30, -5, 2 ** 31 - 1, 12], [5, 2, 40, 30, 60]), ([2, 17, 0, 24], [0, 20, 40, 60, 85])):
        c.read(n, 70, first)
        c.write(n, rows(4, 70, kv * hd), rows(5, 70, kv * hd), first)
        c.check()
    none = Cache(dev, kind, 0, page, kv, hd, [[0, 1]])
    none.write([3], rows(1, 3, kv * hd), rows(2, 3, kv * hd), [0, 3])
    none.check()
    assert not none.attend([16], rows(3, 1, 2 * hd), 2, 1.0).any()
    dev.free_all()


@pytest.mark.parametrize("kind", KINDS)
def test_a_table_without_columns(dev, kind):
    c = Cache(dev, kind, 3, 16, 1, 128, np.zeros((2, 0)))
    assert not c.attend([5, 0], rows(3, 2, 128), 1, 1.0).any()
    c.write([5, 1], rows(1, 2, 128), rows(2, 2, 128))
    c.check()
    dev.free_all()


@pytest.mark.parametrize("kind", KINDS)
def test_sequences_that_share_pages(dev, kind):
    kv, hd, page = 2, 128, 16
    c = filled(dev, kind, [40, 70], page, kv, hd, extra_columns=3)
    c.table[0, :5] = c.table[1, :5]
    c.dtable = dev.put(c.table)
    c.attend([70, 70], rows(3, 2, 8 * hd), 8, hd ** -0.5)
    c.attend([50, 70], rows(3, 2, 8 * hd), 8, hd ** -0.5)
    dev.free_all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("spread", [1e-3, 30.0])
def test_flat_and_sharp_softmax(dev, spread, kind):
    c = filled(dev, kind, [300, 45], 16, 2, 128, spread=spread)
    c.attend([300, 45], rows(3, 2, 1024), 8, 128 ** -0.5)
    dev.free_all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale", [0.0, -0.2])
def test_scales_that_are_not_positive(dev, scale, kind):
    c = filled(dev, kind, [50, 45], 16, 2, 128)
    c.attend([50, 45], rows(3, 2, 1024), 8, scale, kernel="attention_paged_generic")
    dev.free_all()


@pytest.mark.parametrize("hd", [128, 96])
def test_rounding_at_every_code_and_scale(dev, hd):
    """Rows whose largest value is at and around 448 steps, ties, subnormals, zeros, one-sided rows, all scales, and rows that are not numbers"""
    rng = np.random.default_rng(3)
    out = []
    for e in list(range(-133, 128, 3)) + [-133, -132, -127, -126, -120, -119, -118, 120, 126, 127]:
        for top in (1.0, 1.75, 1.7578125, 1.7421875, 1.9921875):
            x = rng.uniform(-1, 1, hd) * rng.choice([1, 2.0 ** -4, 2.0 ** -9, 2.0 ** -14], hd) * top
            x[rng.integers(hd)] = top
            out.append(np.ldexp(x, e))
    ties = np.concatenate([sr.E4M3[:-1] + np.diff(sr.E4M3) / 2, sr.E4M3, -sr.E4M3])            # halves are bf16 values too
    for e in (-100, -3, 0, 40):
        for at in range(0, len(ties), hd - 1):
            x = np.zeros(hd)
            x[:len(ties[at:at + hd - 1])] = ties[at:at + hd - 1]
            x[-1] = 448
            out.append(np.ldexp(x, e))
    out += [np.zeros(hd), -np.zeros(hd)]
    for bad in (np.inf, -np.inf, np.nan):
        x = rng.uniform(-1, 1, hd)
        x[rng.integers(hd)] = bad
        out.append(x)
    with np.errstate(over="ignore", under="ignore", invalid="ignore"):
        k = sr.bf16_round(np.array(out, np.float32))
    n, page = len(k), 16
    c = Cache(dev, "fp8", -(-n // page), page, 1, hd, [list(range(-(-n // page)))])
    c.write([n], k, k[::-1].copy(), [0, n])
    c.check()
    c.read([n], n, [0, n])
    dev.free_all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("length", [1, 15, 31, 33, 63, 100])
def test_what_lies_behind_the_last_token_has_no_part(dev, length, kind):
    """The cache starts with what is not a number; another sequence's rows follow in the same page"""
    kv, hd, heads = 2, 128, 8
    c = filled(dev, kind, [length], 64, kv, hd)
    c.attend([length], rows(3, 1, heads * hd), heads, hd ** -0.5)
    for shorter in sorted({0, 1, length // 2, length - 1}):
        c.attend([shorter], rows(3, 1, heads * hd), heads, hd ** -0.5)
    dev.free_all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_values_that_are_not_numbers_reach_their_own_sequence(dev, bad, kind):
    kv, hd, heads, lengths = 2, 128, 4, [50, 60, 40]
    c = filled(dev, kind, lengths, 16, kv, hd)
    v = rows(9, 60, kv * hd)
    v[20, 7] = sr.bf16_round(np.float32(bad))
    c.write([50, 60, 40], rows(8, 60, kv * hd), v, [0, 0, 60, 60])
    got = sr.bf16_value(c.attend(lengths, rows(3, 3, heads * hd), heads, hd ** -0.5, compare=False)).reshape(3, heads, hd)
    assert np.isfinite(got[[0, 2]]).all() and np.isfinite(got[1, 2:]).all()
    if kind == "fp8":                                       # the row of the head as a whole
        assert np.isnan(got[1, :2]).all()
    else:
        assert np.isfinite(np.delete(got[1, :2], 7, 1)).all()
        assert np.isnan(got[1, :2, 7]).all() if np.isnan(bad) else (got[1, :2, 7] == bad).all()
    dev.free_all()


@pytest.mark.parametrize("bad", [np.inf, -np.inf])
def test_every_infinity_comes_through_as_itself(dev, bad):
    """One in each row of V, in a dim of its own: whatever the probability of the row, the sum over the keys is that infinity in these dims"""
    kv, hd, heads, n = 1, 128, 16, 100
    c = filled(dev, "bf16", [n], 16, kv, hd)
    v = rows(9, n, kv * hd)
    v[np.arange(n), np.arange(n)] = sr.bf16_round(np.float32(bad))
    c.write([n], rows(8, n, kv * hd), v, [0, n])
    got = sr.bf16_value(c.attend([n], rows(3, 1, heads * hd), heads, hd ** -0.5, compare=False)).reshape(heads, hd)
    assert (got[:, :n] == bad).all() and np.isfinite(got[:, n:]).all()
    dev.free_all()


@pytest.mark.parametrize("kind", KINDS)
def test_a_query_that_is_not_a_number_is_the_only_one(dev, kind):
    c = filled(dev, kind, [50, 60, 40], 16, 2, 128)
    q = rows(3, 3, 8 * 128)
    q[1, 128:256] = 0x7fc0
    got = sr.bf16_value(c.attend([50, 60, 40], q, 8, 0.1, compare=False)).reshape(3, 8, 128)
    assert np.isnan(got[1, 1]).all() and np.isfinite(np.delete(got.reshape(24, 128), 9, 0)).all()
    dev.free_all()


@pytest.mark.parametrize("kind", KINDS)
def test_places_past_32_bits(dev, kind):
    """More than 2^32 elements of K: the last pages of such a cache hold the rows"""
    kv, hd, page, heads = 8, 128, 64, 16
    pages = 2 ** 32 // (kv * page * hd) + 40
    size = 2 if kind == "bf16" else 1
    c = Cache(dev, kind, 1, page, kv, hd, [[pages - 1, 3, pages - 17, pages // 2 + 1], [pages - 2, pages - 3, 0, -1]])
    dk, dv = dev.alloc(pages * kv * page * hd * size), dev.alloc(pages * kv * page * hd * size)
    where = (dk, dv) if kind == "bf16" else (dk, dv, dev.alloc(pages * kv * page), dev.alloc(pages * kv * page))
    lengths, first = [230, 140], [0, 230, 370]
    k, v = rows(1, 370, kv * hd), rows(2, 370, kv * hd)
    dl, df, dt = (dev.put(np.asarray(a, np.int32)) for a in (lengths, first, c.table))
    getattr(dev.lib, "iris_dev_cache_write_" + kind)(*where, pages, page, dt, 4, dl, dev.put(k), dev.put(v), kv * hd, df, 2, 370, kv, hd)
    ko, vo = dev.put(np.zeros_like(k)), dev.put(np.zeros_like(k))
    getattr(dev.lib, "iris_dev_cache_read_" + kind)(ko, vo, kv * hd, *where, pages, page, dt, 4, dl, df, 2, 370, kv, hd)
    dev.check()
    held = []
    for d, x in ((ko, k), (vo, v)):
        want = sr.bf16_value(x).astype(np.float64).reshape(370, kv, hd)
        if kind == "fp8":
            code, scale = sr.quantise(want)
            want = sr.e4m3_value(code) * sr.scale_value(scale)[..., None]
        held.append(want)
        assert np.array_equal(dev.get(d, x.shape, np.uint16), sr.bf16_round(want.reshape(370, -1).astype(np.float32)))
    q = rows(3, 2, heads * hd)
    do = dev.put(np.zeros_like(q))
    getattr(dev.lib, "iris_dev_attention_paged_" + kind)(do, heads * hd, dev.put(q), heads * hd, *where, pages, page, dt, 4, dl, 2, heads, kv, hd, 0.1, None)
    dev.check()
    got = sr.bf16_value(dev.get(do, q.shape, np.uint16)).astype(np.float64).reshape(2, heads, hd)
    for g, (a, b) in enumerate(((0, 230), (230, 370))):
        o, w, s = sr.softmax_rows(sr.bf16_value(q[g:g + 1]).astype(np.float64).reshape(1, heads, hd), held[0][a:b], held[1][a:b], 0.1, [b - a])
        sr.check(got[g:g + 1], (o, sr.bound(o, w, s, hd, True)))
    dev.free_all()


@pytest.mark.parametrize("kind", KINDS)
def test_from_a_graph_with_longer_texts_and_other_pages(dev, kind):
    """A captured step (write the newest token, attend) is replayed while lengths and pages change on the device; eager calls run between"""
    from test_gpu_graph import Graphs
    kv, hd, heads, page = 2, 128, 8, 16
    lengths = [46, 3, 500]
    c = filled(dev, kind, lengths, page, kv, hd)
    c.table[0, 3:5] = [p for p in range(c.pages) if p not in c.table]                # for the token behind its third page
    dev.lib.iris_dev_upload(c.dtable, c.table.ctypes.data, c.table.nbytes)
    dl, dk, dv, dq = dev.put(np.asarray(lengths, np.int32)), dev.alloc(3 * kv * hd * 2), dev.alloc(3 * kv * hd * 2), dev.alloc(3 * heads * hd * 2)
    do, ws = dev.alloc(3 * heads * hd * 2), dev.alloc(dev.lib.iris_dev_attention_paged_workspace() or 16)
    g, stream = Graphs(), C.c_void_p(dev.lib.iris_dev_stream())

    def step():
        getattr(dev.lib, "iris_dev_cache_write_" + kind)(*c.where(), c.pages, page, c.dtable, c.table.shape[1], dl, dk, dv, kv * hd, None, 3, 3, kv, hd)
        getattr(dev.lib, "iris_dev_attention_paged_" + kind)(do, heads * hd, dq, heads * hd, *c.where(), c.pages, page, c.dtable, c.table.shape[1], dl, 3, heads, kv,
                                                             hd, 0.1, ws)
    captured = g.capture(stream, step)
    dev.check()
    for t in range(4):
        lengths = [n + 1 for n in lengths]
        k, v, q = rows(20 + t, 3, kv * hd), rows(40 + t, 3, kv * hd), rows(60 + t, 3, heads * hd)
        for d, a in ((dl, np.asarray(lengths, np.int32)), (dk, k), (dv, v), (dq, q)):
            dev.lib.iris_dev_upload(d, a.ctypes.data, a.nbytes)
        assert g.rt.hipGraphLaunch(captured, stream) == 0
        dev.lib.iris_dev_sync()
        got = dev.get(do, (3, heads * hd), np.uint16)
        c.write(lengths, k, v)                                   # the same rows once more, and the host's image
        c.check()
        assert np.array_equal(got, c.attend(lengths, q, heads, 0.1))
    g.rt.hipGraphExecDestroy(captured)
    dev.free_all()
