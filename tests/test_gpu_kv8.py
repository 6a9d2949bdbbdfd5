"""The 8-bit paged key/value cache on the B200 (strata_kv8_append, strata_kv8_select, strata_kv8_attend)
against plain implementations of their definitions: codes, marks, scales and picks equal, attention
within the rounding bound that tests/kv8_reference.py derives for each row."""
import math

import numpy as np
import pytest

import kv8_reference as R

pytestmark = pytest.mark.gpu
BLOCK = 64


class Cache:
    """A DeviceCache of torch tensors with shuffled pages, filled with what no call should leave there."""

    def __init__(self, kv, dim, sequences, blocks, seed=0, pages=None):
        import torch
        from stratacuda_b200.kv8 import DeviceCache
        self.torch, self.kv, self.dim, self.sequences, self.blocks = torch, kv, dim, sequences, blocks
        self.rng = np.random.default_rng(seed)
        p = R.padded(dim)
        self.pages = sequences * blocks + 2 if pages is None else pages
        dev = dict(device="cuda")
        self.codes = torch.full((self.pages, kv, 2, p * BLOCK), 77, dtype=torch.int8, **dev)
        self.marks = torch.full((self.pages, kv, 2, p), 55, dtype=torch.int8, **dev)
        self.scales = torch.full((self.pages, kv, 2), float("nan"), **dev)
        self.open = torch.full((sequences, 2, BLOCK, kv, dim), float("nan"), **dev)
        order = self.rng.permutation(self.pages)[: sequences * blocks].astype(np.int32)
        self.order = order.reshape(sequences, blocks)
        self.table = torch.from_numpy(self.order.copy()).cuda()
        self.workspace = torch.zeros(32 << 20, dtype=torch.uint8, **dev)
        self.status = torch.zeros(1, dtype=torch.int32, **dev)
        self.view = DeviceCache(kv, dim, self.pages, sequences, blocks, self.codes, self.marks, self.scales, self.open, self.table,
                                self.workspace, self.status)

    def i32(self, values):
        return self.torch.tensor(np.asarray(values), dtype=self.torch.int32, device="cuda")

    def rows(self, x):
        """[..., kv, dim] -> [tokens, kv * dim] on the device"""
        return self.torch.from_numpy(np.ascontiguousarray(x, np.float32).reshape(-1, self.kv * self.dim)).cuda()

    def append(self, k, v, sequence, start):
        """k, v [segments, count, kv, dim]"""
        self.view.append(self.rows(k), self.rows(v), self.i32(sequence), self.i32(start), len(sequence), k.shape[1])

    def attend(self, q, heads, sequence, start, scale=None, picks=None, top=0):
        """q [segments, count, heads, dim] -> y of the same shape"""
        s, n = q.shape[:2]
        dq = self.torch.from_numpy(np.ascontiguousarray(q, np.float32).reshape(s * n, -1)).cuda()
        y = self.torch.full((s * n, heads * self.dim), float("nan"), device="cuda")
        dp = None if picks is None else self.torch.from_numpy(np.ascontiguousarray(picks, np.int32)).cuda()
        self.view.attend(dq, heads, y, self.i32(sequence), self.i32(start), s, n, dp, top, scale)
        return y.cpu().numpy().reshape(s, n, heads, self.dim)

    def select(self, q, heads, sequence, start, top, first=1, last=2):
        s, n = q.shape[:2]
        dq = self.torch.from_numpy(np.ascontiguousarray(q, np.float32).reshape(s * n, -1)).cuda()
        picks = self.torch.full((s * n, self.kv, top), -9, dtype=self.torch.int32, device="cuda")
        self.view.select(dq, heads, picks, self.i32(sequence), self.i32(start), s, n, top, first, last)
        return picks.cpu().numpy().reshape(s, n, self.kv, top)

    def errors(self):
        e = int(self.status.item())
        self.status.zero_()
        return e

    def fill(self, lengths, seed=1, size=1.0):
        """Append `lengths[s]` random rows to each sequence; returns keys, values per sequence [n, kv, dim]."""
        rng = np.random.default_rng(seed)
        ks, vs = [], []
        for s, n in enumerate(lengths):
            k = rng.normal(0, size, (n, self.kv, self.dim)).astype(np.float32)
            v = rng.normal(0, size, (n, self.kv, self.dim)).astype(np.float32)
            if n:
                self.append(k[None], v[None], [s], [0])
            ks.append(k)
            vs.append(v)
        return ks, vs

    def check_blocks(self, s, k, v):
        """The pages of sequence s hold exactly the codes, marks and scales of rows k, v."""
        codes, marks, scales = self.codes.cpu().numpy(), self.marks.cpu().numpy(), self.scales.cpu().numpy()
        for h in range(self.kv):
            for b, (kc, ks, vc, vs) in enumerate(R.blocks_of(k[:, h], v[:, h])):
                page = self.order[s, b]
                assert scales[page, h, 0] == ks and scales[page, h, 1] == vs, (s, h, b)
                assert np.array_equal(codes[page, h, 0], R.pack_keys(kc, self.dim)), (s, h, b)
                assert np.array_equal(codes[page, h, 1], R.pack_values(vc, self.dim)), (s, h, b)
                lo, hi = np.zeros(R.padded(self.dim)), np.zeros(R.padded(self.dim))
                lo[: self.dim], hi[: self.dim] = kc.min(0), kc.max(0)
                assert np.array_equal(marks[page, h, 0], lo) and np.array_equal(marks[page, h, 1], hi), (s, h, b)

    def check_attend(self, got, q, k, v, start, scale, picks=None):
        """got, q [count, heads, dim] of one run against its sequence's rows k, v [n, kv, dim]."""
        count, heads = q.shape[:2]
        group = heads // self.kv
        pos = start + np.arange(count)
        for h in range(self.kv):
            n = k.shape[0]
            allowed = np.arange(n)[None] <= pos[:, None]
            if picks is not None:
                chosen = np.zeros((count, (n + BLOCK - 1) // BLOCK + 1), bool)
                for t in range(count):
                    chosen[t, picks[t, h][picks[t, h] >= 0]] = True
                allowed = allowed & np.repeat(chosen[:, :-1], BLOCK, 1)[:, :n]
            if not n:
                assert not got[:, h * group:(h + 1) * group].any()
                continue
            kd, vd = R.dequantised(R.blocks_of(k[:, h], v[:, h]))
            for g in range(group):
                y, bound = R.attend(q[:, h * group + g], kd, vd, scale, allowed)
                err = np.abs(got[:, h * group + g] - y).max(-1)
                assert (err <= bound + 1e-30).all(), (h, g, err.max(), bound[np.argmax(err - bound)])


# ---------------------------------------------------------------- append

@pytest.mark.parametrize("kv,dim", [(1, 1), (2, 8), (3, 64), (2, 80), (1, 128), (4, 130), (2, 256)])
def test_append_is_its_rows_whatever_the_split(kv, dim):
    n = 64 * 3 + 21
    rng = np.random.default_rng(dim)
    k = rng.normal(0, 1, (n, kv, dim)).astype(np.float32)
    v = (rng.normal(0, 1, (n, kv, dim)) * np.exp(rng.normal(0, 2, (n, 1, 1)))).astype(np.float32)
    for split in ([n], [64, 64, 64, 21], [1] * n, [7, 90, 1, 1, 62, n - 161], [63, 1, 128, 21]):
        c = Cache(kv, dim, 1, 4)
        at = 0
        for m in split:
            c.append(k[None, at:at + m], v[None, at:at + m], [0], [at])
            at += m
        assert at == n and c.errors() == 0
        c.check_blocks(0, k, v)
        held = c.open.cpu().numpy()[0]
        assert np.array_equal(held[0, :21], k[192:]) and np.array_equal(held[1, :21], v[192:])


def test_append_many_sequences_and_idle_slots():
    kv, dim, lengths = 2, 72, [0, 1, 63, 64, 65, 130, 5]
    c = Cache(kv, dim, len(lengths), 4)
    ks, vs = c.fill(lengths)
    rng = np.random.default_rng(5)
    for step in range(3):  # one token each, in another order, with idle slots between
        slots = [6, -1, 3, 2, 1, -1, 5, 4]
        k = rng.normal(0, 1 + step, (len(slots), 1, kv, dim)).astype(np.float32)
        v = rng.normal(0, 1, k.shape).astype(np.float32)
        c.append(k, v, slots, [len(ks[s]) if s >= 0 else -5 for s in slots])
        for i, s in enumerate(slots):
            if s >= 0:
                ks[s], vs[s] = np.concatenate([ks[s], k[i]]), np.concatenate([vs[s], v[i]])
    k = rng.normal(0, 1, (3, 100, kv, dim)).astype(np.float32)  # prompts of three sequences in one call
    v = rng.normal(0, 1, k.shape).astype(np.float32)
    c.append(k, v, [0, 5, 2], [len(ks[s]) for s in (0, 5, 2)])
    for i, s in enumerate((0, 5, 2)):
        ks[s], vs[s] = np.concatenate([ks[s], k[i]]), np.concatenate([vs[s], v[i]])
    assert c.errors() == 0
    for s in range(len(lengths)):
        c.check_blocks(s, ks[s], vs[s])
    untouched = np.setdiff1d(np.arange(c.pages), [c.order[s, b] for s in range(len(lengths)) for b in range((len(ks[s]) + 63) // 64)])
    assert (c.codes.cpu().numpy()[untouched] == 77).all() and (c.marks.cpu().numpy()[untouched] == 55).all()


@pytest.mark.parametrize("size", [0.0, 1e-44, 2.0 ** -101, 2.0 ** -99, 3e38])
def test_append_extreme_magnitudes(size):
    c = Cache(1, 40, 1, 2)
    rng = np.random.default_rng(2)
    k = (rng.uniform(-1, 1, (70, 1, 40)) * size).astype(np.float32)
    k[3, 0, 1] = size
    v = k[::-1].copy()
    for at in range(0, 70, 10):
        c.append(k[None, at:at + 10], v[None, at:at + 10], [0], [at])
    c.check_blocks(0, k, v)


def test_append_restarts_a_block_and_keeps_a_smaller_rows_scale():
    c = Cache(1, 64, 1, 2)
    ks, vs = c.fill([50], size=9.0)
    k2, v2 = np.ones((3, 1, 64), np.float32), np.full((3, 1, 64), 0.5, np.float32)
    c.append(k2[None], v2[None], [0], [0])  # the session starts over
    c.check_blocks(0, k2, v2)


def test_append_reports_what_it_leaves_out():
    c = Cache(2, 16, 2, 2)
    x = np.ones((1, 1, 2, 16), np.float32)
    before = c.codes.clone()
    for seq, start in ((2, 0), (-7, 0), (0, 128), (0, -3)):
        c.append(x, x, [seq], [start])
        assert c.errors() == 1, (seq, start)
    c.table[0, 1] = 99
    c.append(x, x, [0], [64])
    assert c.errors() == 1
    assert c.torch.equal(before, c.codes)
    # past the table's end: the tokens that fit go in
    k = np.random.default_rng(0).normal(0, 1, (1, 130, 2, 16)).astype(np.float32)
    c.append(k, k, [1], [0])
    assert c.errors() == 1
    c.check_blocks(1, k[0, :128], k[0, :128])
    # a value that is not finite counts as zero
    k = k[:, :64].copy()
    k[0, 5, 1, 3], k[0, 9, 0, 0] = np.nan, np.inf
    c.append(k, k, [1], [0])
    assert c.errors() == 16
    c.check_blocks(1, np.where(np.isfinite(k[0]), k[0], 0), np.where(np.isfinite(k[0]), k[0], 0))


# ---------------------------------------------------------------- attend

@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 1), (4, 2, 8), (5, 1, 64), (16, 16, 64), (6, 2, 80), (32, 8, 128), (24, 2, 256), (17, 1, 256),
                                          (40, 1, 100), (3, 3, 200)])
def test_attend_single_tokens(heads, kv, dim):
    """One token each of sequences of every length from one on, an idle slot, one that sees nothing yet."""
    lengths = [1, 2, 63, 64, 65, 129, 640, 1000]
    c = Cache(kv, dim, len(lengths), 16, seed=dim)
    ks, vs = c.fill(lengths)
    slots = [7, 0, -1, 5, 1, 2, 3, 4, 6, 3]
    start = [lengths[s] - 1 if s >= 0 else 4 for s in slots]
    start[-1] = -1  # no key at or before it
    q = np.random.default_rng(1).normal(0, 1, (len(slots), 1, heads, dim)).astype(np.float32)
    got = c.attend(q, heads, slots, start)
    assert c.errors() == 0
    for i, s in enumerate(slots):
        if s < 0 or start[i] < 0:
            assert not got[i].any()
        else:
            c.check_attend(got[i], q[i], ks[s], vs[s], start[i], 1 / math.sqrt(dim))


@pytest.mark.parametrize("heads,kv,dim,start,count", [(24, 2, 256, 0, 150), (24, 2, 256, 333, 77), (16, 16, 64, 100, 129), (5, 1, 40, 0, 300),
                                                      (8, 2, 128, 60, 5), (4, 2, 8, 0, 17), (33, 1, 96, 511, 65), (2, 1, 256, 1, 640),
                                                      (9, 3, 128, 130, 200)])
def test_attend_prompt(heads, kv, dim, start, count):
    c = Cache(kv, dim, 2, 12, seed=count)
    ks, vs = c.fill([3, start + count])
    q = np.random.default_rng(2).normal(0, 1, (1, count, heads, dim)).astype(np.float32)
    got = c.attend(q, heads, [1], [start])
    c.check_attend(got[0], q[0], ks[1], vs[1], start, 1 / math.sqrt(dim))
    assert c.errors() == 0


def test_attend_prompts_of_several_sequences():
    """Runs of one call at their own positions; one is idle, one begins before its first key."""
    heads, kv, dim, count = 12, 2, 128, 90
    c = Cache(kv, dim, 4, 5)
    ks, vs = c.fill([90, 200, 95, 300])
    slots, start = [3, 0, -1, 1, 2], [210, 0, 7, 110, -30]
    q = np.random.default_rng(3).normal(0, 1, (5, count, heads, dim)).astype(np.float32)
    got = c.attend(q, heads, slots, start)
    assert c.errors() == 0
    for i, s in enumerate(slots):
        if s < 0:
            assert not got[i].any()
        else:
            c.check_attend(got[i], q[i], ks[s], vs[s], start[i], 1 / math.sqrt(dim))


@pytest.mark.parametrize("count", [1, 70])
def test_attend_ignores_what_is_masked(count):
    """Codes, scales and pages past a token's position change nothing, whatever they hold."""
    heads, kv, dim = 6, 2, 128
    c = Cache(kv, dim, 1, 6)
    ks, vs = c.fill([64 * 3 + 10 + count])
    q = np.random.default_rng(4).normal(0, 1, (1, count, heads, dim)).astype(np.float32)
    want = c.attend(q, heads, [0], [64 * 3 + 10])
    last = c.order[0, (64 * 3 + 10 + count - 1) // 64]
    end = (64 * 3 + 10 + count) % 64
    k = c.codes[last, :, 0].reshape(kv, -1, BLOCK, 64)
    k[:, :, end:] = -128
    c.codes[last, :, 1].reshape(kv, -1, BLOCK)[:, :, end:] = 127
    for b in range((64 * 3 + 10 + count + 63) // 64, 6):
        c.scales[c.order[0, b]] = float("nan")
        c.table[0, b] = -1
    got = c.attend(q, heads, [0], [64 * 3 + 10])
    assert np.array_equal(got.view(np.uint32), want.view(np.uint32)) and c.errors() == 0


@pytest.mark.parametrize("count", [1, 40])
def test_attend_large_logits_and_uneven_scales(count):
    """Logits far apart, blocks whose value or key scales differ by many orders, blocks of zeros."""
    heads, kv, dim = 4, 2, 64
    rng = np.random.default_rng(6)
    n = 64 * 6 + count
    size_k, size_v = np.array([1, 30, 0, 1e-3, 8, 1, 1])[np.arange(n) // 64], np.array([1, 1e-6, 1e4, 0, 1e-20, 1, 1])[np.arange(n) // 64]
    k = (rng.normal(0, 1, (n, kv, dim)) * size_k[:, None, None]).astype(np.float32)
    v = (rng.normal(0, 1, (n, kv, dim)) * size_v[:, None, None]).astype(np.float32)
    c = Cache(kv, dim, 1, 8)
    c.append(k[None], v[None], [0], [0])
    q = rng.normal(0, 3, (1, count, heads, dim)).astype(np.float32)
    got = c.attend(q, heads, [0], [n - count])
    c.check_attend(got[0], q[0], k, v, n - count, 1 / math.sqrt(dim))
    # all values as large as they come
    got = c.attend(q * 0, heads, [0], [n - count], scale=1.0)
    c.check_attend(got[0], q[0] * 0, k, v, n - count, 1.0)


@pytest.mark.parametrize("count", [1, 50])
def test_attend_a_query_that_is_not_finite_spoils_its_own_row(count):
    heads, kv, dim = 6, 2, 128
    c = Cache(kv, dim, 1, 6)
    c.fill([200 + count])
    q = np.random.default_rng(4).normal(0, 1, (1, count, heads, dim)).astype(np.float32)
    want = c.attend(q, heads, [0], [200])
    for bad in (np.nan, np.inf):
        p = q.copy()
        p[0, count // 2, 3, 17] = bad
        got = c.attend(p, heads, [0], [200])
        assert np.isnan(got[0, count // 2, 3]).all()
        got[0, count // 2, 3] = want[0, count // 2, 3]
        assert np.array_equal(got.view(np.uint32), want.view(np.uint32))


def test_attend_extreme_queries():
    """Queries near the ends of F32's range: small ones give an even average, large ones a single key."""
    heads, kv, dim = 2, 1, 32
    c = Cache(kv, dim, 1, 2)
    ks, vs = c.fill([100])
    for size in (1e-38, 1e30):
        q = (np.random.default_rng(8).normal(0, 1, (1, 1, heads, dim)) * size).astype(np.float32)
        got = c.attend(q, heads, [0], [99], scale=1.0 if size < 1 else 1e-25)
        c.check_attend(got[0], q[0], ks[0], vs[0], 99, 1.0 if size < 1 else 1e-25)


def test_attend_reports_bad_sequences_pages_and_positions():
    c = Cache(1, 16, 2, 3)
    ks, vs = c.fill([150, 150])
    q = np.ones((1, 1, 2, 16), np.float32)
    assert not c.attend(q, 2, [5], [10]).any() and c.errors() == 1
    got = c.attend(q, 2, [0], [1000])  # past the table: the keys there are (garbage codes past 150 are finite)
    assert c.errors() == 1 and got.shape == q.shape
    c.table[1, 1] = 12345
    got = c.attend(q, 2, [1], [149])  # the block without a page is left out
    assert c.errors() == 1
    c.check_attend(got[0], q[0], ks[1], vs[1], 149, 0.25, picks=np.array([[[0, 2]]]))


def test_attend_strided_unaligned_queries_and_rows():
    """Rows wider apart than they are long and starting off the 16-byte grid."""
    import torch
    heads, kv, dim = 4, 2, 72
    for count, off in ((1, 1), (45, 3)):
        c = Cache(kv, dim, 1, 4)
        rng = np.random.default_rng(9)
        n = 100 + count
        k, v = rng.normal(0, 1, (2, n, kv, dim)).astype(np.float32)
        wide = torch.zeros(2, n * (kv * dim + 5) + 7, device="cuda")
        rows = wide[:, off:off + n * (kv * dim + 5)].reshape(2, n, kv * dim + 5)
        rows[0, :, :kv * dim] = torch.from_numpy(k.reshape(n, -1)).cuda()
        rows[1, :, :kv * dim] = torch.from_numpy(v.reshape(n, -1)).cuda()
        c.view.append(rows[0], rows[1], c.i32([0]), c.i32([0]), 1, n, row_stride=kv * dim + 5)
        c.check_blocks(0, k, v)
        q = rng.normal(0, 1, (1, count, heads, dim)).astype(np.float32)
        wide = torch.zeros(count * (heads * dim + 3) + 8, device="cuda")
        dq = wide[off:off + count * (heads * dim + 3)].reshape(count, heads * dim + 3)
        dq[:, :heads * dim] = torch.from_numpy(q.reshape(count, -1)).cuda()
        y = torch.zeros(count * heads * dim + 1, device="cuda")[1:]
        c.view.attend(dq, heads, y, c.i32([0]), c.i32([100]), 1, count, row_stride=heads * dim + 3)
        c.check_attend(y.cpu().numpy().reshape(count, heads, dim), q[0], k, v, 100, 1 / math.sqrt(dim))


def test_attend_long_single_sequence_repeats_bit_for_bit():
    heads, kv, dim, n = 12, 2, 128, 20011
    c = Cache(kv, dim, 1, 313)
    ks, vs = c.fill([n])
    q = np.random.default_rng(3).normal(0, 1, (1, 1, heads, dim)).astype(np.float32)
    got = c.attend(q, heads, [0], [n - 1])
    c.check_attend(got[0], q[0], ks[0], vs[0], n - 1, 1 / math.sqrt(dim))
    for _ in range(3):
        assert np.array_equal(c.attend(q, heads, [0], [n - 1]).view(np.uint32), got.view(np.uint32))


def test_attend_many_uneven_sequences():
    """More sequences than multiprocessors, from one token to thousands, some idle."""
    heads, kv, dim = 4, 1, 64
    rng = np.random.default_rng(12)
    lengths = [int(x) for x in np.exp(rng.uniform(0, 7.5, 400))]
    lengths[17] = 5000
    c = Cache(kv, dim, 400, 80)
    ks, vs = c.fill(lengths)
    slots = rng.permutation(400)
    slots[::37] = -1
    q = rng.normal(0, 1, (400, 1, heads, dim)).astype(np.float32)
    got = c.attend(q, heads, slots, [lengths[s] - 1 if s >= 0 else 0 for s in slots])
    for i, s in enumerate(slots):
        if s < 0:
            assert not got[i].any()
        else:
            c.check_attend(got[i], q[i], ks[s], vs[s], lengths[s] - 1, 1 / 8)


def test_offsets_past_32_bits():
    """A pool whose last pages lie more than 4 GiB in."""
    kv, dim = 8, 256
    c = Cache(kv, dim, 1, 4, pages=18000)
    c.order[0] = [17999, 3, 17998, 16500]
    c.table.copy_(c.torch.from_numpy(c.order))
    ks, vs = c.fill([230])
    assert c.codes.numel() > 1 << 32
    page = c.order[0, 2]
    kc, kscale, _, _ = R.blocks_of(ks[0][:, 7], vs[0][:, 7])[2]
    assert np.array_equal(c.codes[page, 7, 0].cpu().numpy(), R.pack_keys(kc, dim)) and float(c.scales[page, 7, 0]) == kscale
    for count in (1, 60):
        q = np.random.default_rng(3).normal(0, 1, (1, count, 16, dim)).astype(np.float32)
        got = c.attend(q, 16, [0], [230 - count])
        c.check_attend(got[0], q[0], ks[0], vs[0], 230 - count, 1 / 16)
    assert c.errors() == 0


# ---------------------------------------------------------------- select, and attention over what it picks

def _want_picks(c, ks, vs, q, heads, s, start, top, first, last):
    count, group = q.shape[0], heads // c.kv
    out = np.full((count, c.kv, top), -1, np.int32)
    for h in range(c.kv):
        for t in range(count):
            see = start + t + 1
            have = (see + 63) // 64
            if s < 0 or have <= 0:
                continue
            blocks = R.blocks_of(ks[s][:, h], vs[s][:, h])[:have]
            lo, hi = np.stack([b[0].min(0) for b in blocks]), np.stack([b[0].max(0) for b in blocks])
            got = R.select(q[t, h * group:(h + 1) * group], (lo, hi), np.array([b[1] for b in blocks]), have, top, first, last)
            out[t, h, : len(got)] = got
    return out


@pytest.mark.parametrize("heads,kv,dim,top,first,last", [(24, 2, 256, 8, 1, 2), (4, 4, 64, 5, 0, 0), (6, 2, 80, 3, 1, 1), (16, 1, 128, 30, 2, 3),
                                                         (2, 1, 8, 1, 0, 1), (3, 1, 1, 7, 0, 7)])
def test_select_single_tokens(heads, kv, dim, top, first, last):
    lengths = [1, 64 * 8, 64 * 8 + 1, 1999, 700]
    c = Cache(kv, dim, len(lengths), 32, seed=top)
    ks, vs = c.fill(lengths)
    slots = [3, -1, 0, 1, 2, 4]
    start = [lengths[s] - 1 if s >= 0 else 0 for s in slots]
    q = np.random.default_rng(1).normal(0, 1, (len(slots), 1, heads, dim)).astype(np.float32)
    got = c.select(q, heads, slots, start, top, first, last)
    for i, s in enumerate(slots):
        assert np.array_equal(got[i], _want_picks(c, ks, vs, q[i], heads, s, start[i], top, first, last)), (i, s)
    assert c.errors() == 0


@pytest.mark.parametrize("heads,kv,dim,count", [(24, 2, 256, 70), (5, 1, 40, 33), (8, 4, 128, 200)])
def test_select_and_sparse_prompt(heads, kv, dim, count):
    c = Cache(kv, dim, 2, 40, seed=4)
    ks, vs = c.fill([10, 2000])
    start = 2000 - count
    q = np.random.default_rng(7).normal(0, 1, (1, count, heads, dim)).astype(np.float32)
    picks = c.select(q, heads, [1], [start], 6)
    assert np.array_equal(picks[0], _want_picks(c, ks, vs, q[0], heads, 1, start, 6, 1, 2))
    got = c.attend(q, heads, [1], [start], picks=picks, top=6)
    c.check_attend(got[0], q[0], ks[1], vs[1], start, 1 / math.sqrt(dim), picks=picks[0])


def test_select_ties_go_to_the_lower_block():
    c = Cache(1, 16, 1, 20)
    row = np.random.default_rng(0).normal(0, 1, (64, 1, 16)).astype(np.float32)
    k = np.concatenate([row] * 20)
    c.append(k[None], k[None], [0], [0])
    q = np.random.default_rng(1).normal(0, 1, (1, 1, 2, 16)).astype(np.float32)
    assert c.select(q, 2, [0], [64 * 20 - 1], 5, 0, 0)[0, 0, 0].tolist() == [0, 1, 2, 3, 4]
    assert c.select(q, 2, [0], [64 * 20 - 1], 5, 1, 2)[0, 0, 0].tolist() == [0, 1, 2, 18, 19]
    assert c.select(q * 0, 2, [0], [64 * 20 - 1], 4, 0, 1)[0, 0, 0].tolist() == [0, 1, 2, 19]
    bad = q.copy()
    bad[0, 0, :, :] = np.nan
    assert c.select(bad, 2, [0], [64 * 20 - 1], 4, 0, 1)[0, 0, 0].tolist() == [0, 1, 2, 19]


def test_sparse_rows_that_are_empty_or_partly_listed():
    """No block at all, only blocks past the token, single blocks, -1 between blocks."""
    heads, kv, dim = 6, 2, 128
    c = Cache(kv, dim, 1, 8)
    ks, vs = c.fill([500])
    q = np.random.default_rng(7).normal(0, 1, (1, 5, heads, dim)).astype(np.float32)
    picks = np.full((5, kv, 4), -1, np.int32)
    picks[1, 0], picks[2, 1], picks[3, 0], picks[3, 1] = [7, -1, -1, -1], [-1, 3, -1, 0], [5, 2, 1, 0], [-1, -1, -1, 6]
    picks[4] = [7, 6, 3, -1]
    start = 64 * 7 - 4  # tokens 0 .. 3 end in block 6, token 4 opens block 7
    got = c.attend(q, heads, [0], [start], picks=picks, top=4)
    assert not got[0, 0].any() and not got[0, 1].any() and not got[0, 2, :3].any()
    c.check_attend(got[0], q[0], ks[0], vs[0], start, 1 / math.sqrt(dim), picks=picks)
    assert c.errors() == 0


def test_every_block_picked_is_dense_attention():
    heads, kv, dim = 8, 2, 96
    c = Cache(kv, dim, 1, 8)
    c.fill([480])
    q = np.random.default_rng(7).normal(0, 1, (1, 1, heads, dim)).astype(np.float32)
    picks = np.broadcast_to(np.arange(8, dtype=np.int32), (1, kv, 8))
    assert np.array_equal(c.attend(q, heads, [0], [479], picks=picks, top=8).view(np.uint32), c.attend(q, heads, [0], [479]).view(np.uint32))


# ---------------------------------------------------------------- streams, graphs, handles

def test_another_stream_than_the_default():
    import torch
    heads, kv, dim = 8, 2, 128
    c = Cache(kv, dim, 1, 40)
    ks, vs = c.fill([2500])
    q = torch.randn(1, heads * dim, device="cuda")
    y0, y1 = torch.zeros(1, heads * dim, device="cuda"), torch.zeros(1, heads * dim, device="cuda")
    seq, start = c.i32([0]), c.i32([2499])
    c.view.attend(q, heads, y0, seq, start)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for _ in range(20):
            q2 = q + 0  # produced on that stream just before
            c.view.attend(q2, heads, y1, seq, start, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(y0, y1)


def test_handles_graph_replay_and_device_errors():
    """Kv8Cache on the backend's stream: the append, selection and attention of a decode step captured once and
    replayed with other positions gives what eager calls give; bad indices come with the next read."""
    from stratacuda_b200.backend import CudaBackend, StrataError
    from stratacuda_b200.kv8 import Kv8Cache
    heads, kv, dim, n, top = 8, 2, 64, 700, 4
    rng = np.random.default_rng(1)
    k, v = rng.normal(0, 1, (2, n + 8, kv * dim)).astype(np.float32)
    qs = rng.normal(0, 1, (8, heads * dim)).astype(np.float32)
    with CudaBackend(0) as b:
        def session():
            c = Kv8Cache(b, kv, dim, 2, 16)
            seq, start = b.alloc(np.array([1], np.int32), "i32"), b.alloc(np.array([0], np.int32), "i32")
            c.append(b.alloc(k[:n]), b.alloc(v[:n]), seq, start, 1, n)
            bufs = [b.alloc(kv * dim), b.alloc(kv * dim), b.alloc(heads * dim), b.alloc(kv * top, "i32"), b.alloc(heads * dim)]

            def step():
                c.append(bufs[0], bufs[1], seq, start)
                c.select(bufs[2], heads, bufs[3], seq, start, top=top)
                c.attend(bufs[2], heads, bufs[4], seq, start, picks=bufs[3], top=top)

            def feed(i):
                for buf, x in zip(bufs, (k[n + i], v[n + i], qs[i])):
                    b.write(buf, x)
                b.write(start, np.array([n + i], np.int32))
            return c, step, feed, bufs
        c, step, feed, bufs = session()
        want = []
        for i in range(8):
            feed(i)
            step()
            want.append((b.read(bufs[3]), b.read(bufs[4])))
        c2, step2, feed2, bufs2 = session()
        feed2(0)
        step2()
        b.capture_begin()
        step2()
        graph = b.capture_end()
        for i in range(8):
            feed2(i)
            b.graph_launch(graph)
            assert np.array_equal(b.read(bufs2[3]), want[i][0])
            assert np.array_equal(b.read(bufs2[4]).view(np.uint32), want[i][1].view(np.uint32))
        b.graph_free(graph)
        seq, start = b.alloc(np.array([9], np.int32), "i32"), b.alloc(np.array([0], np.int32), "i32")
        c.append(bufs[0], bufs[1], seq, start)
        with pytest.raises(StrataError, match="index outside"):
            b.idle()
        b.write(bufs[0], np.full(kv * dim, np.nan, np.float32))
        b.write(seq, np.array([0], np.int32))
        c.append(bufs[0], bufs[1], seq, start)
        with pytest.raises(StrataError, match="Non-finite key or value"):
            b.idle()
        with pytest.raises(StrataError, match="needs"):
            c.attend(bufs[2], heads * 2, bufs[4], seq, start)
        with pytest.raises(StrataError, match="needs"):
            c.append(bufs[0], bufs[1], seq, start, 1, 2)
        with pytest.raises(StrataError, match="divisible"):
            c.attend(bufs[2], 7, bufs[4], seq, start)
        with pytest.raises(StrataError, match="live buffer"):
            from stratacuda_b200.backend import Buffer
            c.attend(bufs[2], heads, Buffer(b, 123456, 4, "f32"), seq, start)
        b.idle()


# ---------------------------------------------------------------- later additions
@pytest.mark.parametrize("kv,dim", [(1, 16), (2, 96), (2, 256)])
def test_append_again_from_inside_an_open_block(kv, dim):
    """A run that starts inside the open block takes the place of its rows from there on: scale, codes and marks are
    those of the rows that remain and the new ones, also where a dropped row had set the scale or a mark."""
    c = Cache(kv, dim, 1, 2)
    rng = np.random.default_rng(4)
    k, v = (rng.normal(0, 1, (40, kv, dim)).astype(np.float32) for _ in range(2))
    c.append(k[None], v[None], [0], [0])
    for at, rows, size in ((38, 2, 1.0), (30, 1, 50.0), (30, 1, 0.01), (29, 3, 1.0), (10, 2, 1e-3)):
        k2, v2 = (rng.normal(0, size, (rows, kv, dim)).astype(np.float32) for _ in range(2))
        c.append(k2[None], v2[None], [0], [at])
        k, v = np.concatenate([k[:at], k2]), np.concatenate([v[:at], v2])
        page, p = c.order[0, 0], R.padded(dim)
        for h in range(kv):
            keys = c.codes[page, h, 0].cpu().numpy().reshape(p // 64, BLOCK, 64).transpose(1, 0, 2).reshape(BLOCK, p)
            values = c.codes[page, h, 1].cpu().numpy().reshape(p, BLOCK).T
            for kind, (got, x) in enumerate(((keys, k), (values, v))):
                want, scale = R.quantise(x[:, h])
                assert c.scales[page, h, kind].item() == scale, (at, h, kind)
                np.testing.assert_array_equal(got[:at + rows, :dim], want)
                if kind == 0:
                    np.testing.assert_array_equal(c.marks[page, h].cpu().numpy()[:, :dim], [want.min(0), want.max(0)])


class WideCache(Cache):
    """A cache whose table has room for more blocks than there are pages; the test fills the table."""

    def __init__(self, kv, dim, sequences, blocks, pages):
        from stratacuda_b200.kv8 import DeviceCache
        super().__init__(kv, dim, 1, pages - 2)
        self.sequences, self.blocks = sequences, blocks
        self.open = self.torch.full((sequences, 2, BLOCK, kv, dim), float("nan"), device="cuda")
        self.table = self.torch.full((sequences, blocks), -1, dtype=self.torch.int32, device="cuda")
        self.view = DeviceCache(kv, dim, self.pages, sequences, blocks, self.codes, self.marks, self.scales, self.open, self.table,
                                self.workspace, self.status)


def _rising(rng, n, kv, dim, q, slope):
    """Keys whose logits with the queries' common direction rise by about `slope` (log2) every 128 tokens, and values whose
    blocks differ in size."""
    k = rng.normal(0, 0.2, (n, kv, dim))
    direction = q / np.sum(q * q)
    k += (np.arange(n) / 128 * slope * math.log(2) * math.sqrt(dim))[:, None, None] * direction
    v = rng.normal(0, 1, (n, kv, dim)) * 2.0 ** rng.integers(-3, 4, (n + 63) // 64).repeat(64)[:n, None, None]
    return k.astype(np.float32), v.astype(np.float32)


@pytest.mark.parametrize("heads,kv,dim", [(5, 1, 64), (16, 2, 96), (12, 1, 256), (17, 1, 40)])
@pytest.mark.parametrize("slope", [0.0, 2.5, 5.0, 7.5, 30.0, -6.0])
def test_attend_long_lists_with_a_rising_maximum(heads, kv, dim, slope):
    """Sequences of some dozens of pages, all of one sequence's, and short ones between them: units that begin and end
    anywhere in a CTA's list, and whose references have to move by little and by much."""
    sequences, n, short, blocks = 96, 64 * 45 + 17, 70, 46
    c = WideCache(kv, dim, sequences, blocks, blocks + 2)
    rng = np.random.default_rng(8)
    direction = rng.normal(0, 1, dim)
    k, v = _rising(rng, n, kv, dim, direction, slope)
    c.table[:] = c.i32(np.arange(blocks))
    c.append(k[None], v[None], [0], [0])
    q = (direction + rng.normal(0, 0.05, (sequences, 1, heads, dim))).astype(np.float32)
    start = np.where(np.arange(sequences) % 5 == 3, short - 1, n - 1 - np.arange(sequences))
    got = c.attend(q, heads, np.arange(sequences), start)
    # the same lists as picks
    picks = np.arange(blocks)[None, None].repeat(kv, 1).repeat(sequences, 0)
    picks = np.where(picks <= (start // BLOCK)[:, None, None], picks, -1)
    again = c.attend(q, heads, np.arange(sequences), start, picks=picks, top=blocks)
    for s in (0, 1, 3, 31, 32, 50, 95):
        for y in (got, again):
            c.check_attend(y[s], q[s], k, v, start[s], 1 / math.sqrt(dim))
    assert c.errors() == 0


def test_attend_more_steps_than_whole_number_sums_hold():
    """A unit of more than 256 pages on one CTA: its whole-number sums have to move on the way."""
    kv, dim, heads, n = 1, 16, 2, 64 * 300
    sequences = 160  # as many units as keep a unit on one CTA or two
    c = WideCache(kv, dim, sequences, 300, 300)
    rng = np.random.default_rng(9)
    k = rng.normal(0, 0.05, (n, kv, dim)).astype(np.float32)
    v = rng.normal(1, 0.01, (n, kv, dim)).astype(np.float32)
    c.table[:] = c.i32(np.arange(300))
    c.append(k[None], v[None], [0], [0])
    q = rng.normal(0, 1, (sequences, 1, heads, dim)).astype(np.float32)
    got = c.attend(q, heads, np.arange(sequences), np.full(sequences, n - 1))
    for s in (0, 1, 77, 159):
        c.check_attend(got[s], q[s], k, v, n - 1, 1 / math.sqrt(dim))


def test_sparse_prompt_of_more_tokens_than_are_counted_up():
    kv, dim, heads, count, top = 1, 24, 3, 1100, 5
    c = Cache(kv, dim, 1, 18)
    ks, vs = c.fill([count])
    rng = np.random.default_rng(3)
    q = rng.normal(0, 1, (1, count, heads, dim)).astype(np.float32)
    picks = np.full((1, count, kv, top), -1, np.int32)
    for t in range(count):
        have = rng.permutation(t // 64 + 1)[:top]
        picks[0, t, 0, :len(have)] = np.sort(have)
    got = c.attend(q, heads, [0], [0], picks=picks.reshape(count, kv, top), top=top)
    c.check_attend(got[0], q[0], ks[0], vs[0], 0, 1 / math.sqrt(dim), picks[0])


@pytest.mark.parametrize("heads,kv,dim,count", [(1, 1, 64, 130), (6, 2, 96, 64), (12, 1, 256, 40)])
@pytest.mark.parametrize("slope", [0.0, 3.0, 9.0, -6.0])
def test_attend_prompt_after_many_pages(heads, kv, dim, count, slope):
    """More pages than add up in one accumulator, on as few CTAs as there are units' pages to share."""
    c = Cache(kv, dim, 1, 90)
    rng = np.random.default_rng(12)
    direction = rng.normal(0, 1, dim)
    n = 64 * 88 + 11
    k, v = _rising(rng, n, kv, dim, direction, slope)
    c.append(k[None], v[None], [0], [0])
    q = (direction + rng.normal(0, 0.05, (1, count, heads, dim))).astype(np.float32)
    got = c.attend(q, heads, [0], [n - count])
    c.check_attend(got[0], q[0], k, v, n - count, 1 / math.sqrt(dim))
    assert c.errors() == 0


@pytest.mark.parametrize("dim,segments,count,blocks", [(16, 300, 70, 3), (256, 40, 70, 40)])
def test_attend_prompts_of_many_sequences(dim, segments, count, blocks):
    """Whole units a CTA (many sequences), and long lists that one CTA walks over more than one accumulator."""
    kv = 4 if segments > 100 else 2
    c = Cache(kv, dim, segments, blocks) if segments > 100 else WideCache(kv, dim, segments, blocks, blocks + 2)
    rng = np.random.default_rng(6)
    n = 64 * blocks - 20
    if segments <= 100:  # all read one sequence's pages
        c.table[:] = c.i32(np.arange(blocks))
        ks, vs = c.fill([n])
        ks, vs = ks * segments, vs * segments
    else:
        ks, vs = c.fill([n] * segments)
    q = rng.normal(0, 1, (segments, count, kv, dim)).astype(np.float32)
    start = [(n - count) - (i % 7) for i in range(segments)]
    got = c.attend(q, kv, np.arange(segments), start)
    for s in range(0, segments, 13):
        c.check_attend(got[s], q[s], ks[s], vs[s], start[s], 1 / math.sqrt(dim))
    assert c.errors() == 0


@pytest.mark.parametrize("heads,kv,dim", [(16, 1, 128), (16, 1, 256), (33, 1, 100), (3, 1, 200)])
@pytest.mark.parametrize("slope", [0.5, 5.0, 12.0, -6.0])
def test_attend_groups_of_many_heads_in_wide_tables(heads, kv, dim, slope):
    """Tables with room for long sessions, as many of whose blocks as a session has are read: 16 rows a unit, and units of
    16 and of fewer rows side by side (33 heads)."""
    sequences, n, used = 70, 64 * 20 + 3, 21
    c = WideCache(kv, dim, sequences, 500, used + 2)
    rng = np.random.default_rng(10)
    direction = rng.normal(0, 1, dim)
    k, v = _rising(rng, n, kv, dim, direction, slope)
    c.table[:, :used] = c.i32(np.arange(used))
    c.append(k[None], v[None], [0], [0])
    q = (direction + rng.normal(0, 0.05, (sequences, 1, heads, dim))).astype(np.float32)
    start = n - 1 - 3 * np.arange(sequences)
    start[5] = 0
    got = c.attend(q, heads, np.arange(sequences), start)
    for s in (0, 5, 6, 41, 69):
        c.check_attend(got[s], q[s], k, v, start[s], 1 / math.sqrt(dim))
    assert c.errors() == 0
