"""The forms that the 8-bit cache's operators take by the size of a call, each run at sizes that reach it
(on 148 multiprocessors), against the definitions in tests/kv8_reference.py."""
import math

import numpy as np
import pytest

import kv8_reference as R
from test_gpu_kv8 import BLOCK, WideCache

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- select

def _marked(kv, dim, sequences, blocks, seed, levels=127):
    """A cache whose pages have random marks and scales: all that a selection reads. Every sequence has every page, in an
    order of its own. With few `levels` many blocks' bounds are equal."""
    c = WideCache(kv, dim, sequences, blocks, blocks)
    rng = np.random.default_rng(seed)
    a, b = rng.integers(-levels, levels + 1, (2, blocks, kv, dim))
    lo, hi = np.minimum(a, b), np.maximum(a, b)
    marks = np.zeros((blocks, kv, 2, R.padded(dim)), np.int8)
    marks[:, :, 0, :dim], marks[:, :, 1, :dim] = lo, hi
    scales = np.ones((blocks, kv), np.float32) if levels < 127 else np.exp(rng.normal(0, 0.3, (blocks, kv))).astype(np.float32)
    order = np.stack([rng.permutation(blocks) for _ in range(sequences)])
    c.marks.copy_(c.torch.from_numpy(marks))
    c.scales[:, :, 0] = c.torch.from_numpy(scales).cuda()
    c.table[:] = c.i32(order)
    return c, lo, hi, scales, order, rng


def _check_picks(got, q, lo, hi, scales, order, heads, have, top, first, last):
    """got [kv, top], q [heads, dim] of one token that sees `have` blocks of the sequence with pages `order`."""
    kv = got.shape[0]
    group = heads // kv
    for h in range(kv):
        want = np.full(top, -1)
        if have > 0:
            at = order[:have]
            picked = R.select(q[h * group:(h + 1) * group], (lo[at, h], hi[at, h]), scales[at, h], have, top, first, last)
            want[:len(picked)] = picked
        assert np.array_equal(got[h], want), h


@pytest.mark.parametrize("blocks,heads,kv,dim,segments,top", [(128, 24, 2, 256, 3, 8), (300, 5, 1, 40, 5, 40), (1024, 24, 2, 256, 16, 32),
                                                              (1024, 8, 4, 128, 30, 3), (32768, 2, 1, 64, 3, 100), (32768, 3, 1, 16, 1, 20000),
                                                              (1000, 4, 4, 64, 80, 16), (700, 2, 1, 24, 400, 65)])
@pytest.mark.parametrize("levels", [127, 1])
def test_select_tokens_in_wide_tables(blocks, heads, kv, dim, segments, top, levels):
    """A token's blocks shared by 2, 4 or 8 CTAs, or by the warps of one; lengths around `top` and up to the whole table."""
    first, last = (1, 2) if top >= 3 else (0, 0)
    c, lo, hi, scales, order, rng = _marked(kv, dim, segments, blocks, top, levels)
    have = np.minimum(np.exp(rng.uniform(0, math.log(blocks), segments)).astype(int) + 1, blocks)
    have[0] = blocks
    for i, n in enumerate((top, top + 1, blocks - 1)[:segments - 1]):
        have[i + 1] = min(n, blocks)
    sequence, start = np.arange(segments), have * BLOCK - 1 - rng.integers(0, BLOCK, segments)
    if segments > 4:
        sequence[4] = -1
    q = rng.normal(0, 1, (segments, 1, heads, dim)).astype(np.float32)
    got = c.select(q, heads, sequence, start, top, first, last)
    again = c.select(q, heads, sequence, start, top, first, last)
    assert np.array_equal(got, again)
    for s in range(segments):
        n = 0 if sequence[s] < 0 else start[s] // BLOCK + 1
        _check_picks(got[s, 0], q[s, 0], lo, hi, scales, order[s], heads, n, top, first, last)
    assert c.errors() == 0


@pytest.mark.parametrize("blocks,heads,kv,dim,segments,count", [(400, 24, 2, 256, 1, 1200), (300, 6, 1, 40, 2, 1301), (4000, 5, 1, 128, 1, 900)])
@pytest.mark.parametrize("top,levels", [(8, 127), (40, 127), (100, 127), (8, 1), (40, 1)])
def test_select_prompts_in_tiles(blocks, heads, kv, dim, segments, count, top, levels):
    """Prompts long enough for tiles of 32 tokens (of 11, where a table of 4000 blocks leaves room for no more)."""
    c, lo, hi, scales, order, rng = _marked(kv, dim, segments, blocks, top, levels)
    start = np.array([blocks * BLOCK - count - 1 - 700 * s for s in range(segments)])
    q = rng.normal(0, 1, (segments, count, heads, dim)).astype(np.float32)
    got = c.select(q, heads, np.arange(segments), start, top)
    for s in range(segments):
        for t in np.unique(np.concatenate([np.arange(0, count, 53), [1, 15, 16, 31, 32, count - 2, count - 1]])):
            _check_picks(got[s, t], q[s, t], lo, hi, scales, order[s], heads, (start[s] + t) // BLOCK + 1, top, 1, 2)
    assert c.errors() == 0


def test_select_prompt_from_the_first_token_on():
    """Tiles whose first tokens see nothing or a block or two and whose last see more than `top`."""
    blocks, heads, kv, dim, count, top = 300, 4, 2, 96, 2500, 5
    c, lo, hi, scales, order, rng = _marked(kv, dim, 1, blocks, 3)
    q = rng.normal(0, 1, (1, count, heads, dim)).astype(np.float32)
    for start in (0, -40):
        got = c.select(q, heads, [0], [start], top)
        for t in list(range(0, 450, 7)) + list(range(450, count, 211)):
            _check_picks(got[0, t], q[0, t], lo, hi, scales, order[0], heads, (start + t + 64) // BLOCK, top, 1, 2)
    assert c.errors() == 0


# ---------------------------------------------------------------- attend

@pytest.mark.parametrize("holes", [False, True])
def test_short_form_over_more_pages_than_it_looks_up_at_a_time(holes):
    """16 heads of 64 channels on mma.sync tiles with more than 256 pages of a unit on one CTA, also with gaps among them."""
    heads, kv, dim, blocks, sequences = 16, 1, 64, 600, 160
    c = WideCache(kv, dim, sequences, blocks, blocks)
    rng = np.random.default_rng(3)
    n = blocks * BLOCK - 5
    k, v = rng.normal(0, 1, (2, n, kv, dim)).astype(np.float32)
    c.table[:] = c.i32(rng.permutation(blocks))
    c.append(k[None], v[None], [0], [0])
    q = rng.normal(0, 1, (sequences, 1, heads, dim)).astype(np.float32)
    start = n - 1 - np.arange(sequences)
    picks = None
    if holes:
        picks = np.arange(blocks)[None, None].repeat(sequences, 0)
        picks[rng.random(picks.shape) < 0.3] = -1
    got = c.attend(q, heads, np.arange(sequences), start, picks=picks, top=blocks if holes else 0)
    for s in (0, 1, 80, 159):
        c.check_attend(got[s], q[s], k, v, start[s], 1 / math.sqrt(dim), None if picks is None else picks[s:s + 1])
    assert c.errors() == 0


# ---------------------------------------------------------------- calls from several threads

# One thread a call, each its own `times` times; returns the calls that were refused. (Python's threads overlap too seldom.)
_THREADS = """
#include <atomic>
#include <cstdint>
#include <thread>
#include <vector>
struct Call { const void *cache; const float *q; const int32_t *sequence, *start; int32_t *picks; void *stream; int32_t heads, top; };
using Select = int (*)(const void *, const float *, uint64_t, int32_t, int32_t, int32_t, const int32_t *, const int32_t *, int32_t, int32_t, int32_t,
                       int32_t *, void *, char *, size_t);
extern "C" long hammer(Select select, const Call *calls, int n, long times) {
    std::atomic<long> refused{0};
    std::vector<std::thread> threads;
    for (int i = 0; i < n; ++i)
        threads.emplace_back([&, i] {
            const Call c = calls[i];
            for (long k = 0; k < times; ++k)
                refused += select(c.cache, c.q, 0, c.heads, 1, 1, c.sequence, c.start, c.top, 1, 2, c.picks, c.stream, nullptr, 0) != 0;
        });
    for (auto &t : threads) t.join();
    return refused;
}
"""


def test_select_from_several_threads_over_tables_of_different_widths(tmp_path):
    """A selection's shared memory goes by the table's width; what one thread's call needs must not depend on another's."""
    import ctypes as C
    import shutil
    import subprocess

    from stratacuda_b200 import _lib as L

    if not shutil.which("g++"):
        pytest.skip("no C++ compiler for the calling threads")
    (tmp_path / "hammer.cc").write_text(_THREADS)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-pthread", str(tmp_path / "hammer.cc"), "-o", str(tmp_path / "hammer.so")],
                   check=True)

    class Call(C.Structure):
        _fields_ = [(n, C.c_void_p) for n in ("cache", "q", "sequence", "start", "picks", "stream")] + [("heads", C.c_int32), ("top", C.c_int32)]

    widths, keep, calls = (32768, 40, 32768, 100), [], []
    for blocks in widths:
        c, lo, hi, scales, order, rng = _marked(1, 16, 1, blocks, 1)
        torch = c.torch
        q = rng.normal(0, 1, (2, 16)).astype(np.float32)
        dq, seq, start = torch.from_numpy(q.reshape(1, -1)).cuda(), c.i32([0]), c.i32([blocks * BLOCK - 1])
        picks, stream = torch.full((1, 1, 8), -9, dtype=torch.int32, device="cuda"), torch.cuda.Stream()
        keep.append((c, lo, hi, scales, order, q, dq, seq, start, picks, stream))
        calls.append(Call(C.addressof(c.view._cache), dq.data_ptr(), seq.data_ptr(), start.data_ptr(), picks.data_ptr(), stream.cuda_stream, 2, 8))
    torch.cuda.synchronize()
    hammer = C.CDLL(str(tmp_path / "hammer.so")).hammer
    hammer.restype, hammer.argtypes = C.c_long, [C.c_void_p, C.POINTER(Call), C.c_int, C.c_long]
    refused = hammer(C.cast(L.load().strata_kv8_select_dev, C.c_void_p), (Call * len(calls))(*calls), len(calls), 20000)
    torch.cuda.synchronize()
    assert refused == 0
    for blocks, (c, lo, hi, scales, order, q, dq, seq, start, picks, stream) in zip(widths, keep):
        _check_picks(picks.cpu().numpy()[0], q, lo, hi, scales, order[0], 2, blocks, 8, 1, 2)


# ---------------------------------------------------------------- value scales far apart

@pytest.mark.parametrize("heads,kv,dim,start,count", [(1, 1, 64, 0, 200), (5, 1, 128, 0, 150), (6, 2, 256, 0, 140), (3, 1, 40, 64 * 9 + 30, 300)])
@pytest.mark.parametrize("growth", [12, 20, 33, 60])
def test_prompt_rows_do_not_lose_bits_to_values_they_cannot_see(heads, kv, dim, start, count, growth):
    """Each block's values are 2^growth times those of the block before (from the chunk's on, at most 2^60 in all): every row
    is within the bound that the largest value in its own sight gives."""
    c = WideCache(kv, dim, 1, 20, 20)
    rng = np.random.default_rng(growth)
    n = start + count
    k, v = rng.normal(0, 1, (2, n, kv, dim))
    v *= 2.0 ** np.minimum(growth * np.maximum(np.arange(n) // BLOCK - start // BLOCK, 0), 60)[:, None, None] * 1e-9
    k, v = k.astype(np.float32), v.astype(np.float32)
    c.table[0] = c.i32(rng.permutation(20))
    c.append(k[None], v[None], [0], [0])
    q = rng.normal(0, 1, (1, count, heads, dim)).astype(np.float32)
    got = c.attend(q, heads, [0], [start])
    c.check_attend(got[0], q[0], k, v, start, 1 / math.sqrt(dim))
    assert c.errors() == 0


@pytest.mark.parametrize("count", [1, 70])
@pytest.mark.parametrize("heads,kv,dim,blocks", [(4, 1, 64, 12), (6, 2, 128, 40), (12, 1, 256, 300)])
@pytest.mark.parametrize("small", [9, 16, 24, 40])
def test_results_from_blocks_of_small_values(heads, kv, dim, blocks, small, count):
    """Rows whose weight lies on blocks with values 2^-small of the other blocks', which have weights below 2^-100: the result is
    as exact against the small values as it would be without the others."""
    c = WideCache(kv, dim, 1, blocks, blocks)
    rng = np.random.default_rng(small)
    n = blocks * BLOCK - 3
    heavy = np.arange(n) // BLOCK % 3 == 1  # these have the weight
    direction = rng.normal(0, 1, dim)
    k = rng.normal(0, 0.1, (n, kv, dim)) - 100 * math.sqrt(dim) * np.where(heavy, 0, 1)[:, None, None] * direction / np.sum(direction ** 2)
    v = rng.normal(0, 1, (n, kv, dim)) * np.where(heavy, 2.0 ** -small, 1.0)[:, None, None]
    k, v = k.astype(np.float32), v.astype(np.float32)
    c.table[0] = c.i32(rng.permutation(blocks))
    c.append(k[None], v[None], [0], [0])
    q = (direction + rng.normal(0, 0.01, (1, count, heads, dim))).astype(np.float32)
    start = n - count
    got = c.attend(q, heads, [0], [start])
    heavy_blocks = np.arange(1, blocks, 3)
    picks = np.broadcast_to(heavy_blocks, (count, kv, len(heavy_blocks)))
    c.check_attend(got[0], q[0], k, v, start, 1 / math.sqrt(dim), picks)  # (the others' share is below 2^-100)
    assert c.errors() == 0


@pytest.mark.parametrize("heads,kv,dim,blocks,sequences", [(4, 1, 64, 300, 16), (12, 1, 256, 200, 24), (8, 2, 128, 300, 9), (4, 1, 64, 20, 2)])
@pytest.mark.parametrize("sizes", [(0.0, 2.0 ** -60), (2.0 ** -90, 2.0 ** 60), (0.0, 2.0 ** -90, 2.0 ** 20), (2.0 ** -60, 2.0 ** -20, 2.0 ** 20, 2.0 ** 60, 0.0)])
def test_tokens_over_blocks_of_zeros_and_of_very_different_values(heads, kv, dim, blocks, sequences, sizes):
    """Token steps over long lists (and a short one) whose blocks' values are of the given sizes, in no order."""
    c = WideCache(kv, dim, sequences, blocks, blocks)
    rng = np.random.default_rng(len(sizes))
    n = blocks * BLOCK - 7
    k, v = rng.normal(0, 1, (2, n, kv, dim))
    v *= rng.choice(sizes, blocks).repeat(BLOCK)[:n, None, None]
    k, v = k.astype(np.float32), v.astype(np.float32)
    c.table[:] = c.i32(rng.permutation(blocks))
    c.append(k[None], v[None], [0], [0])
    q = rng.normal(0, 1, (sequences, 1, heads, dim)).astype(np.float32)
    start = n - 1 - 50 * np.arange(sequences)
    got = c.attend(q, heads, np.arange(sequences), start)
    for s in (0, 1, sequences - 1):
        c.check_attend(got[s], q[s], k, v, start[s], 1 / math.sqrt(dim))
    assert c.errors() == 0


def test_value_scales_too_far_apart_are_reported():
    """A list whose later values are 2^150 times those of its first pages has no result in F32's exponents, and says so."""
    heads, kv, dim, blocks, sequences = 4, 1, 64, 300, 40
    c = WideCache(kv, dim, sequences, blocks, blocks)
    rng = np.random.default_rng(1)
    n = blocks * BLOCK
    k, v = rng.normal(0, 1, (2, n, kv, dim))
    v *= np.where(np.arange(n) < n // 2, 2.0 ** -90, 2.0 ** 60)[:, None, None]
    c.table[:] = c.i32(np.arange(blocks))
    c.append(k[None].astype(np.float32), v[None].astype(np.float32), [0], [0])
    q = rng.normal(0, 1, (sequences, 1, heads, dim)).astype(np.float32)
    c.attend(q, heads, np.arange(sequences), np.full(sequences, n // 2 - 1))  # small ones alone
    assert c.errors() == 0
    c.attend(q, heads, np.arange(sequences), np.full(sequences, n - 1))
    assert c.errors() == 32


# ---------------------------------------------------------------- token steps on tcgen05, by heads and channels

def _strided_attend(c, q, heads, sequence, start, picks=None, top=0, off=1):
    """c.attend with queries in rows three floats longer than they need be, `off` floats past a 16-byte boundary."""
    s, n = q.shape[:2]
    w = heads * c.dim
    wide = c.torch.zeros(s * n * (w + 3) + off, device="cuda")
    rows = wide[off:].reshape(s * n, w + 3)
    rows[:, :w] = c.torch.from_numpy(q.reshape(s * n, w)).cuda()
    y = c.torch.full((s * n * w + 1,), float("nan"), device="cuda")[1:]
    c.view.attend(rows, heads, y, c.i32(sequence), c.i32(start), s, n, None if picks is None else c.i32(picks), top, row_stride=w + 3)
    return y.cpu().numpy().reshape(s, n, heads, c.dim)


@pytest.mark.parametrize("heads,dim,blocks", [(3, 64, 45), (8, 40, 85), (11, 64, 310), (3, 128, 45), (7, 72, 60), (12, 128, 140), (16, 100, 600),
                                              (4, 256, 40), (8, 256, 60), (10, 200, 90), (15, 256, 160)])
def test_tokens_of_long_sessions_by_heads_and_channels(heads, dim, blocks):
    """Pages of 40 sessions shared over the CTAs, for every width of the operands that a call of this kind takes: queries off the
    16-byte grid, one that is not finite, blocks of zeros, garbage past each token's position and in the table past its block."""
    kv, sequences = 1, 40
    c = WideCache(kv, dim, sequences, blocks + 3, blocks)
    rng = np.random.default_rng(dim + heads)
    n = blocks * BLOCK - 21
    k, v = rng.normal(0, 1, (2, n, kv, dim)).astype(np.float32)
    for b in (1, 6, 7, blocks // 2):
        k[b * BLOCK:(b + 1) * BLOCK] = 0
        v[(b + 1) * BLOCK:(b + 2) * BLOCK] = 0
    c.table[:, :blocks] = c.i32(rng.permutation(blocks))
    c.table[:, blocks:] = c.i32([-1, 1 << 30, -7])
    c.append(k[None], v[None], [0], [0])
    last = int(c.table[0, blocks - 1])
    c.codes[last, :, 0].reshape(kv, -1, BLOCK, 64)[:, :, n % BLOCK:] = -128
    c.codes[last, :, 1].reshape(kv, -1, BLOCK)[:, :, n % BLOCK:] = 127
    q = rng.normal(0, 1, (sequences, 1, heads, dim)).astype(np.float32)
    start = n - 1 - 70 * np.arange(sequences) % (n // 2)
    sequence = np.arange(sequences)
    sequence[3], start[4] = -1, -1
    want = _strided_attend(c, q, heads, sequence, start)
    assert c.errors() == 0 and not want[3].any() and not want[4].any()
    for s in (0, 1, 5, sequences - 1):
        c.check_attend(want[s], q[s], k, v, start[s], 1 / math.sqrt(dim))
    for bad in (np.nan, -np.inf):
        p = q.copy()
        p[5, 0, heads - 1, dim // 2] = bad
        got = _strided_attend(c, p, heads, sequence, start, off=4)
        assert np.isnan(got[5, 0, heads - 1]).all()
        got[5, 0, heads - 1] = want[5, 0, heads - 1]
        assert np.array_equal(got.view(np.uint32), want.view(np.uint32))
    # a block whose page is none is left out and reported; others' tokens stay as they are
    c.table[7, 2] = blocks
    got = _strided_attend(c, q, heads, sequence, start)
    assert c.errors() == 1
    listed = np.setdiff1d(np.arange(blocks), [2])[None, None]
    c.check_attend(got[7], q[7], k, v, start[7], 1 / math.sqrt(dim), listed)
    assert np.array_equal(got[:7].view(np.uint32), want[:7].view(np.uint32))


@pytest.mark.parametrize("heads,dim", [(3, 64), (8, 40), (11, 64), (16, 64), (3, 128), (7, 72), (12, 128), (16, 100), (4, 256), (8, 256), (12, 256),
                                       (15, 200)])
@pytest.mark.parametrize("picked", [True, False])
def test_more_tokens_than_share_pages_by_heads_and_channels(heads, dim, picked):
    """1200 tokens, each of whose units one CTA has whole: lists of picks with gaps, or all blocks of sessions of all lengths."""
    kv, blocks, top, tokens = 1, 30, 7, 1200
    c = WideCache(kv, dim, tokens, blocks, blocks)
    rng = np.random.default_rng(dim + heads)
    n = blocks * BLOCK
    k, v = rng.normal(0, 1, (2, n, kv, dim)).astype(np.float32)
    c.table[:] = c.i32(rng.permutation(blocks))
    c.append(k[None], v[None], [0], [0])
    q = rng.normal(0, 1, (tokens, 1, heads, dim)).astype(np.float32)
    start, sequence, picks = rng.integers(0, n, tokens), np.arange(tokens), None
    sequence[11], start[12], start[13] = -1, -1, 0
    if picked:
        picks = np.full((tokens, kv, top), -1)
        for t in range(tokens):
            some = np.sort(rng.permutation(max(start[t] // BLOCK + 1, 1))[:top])
            picks[t, 0, rng.permutation(top)[:len(some)]] = some
        picks[14] = -1
    q[15, 0, 0, 0] = np.nan
    got = _strided_attend(c, q, heads, sequence, start, picks, top if picked else 0)
    assert c.errors() == 0
    assert not got[11].any() and not got[12].any() and np.isnan(got[15, 0, 0]).all() and not np.isnan(np.delete(got, 15, 0)).any()
    for t in list(range(0, tokens, 61)) + [13, 14, tokens - 1]:
        c.check_attend(got[t], q[t], k, v, start[t], 1 / math.sqrt(dim), None if picks is None else picks[t][None])
