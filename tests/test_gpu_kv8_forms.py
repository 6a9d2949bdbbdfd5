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
