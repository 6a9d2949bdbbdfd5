"""Sessions that come and go in a batch with 8-bit caches, and that attend to some of their blocks, on the B200."""
import math

import numpy as np
import pytest

import kv8_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def world():
    """Three prefilled sessions of a small synthetic model: (backend, engines, their next tokens)."""
    from stratacuda_b200.backend import CudaBackend
    from stratacuda_b200.engine import StrataEngine
    from stratacuda_b200.synthetic import MODEL_GEOMETRY, DeviceStore
    b = CudaBackend(0)
    store = DeviceStore(b, MODEL_GEOMETRY, seed=9)
    rng, engines, first = np.random.default_rng(2), [], []
    for n in (700, 333, 90):
        e = StrataEngine.create(store, b, 1)
        first.append(e.prefill(rng.integers(0, MODEL_GEOMETRY["vocab"], n).tolist(), chunk_size=64)["token"])
        engines.append(e)
    yield b, engines, first
    for e in engines:
        e.dispose()
    store.free()
    b.dispose()


def test_sessions_attend_to_the_blocks_that_are_picked(world):
    """Sessions with more blocks than are picked: the first attention layer's picks are those of the definition over its cache's
    marks, and its output is attention over them."""
    from stratacuda_b200.engine import SequenceBatch
    b, engines, first = world
    top = 4
    batch = SequenceBatch(engines[0], 3, kv8=True, top=top)
    for s, e in enumerate(engines):
        batch.admit(s, e)
    g = engines[0].g
    layer = next(i for i in range(g["layers"]) if engines[0].is_attention(i))
    cache, seen = batch.states[layer]["cache"], {}
    attend = cache.attend

    def watched(q, heads, y, sequence, start, segments, count, picks, *rest):
        attend(q, heads, y, sequence, start, segments, count, picks, *rest)
        seen.update(q=b.read(q).copy(), y=b.read(y).copy(), picks=b.read(picks, "i32").copy())

    cache.attend = watched
    tokens = first
    for _ in range(3):
        tokens = batch.step(tokens)["tokens"]
    kv, hd, heads, p = g["kvHeads"], g["headDim"], g["heads"], R.padded(g["headDim"])
    codes = b.read(cache.codes).view(np.int8).reshape(cache.pages, kv, 2, p * 64)
    marks = b.read(cache.marks).view(np.int8).reshape(cache.pages, kv, 2, p)
    scales, table = b.read(cache.scales).reshape(cache.pages, kv, 2), b.read(cache.table, "i32").reshape(3, -1)
    q, y, picks = seen["q"].reshape(3, heads, hd), seen["y"].reshape(3, heads, hd), seen["picks"].reshape(3, kv, top)
    group, scale = heads // kv, float(np.float32(1 / math.sqrt(hd)))
    for s in range(3):
        n = batch.positions[s]
        have = (n + 63) // 64
        pages = table[s, :have]
        for h in range(kv):
            want = R.select(q[s, h * group:(h + 1) * group], (marks[pages, h, 0, :hd], marks[pages, h, 1, :hd]), scales[pages, h, 0], have, top, 1, 2)
            assert np.array_equal(picks[s, h, :len(want)], want) and (picks[s, h, len(want):] == -1).all()
            assert s == 2 or len(want) < have  # something is left out
            k = codes[pages, h, 0].reshape(have, p // 64, 64, 64).transpose(0, 2, 1, 3).reshape(have, 64, p)[..., :hd] * scales[pages, h, 0].astype(float)[:, None, None]
            v = codes[pages, h, 1].reshape(have, p, 64).transpose(0, 2, 1)[..., :hd] * scales[pages, h, 1].astype(float)[:, None, None]
            at = (want[:, None] * 64 + np.arange(64)).ravel()
            at = at[at < n]
            for i in range(h * group, (h + 1) * group):
                yd, bound = R.attend(q[s, i][None], k.reshape(-1, hd)[at], v.reshape(-1, hd)[at], scale, np.ones((1, len(at)), bool))
                assert np.abs(y[s, i] - yd[0]).max() <= bound[0], (s, i)
    batch.dispose()


@pytest.mark.parametrize("graph,top", [(False, 0), (True, 3)])
def test_a_slot_that_was_used_holds_nothing_of_its_last_session(world, graph, top):
    """Sessions admitted into slots where longer and shorter ones have been go on as in a new batch, bit for bit."""
    from stratacuda_b200.engine import SequenceBatch
    b, engines, first = world

    def run(batch, slots, steps):
        for s, e in enumerate(slots):
            batch.admit(s, engines[e])
        tokens, logits = [first[e] for e in slots], []
        for _ in range(steps):
            r = batch.step(tokens, logits=True)
            tokens = r["tokens"]
            logits.append(r["logits"].copy())
        return np.array(logits)

    used, new = (SequenceBatch(engines[0], 2, graph=graph, kv8=True, top=top) for _ in range(2))
    run(used, (0, 2), 40)
    got = run(used, (1, 0), 5)
    assert np.array_equal(got, run(new, (1, 0), 5))
    used.dispose()
    new.dispose()
