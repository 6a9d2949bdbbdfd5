"""Decode of many sessions whose attention caches are held in 8 bits (SequenceBatch with kv8) on the B200.

The layers before a model's first attention layer do not see the cache, so that layer's keys, values and queries are
those of the F32 batch bit for bit; its 8-bit cache has to hold exactly their rounding, and its output has to be
attention over that, within the rounding bound that tests/kv8_reference.py derives."""
import math

import numpy as np
import pytest

import kv8_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def b():
    from stratacuda_b200.backend import CudaBackend
    be = CudaBackend(0)
    yield be
    be.dispose()


def _first(engine):
    return next(i for i in range(engine.g["layers"]) if engine.is_attention(i))


def test_first_attention_layer_is_the_f32_batchs_rounded(b):
    from stratacuda_b200.engine import SequenceBatch, StrataEngine
    from stratacuda_b200.synthetic import MODEL_GEOMETRY, DeviceStore
    store = DeviceStore(b, MODEL_GEOMETRY, seed=4)
    try:
        rng = np.random.default_rng(5)
        prompts = [rng.integers(0, MODEL_GEOMETRY["vocab"], n).tolist() for n in (1, 70, 130)]
        engines, tokens = [], []
        for p in prompts:
            e = StrataEngine.create(store, b, 1)
            tokens.append(e.prefill(p, chunk_size=64)["token"])
            engines.append(e)
        plain, small = SequenceBatch(engines[0], 3), SequenceBatch(engines[0], 3, kv8=True)
        for s, e in enumerate(engines):
            plain.admit(s, e)
            small.admit(s, e)
        layer, g = _first(engines[0]), engines[0].g
        cache, seen = small.states[layer]["cache"], []
        attend = cache.attend

        def watched(q, heads, y, *rest):
            attend(q, heads, y, *rest)
            seen.append((b.read(q).copy(), b.read(y).copy()))

        cache.attend = watched
        for step in range(3):
            plain.step(tokens)
            small.step(tokens)  # the same inputs, whatever either would go on with
            tokens = [(t * 7 + step) % g["vocab"] for t in tokens]
        kv, hd, heads, width = g["kvHeads"], g["headDim"], g["heads"], g["kvHeads"] * g["headDim"]
        keys = b.read(plain.states[layer]["keys"]).reshape(3, g["context"], kv, hd)
        values = b.read(plain.states[layer]["values"]).reshape(3, g["context"], kv, hd)
        for s in range(3):
            n = small.positions[s]
            assert n == len(prompts[s]) + 3
            q, y = (x.reshape(3, heads, hd)[s] for x in seen[-1])
            for h in range(kv):
                k, v = R.dequantised(R.blocks_of(keys[s, :n, h], values[s, :n, h]))
                for i in range(heads // kv):
                    at = h * (heads // kv) + i
                    want, bound = R.attend(q[at][None], k, v, np.float64(np.float32(1 / math.sqrt(hd))), np.ones((1, n), bool))
                    assert np.abs(y[at] - want[0]).max() <= bound[0], (s, h, i)
        with pytest.raises(ValueError, match="cannot be exported"):
            small.export(0, engines[0])
        plain.dispose()
        small.dispose()
        for e in engines:
            e.dispose()
    finally:
        store.free()


def test_picking_every_block_and_graph_replay_change_nothing(b):
    """Sessions of 4 blocks: attention over 4 picked blocks is attention over all, bit for bit, and a replayed step is a step."""
    from stratacuda_b200.engine import SequenceBatch, StrataEngine
    from stratacuda_b200.synthetic import MODEL_GEOMETRY, DeviceStore
    store = DeviceStore(b, MODEL_GEOMETRY, seed=6)
    try:
        rng = np.random.default_rng(7)
        prompts = [rng.integers(0, MODEL_GEOMETRY["vocab"], n).tolist() for n in (200, 220)]
        engines = [StrataEngine.create(store, b, 1) for _ in prompts]
        first = [e.prefill(p, chunk_size=64)["token"] for e, p in zip(engines, prompts)]
        runs = []
        for graph, top in ((False, 0), (True, 0), (True, 4)):
            batch, tokens, got = SequenceBatch(engines[0], 2, graph=graph, kv8=True, top=top), first, []
            for s, e in enumerate(engines):
                batch.admit(s, e)
            for _ in range(4):
                r = batch.step(tokens, logits=True)
                tokens = r["tokens"]
                got.append(r["logits"].copy())
            batch.dispose()
            runs.append(np.array(got))
        assert np.array_equal(runs[0], runs[1])
        assert np.array_equal(runs[0], runs[2])
        for e in engines:
            e.dispose()
    finally:
        store.free()
