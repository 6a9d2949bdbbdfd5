"""Sessions with the token mixers over runs (``mixers=1``) on a B200: what they write, batches with 8-bit caches by value, and long
chunks with the fast mixture of experts by value.

The fast mixture takes chunks of more than 64 tokens with FP16 operands, 2e-3 of a layer's output. Behind n such layers a row is off by
2e-3 sqrt(n), were each layer's output as large as what it is added to. Where a router has a near tie another expert of ten may come in,
which changes a part of such a row; a row of another token or another sequence is sqrt(2) off. So half of all rows keep the first bound,
nearly all four times that, and all of them 1/2."""
import numpy as np
import pytest

from engine_conformance import TOL
from oracle.engine_ref import compare

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def b():
    from stratacuda_b200.backend import CudaBackend
    be = CudaBackend(0)
    yield be
    be.dispose()


@pytest.fixture(scope="module")
def store(b):
    """Eight layers of the 48-layer model, two of them attention."""
    from stratacuda_b200.synthetic import MODEL_GEOMETRY, DeviceStore
    s = DeviceStore(b, dict(MODEL_GEOMETRY, layers=8), seed=1)
    yield s
    s.free()


def test_an_eager_step_and_a_chunk_write_the_position_once(b, store, monkeypatch):
    """Not once a layer; and always the one at which they stand, whatever wrote the scalar before."""
    from stratacuda_b200.engine import StrataEngine
    engine, again = (StrataEngine.create(store, b, mixers=1) for _ in range(2))
    written, write = [], b.write

    def watched(buf, data, *rest):
        if engine._dev is not None and buf is engine._dev["position"]:
            written.append(int(np.asarray(data)[0]))
        return write(buf, data, *rest)

    monkeypatch.setattr(b, "write", watched)
    engine.step(2, predict=False)  # (the scalar is made during this one)
    written.clear()
    engine.step(7)
    engine.prefill([4, 8, 7, 4, 1], chunk_size=2)
    engine.step(3)
    assert written == [1, 2, 4, 6, 7]
    engine.reset()
    write(engine._dev["position"], np.array([5], np.int32))
    engine.step(2, predict=False)
    got = engine.step(7, logits=True)
    again.step(2, predict=False)
    assert np.array_equal(got["logits"], again.step(7, logits=True)["logits"])
    engine.dispose()
    again.dispose()


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("chunk", [1024, 200, 65])
def test_long_chunks_with_the_fast_mixture(b, store, chunk, graph):
    """Keys, values and the rule's states of every layer against the exact entries' and the exact mixture's 64-token chunks."""
    from stratacuda_b200.engine import StrataEngine
    prompt = [int(t) for t in np.random.default_rng(3).integers(0, store.config["vocab"], 601)]
    exact, runs = StrataEngine.create(store, b), StrataEngine.create(store, b, 1, graph=graph, mixers=1)
    want, got = exact.prefill(prompt, chunk_size=64, logits=True), runs.prefill(prompt, chunk_size=chunk, logits=True)

    def off(kind, layer, width, rows):
        x, y = (b.read(e.states[layer][kind]).reshape(-1, width)[:rows].astype(np.float64) for e in (exact, runs))
        return np.linalg.norm(x - y, axis=1) / np.linalg.norm(x, axis=1)

    g = exact.g
    for layer in range(g["layers"]):
        one = 2e-3 * np.sqrt(layer + 1)
        if exact.is_attention(layer):
            for kind in ("keys", "values"):
                rows = off(kind, layer, g["kvHeads"] * g["headDim"], len(prompt))
                assert np.median(rows) <= one and np.quantile(rows, 0.9) <= 4 * one and rows.max() <= 0.5
        else:
            rows = off("state", layer, g["ssmDim"], g["ssmDim"] * g["valueHeads"])  # a key's values in a head
            assert np.median(rows) <= one and np.quantile(rows, 0.9) <= 4 * one and rows.max() <= 0.5
    assert np.linalg.norm(want["logits"] - got["logits"]) <= 0.5 * np.linalg.norm(want["logits"])
    exact.dispose()
    runs.dispose()


@pytest.mark.parametrize("top", [0, 3])
def test_a_batch_with_8_bit_caches_by_value(b, top):
    """The same sessions in a batch of the exact entries and in one of the run forms, both with 8-bit caches: the caches round the same
    values, so that the fixture model's bar holds. Slots are filled out of order, and one anew between steps."""
    from stratacuda_b200.engine import SequenceBatch, StrataEngine
    from stratacuda_b200.model import create_fixture
    fixture = create_fixture()
    exact, runs, session = StrataEngine.create(fixture, b), StrataEngine.create(fixture, b, mixers=1), StrataEngine.create(fixture, b)
    batches = [SequenceBatch(e, 3, kv8=True, top=top) for e in (exact, runs)]
    tokens = [0] * 3

    def admit(slot, prompt):
        session.reset()
        tokens[slot] = session.prefill(prompt)["token"]
        for batch in batches:
            batch.admit(slot, session)

    for slot, prompt in ((2, [2, 7, 4]), (0, [5]), (1, [9, 1, 3, 3, 8])):
        admit(slot, prompt)
    for step in range(6):
        if step == 3:
            admit(0, [6, 6, 2, 1, 30, 12, 7])
        want, got = (batch.step(list(tokens), logits=True) for batch in batches)
        for slot in range(3):
            compare(got["logits"][slot], want["logits"][slot], TOL)
            assert got["tokens"][slot] == want["tokens"][slot]
        tokens = [int(t) for t in want["tokens"]]
    for x in (*batches, session, exact, runs):
        x.dispose()
