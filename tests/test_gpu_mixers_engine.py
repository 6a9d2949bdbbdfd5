"""The engine and the batch with the token mixers over runs (``mixers=1``) on a B200.

Their inner parts agree with the reference's entries to F32 rounding, so the fixture model keeps the reference's bar against its F64
engine: 8e-5 relative on the logits, the same tokens and routed experts. In the 48-layer model a layer's output may be 2^-20 of
itself off (the rule's bound); 48 of them, were they all of one sign, 5e-5 of the logits; a near tie of the router may add an
expert's difference: the bound is 1e-3. The fast mixture of experts takes chunks of more than 64 tokens with FP16 operands, 2e-3 a layer
and other last bits from run to run, which 48 layers and their routers magnify: such chunks are compared with the exact mixture."""
import numpy as np
import pytest

from engine_conformance import TOL
from oracle.engine_ref import ReferenceEngine, compare

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def b():
    from stratacuda_b200.backend import CudaBackend
    be = CudaBackend(0)
    yield be
    be.dispose()


def test_fixture_model_keeps_the_reference_bar(b):
    from stratacuda_b200.engine import StrataEngine
    from stratacuda_b200.model import create_fixture
    store = create_fixture()
    engine = StrataEngine.create(store, b, mixers=1)
    ref = ReferenceEngine(store)
    for token in [2, 7, 4, 7, 4]:
        want, got = ref.step(token), engine.step(token, logits=True)
        compare(got["logits"], want["logits"], TOL)
        assert got["token"] == want["token"]
        assert [r["ids"] for r in engine.stats["routes"]] == want["routes"]
    snap = engine.checkpoint()
    first = engine.step(8, logits=True)
    engine.restore(snap)
    assert np.array_equal(first["logits"], engine.step(8, logits=True)["logits"])
    for chunk in [1, 2, 5, 100]:
        engine.reset()
        ref = ReferenceEngine(store)
        engine.step(2, predict=False)
        ref.step(2)
        for t in [7, 4, 8, 7, 4]:
            want = ref.step(t)
        got = engine.prefill([7, 4, 8, 7, 4], chunk_size=chunk, logits=True)
        compare(got["logits"], want["logits"], TOL)
        assert got["token"] == want["token"]
        compare(engine.step(8, logits=True)["logits"], ref.step(8)["logits"], TOL)
    engine.dispose()
    engine.dispose()


@pytest.mark.parametrize("kv8", [False, True])
def test_fixture_batch_of_sequences(b, kv8):
    """Three sequences of a batch against an engine each, over steps; one goes back into its engine and goes on there."""
    from stratacuda_b200.engine import SequenceBatch, StrataEngine
    from stratacuda_b200.model import create_fixture
    store = create_fixture()
    prompts = [[2, 7, 4], [5], [9, 1, 3, 3, 8]]
    engines = [StrataEngine.create(store, b, mixers=1) for _ in prompts]
    nxt = [e.prefill(p)["token"] for e, p in zip(engines, prompts)]
    batch = SequenceBatch(engines[0], 3, kv8=kv8)
    for slot, e in enumerate(engines):
        batch.admit(slot, e)
    tokens = list(nxt)
    for _ in range(4):
        got = batch.step(tokens, logits=True)
        for s, e in enumerate(engines):
            want = e.step(tokens[s], logits=True)
            if not kv8:  # (an 8-bit cache rounds what it holds)
                compare(got["logits"][s], want["logits"], TOL)
                assert got["tokens"][s] == want["token"]
            else:
                assert np.isfinite(got["logits"]).all()
        tokens = [int(t) for t in got["tokens"]]
    if not kv8:
        more = StrataEngine.create(store, b, mixers=1)
        batch.export(1, more)
        compare(more.step(tokens[1], logits=True)["logits"], engines[1].step(tokens[1], logits=True)["logits"], TOL)
        more.dispose()
    batch.dispose()
    for e in engines:
        e.dispose()


def test_refusals(b):
    from oracle.backend import OracleBackend
    from oracle.oracle import Oracle
    from stratacuda_b200.engine import StrataEngine
    from stratacuda_b200.model import create_fixture
    store = create_fixture()
    with pytest.raises(ValueError, match="CUDA backend"):
        StrataEngine(store, OracleBackend(Oracle("port")), mixers=1)
    with pytest.raises(ValueError, match="mixers"):
        StrataEngine(store, b, mixers=2)
    exact, runs = StrataEngine.create(store, b), StrataEngine.create(store, b, mixers=1)
    with pytest.raises(ValueError, match="chunk size"):
        exact.prefill([1, 2], chunk_size=65)
    with pytest.raises(ValueError, match="chunk size"):
        runs.prefill([1, 2], chunk_size=1025)
    exact.dispose()
    runs.dispose()


@pytest.mark.parametrize("moe_mode,whole,part", [(0, 1024, 200), (1, 64, 50)])
def test_48_layer_model(b, moe_mode, whole, part):
    """A prompt through the run forms, in one chunk and in several, captured chunks and steps among them, against the exact
    entries' 64-token chunks; then a batch of sessions."""
    from stratacuda_b200.engine import SequenceBatch, StrataEngine
    from stratacuda_b200.synthetic import MODEL_GEOMETRY, DeviceStore
    store = DeviceStore(b, dict(MODEL_GEOMETRY), seed=1)
    worst = [0.0]

    def near(got, ref):
        worst[0] = max(worst[0], float(np.linalg.norm(got - ref) / np.linalg.norm(ref)))
        assert worst[0] <= 1e-3, worst[0]

    try:
        prompt = [int(t) for t in np.random.default_rng(1).integers(0, store.config["vocab"], 601)]
        exact = StrataEngine.create(store, b, moe_mode)
        want = exact.prefill(prompt, chunk_size=64, logits=True)
        runs = StrataEngine.create(store, b, moe_mode, graph=True, mixers=1)
        near(runs.prefill(prompt, chunk_size=whole, logits=True)["logits"], want["logits"])
        token = want["token"]
        for _ in range(3):  # eager, captured, replayed
            w, r = exact.step(token, logits=True), runs.step(token, logits=True)
            near(r["logits"], w["logits"])
            assert r["token"] == w["token"]
            token = w["token"]
        again = StrataEngine.create(store, b, moe_mode, graph=True, mixers=1)
        near(again.prefill(prompt, chunk_size=part, logits=True)["logits"], want["logits"])  # eager and captured, replayed, the rest
        batch = SequenceBatch(runs, 2, graph=True)
        batch.admit(0, runs)
        batch.admit(1, again)
        t = [token, want["token"]]
        for _ in range(3):
            got = batch.step(t, logits=True)
            a, c = runs.step(t[0], logits=True), again.step(t[1], logits=True)
            near(got["logits"][0], a["logits"])
            near(got["logits"][1], c["logits"])
            t = [a["token"], c["token"]]
        again.reset()
        got = again.prefill(prompt, chunk_size=1024, logits=True)
        assert got["position"] == len(prompt) - 1 and np.isfinite(got["logits"]).all()
        print(f"largest relative difference of the logits {worst[0]:.3g}")
        batch.dispose()
        for e in (exact, runs, again):
            e.dispose()
    finally:
        store.free()
