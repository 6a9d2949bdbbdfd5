"""Sessions with the token mixers over runs (``mixers=1``) on a B200: what they write."""
import numpy as np
import pytest

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
