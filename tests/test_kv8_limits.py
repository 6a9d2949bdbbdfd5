"""Limits of the 8-bit cache's entries and Python classes that need no GPU: what they refuse, and what they leave behind."""
import pytest

from stratacuda_b200 import _lib as L
from test_kv8_host import A, CALLS, cache, refuse
from stratacuda_b200 import kv8


@pytest.mark.parametrize("top", [0x7fffffff // 64 + 1, 1 << 30, 0x7fffffff])
def test_attend_refuses_longer_lists_than_a_table_has_blocks(top):
    """A list is walked with 32-bit indices some steps past its end."""
    assert refuse(kv8.StrataRangeError, "top", lambda: CALLS["attend"](cache(), picks=A, top=top)) == L.ERR_RANGE


@pytest.mark.parametrize("count,heads", [(1 << 24, 128), (1 << 20, 2048), (1 << 16, 32768), ((1 << 24) - 1, 129)])
def test_attend_refuses_runs_of_more_rows_than_32_bits_count(count, heads):
    """A prompt's rows, tokens times query heads a key/value head, are counted in 32 bits."""
    assert refuse(kv8.StrataRangeError, "2\\^31", lambda: CALLS["attend"](cache(kv_heads=1, dim=1), count=count, heads=heads)) == L.ERR_RANGE


class Backend:
    """Hands out buffers and takes them back; the `fails`-th allocation (or the first write) does not succeed."""
    kind = "cuda"

    def __init__(self, fails=None, writes=True):
        self.fails, self.writes, self.made, self.live = fails, writes, 0, set()

    def alloc(self, length, type="f32", zero=True):
        self.made += 1
        if self.made == self.fails:
            raise kv8.StrataError(L.ERR_ALLOC, "device allocation failed")
        self.live.add(self.made)
        return self.made

    def write(self, buf, data, offset=0):
        if not self.writes:
            raise kv8.StrataError(L.ERR_CUDA, "write failed")

    def free(self, buf):
        self.live.remove(buf)


@pytest.mark.parametrize("fails", [1, 2, 3, 4, 5, 6, None])
def test_a_cache_that_cannot_be_had_leaves_no_buffer_behind(fails):
    backend = Backend(fails, writes=False)
    with pytest.raises(kv8.StrataError):
        kv8.Kv8Cache(backend, kv_heads=2, dim=64, sequences=3, blocks=5)
    assert backend.made == (fails or 6) and not backend.live
    shared = Backend()
    workspace = shared.alloc(8)
    shared.fails = 4
    with pytest.raises(kv8.StrataError):
        kv8.Kv8Cache(shared, kv_heads=2, dim=64, sequences=3, blocks=5, workspace=workspace)
    assert shared.live == {workspace}  # a workspace that others use stays


def test_a_cache_gives_its_buffers_back_once():
    backend = Backend()
    c = kv8.Kv8Cache(backend, kv_heads=2, dim=64, sequences=3, blocks=5)
    assert len(backend.live) == 6
    c.free()
    c.free()
    assert not backend.live


def test_a_cache_asks_for_the_cuda_backend():
    """Its operators have no other: a batch on a host backend is refused when it is made, not at its first step."""
    from oracle.backend import OracleBackend
    from oracle.oracle import Oracle
    from stratacuda_b200.engine import SequenceBatch, StrataEngine
    from stratacuda_b200.model import create_fixture
    host = OracleBackend(Oracle("port"))
    with pytest.raises(ValueError, match="CUDA backend"):
        kv8.Kv8Cache(host, kv_heads=2, dim=64, sequences=3, blocks=5)
    engine = StrataEngine.create(create_fixture(), host)
    for top in (0, 8):
        with pytest.raises(ValueError, match="CUDA backend"):
            SequenceBatch(engine, 2, kv8=True, top=top)
    SequenceBatch(engine, 2).dispose()


@pytest.mark.parametrize("fails", [1, 2, 5, 9])
def test_a_batch_that_cannot_be_had_leaves_no_buffer_behind(fails):
    """The allocation's own error comes through, and the buffers made before it are given back."""
    from oracle.backend import OracleBackend
    from oracle.oracle import Oracle
    from stratacuda_b200.engine import SequenceBatch, StrataEngine
    from stratacuda_b200.model import create_fixture
    host = OracleBackend(Oracle("port"))
    engine = StrataEngine.create(create_fixture(), host)
    live, alloc, free = [], host.alloc, host.free

    def counted(*args, **kw):
        if len(live) + 1 == fails:
            raise MemoryError("no more")
        live.append(alloc(*args, **kw))
        return live[-1]

    host.alloc, host.free = counted, lambda buf: (live.remove(buf), free(buf))
    with pytest.raises(MemoryError, match="no more"):
        SequenceBatch(engine, 2)
    assert not live


@pytest.mark.parametrize("name,bad", [("append", dict(segments=(1 << 32) + 1)), ("append", dict(count=(1 << 32) + 1)), ("select", dict(top=(1 << 32) + 4)),
                                      ("select", dict(first=1 << 32)), ("attend", dict(heads=(1 << 32) + 4)), ("attend", dict(count=-(1 << 32) + 1)),
                                      ("attend", dict(picks=A, top=(1 << 33) + 1)), ("append", dict(row_stride=-1)), ("attend", dict(scale=1e300))])
def test_refuses_integers_past_their_range(name, bad):
    """2^32 + 1 rows are not one row."""
    with pytest.raises(kv8.StrataError) as e:
        CALLS[name](cache(), **bad)
    assert e.value.code in (L.ERR_RANGE, L.ERR_LAYOUT)


def test_a_cache_refuses_integers_past_their_range():
    for bad in (dict(kv_heads=(1 << 32) + 2), dict(dim=(1 << 32) + 64), dict(pages=1 << 32), dict(sequences=(1 << 32) + 1), dict(blocks=-(1 << 32) + 4)):
        with pytest.raises(kv8.StrataError) as e:
            CALLS["append"](cache(**bad))
        assert e.value.code == L.ERR_RANGE


def test_a_cache_on_the_backend_refuses_integers_past_their_range():
    class Library:
        def __getattr__(self, name):
            raise AssertionError("the call went through")

    class Buf:
        handle = 1

    big = (1 << 32) + 1
    backend = Backend()
    with pytest.raises(kv8.StrataRangeError, match="sequences"):
        kv8.Kv8Cache(backend, kv_heads=2, dim=64, sequences=big, blocks=1)
    with pytest.raises(kv8.StrataRangeError, match="pages"):
        kv8.Kv8Cache(backend, kv_heads=2, dim=64, sequences=1 << 20, blocks=1 << 20)
    assert not backend.live
    c = kv8.Kv8Cache(backend, kv_heads=2, dim=64, sequences=3, blocks=5)
    backend.lib = Library()
    b = Buf()
    for name, call in (("segments", lambda: c.append(b, b, b, b, big)), ("count", lambda: c.append(b, b, b, b, 1, big)),
                       ("top", lambda: c.select(b, 4, b, b, b, top=big)), ("last", lambda: c.select(b, 4, b, b, b, last=big)),
                       ("heads", lambda: c.attend(b, big, b, b, b)), ("top", lambda: c.attend(b, 4, b, b, b, picks=b, top=big))):
        with pytest.raises(kv8.StrataRangeError, match=name):
            call()


def test_a_refusals_message_is_its_own_threads():
    """Another thread's refusal by the same cache, between a call's return and its message's reading, changes nothing."""
    import threading
    c = cache()
    entry, inside = c.lib.strata_kv8_call_dev, []

    class Library:
        def strata_kv8_call_dev(self, call):
            rc = entry(call)
            if not inside:
                inside.append(1)
                other = threading.Thread(target=lambda: refuse(kv8.StrataRangeError, "divisible", lambda: CALLS["attend"](c, heads=5)))
                other.start()
                other.join()
            return rc

    c.lib = Library()
    refuse(kv8.StrataRangeError, "segments", lambda: CALLS["append"](c, segments=0))
