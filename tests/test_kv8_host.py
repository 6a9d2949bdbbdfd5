"""Refusals of the 8-bit cache's pointer entries and host-side sizes: no GPU is touched."""
import ctypes as C

import numpy as np
import pytest

import kv8_reference as R
from stratacuda_b200 import _lib as L
from stratacuda_b200 import kv8

A = 0x1000  # an aligned address that is never followed


def cache(**kw):
    parts = dict(kv_heads=2, dim=64, pages=8, sequences=2, blocks=4, codes=A, marks=A, scales=A, open=A, table=A, workspace=A)
    parts.update(kw)
    return kv8.DeviceCache(**parts)


def refuse(kind, text, call):
    with pytest.raises(kind, match=text) as e:
        call()
    return e.value.code


CALLS = {
    "append": lambda c, **kw: c.append(**{**dict(k=A, v=A, sequence=A, start=A), **kw}),
    "select": lambda c, **kw: c.select(**{**dict(q=A, heads=4, picks=A, sequence=A, start=A, top=4), **kw}),
    "attend": lambda c, **kw: c.attend(**{**dict(q=A, heads=4, y=A, sequence=A, start=A), **kw}),
}


@pytest.mark.parametrize("name", sorted(CALLS))
@pytest.mark.parametrize("bad,text", [(dict(kv_heads=0), "kv_heads"), (dict(dim=0), "dim"), (dict(dim=257), "dim"), (dict(pages=0), "pages"),
                                      (dict(sequences=0), "sequences"), (dict(blocks=0), "blocks"), (dict(blocks=1 << 26), "blocks"),
                                      (dict(codes=None), "null"), (dict(table=None), "null"), (dict(workspace=None), "null")])
def test_refuses_a_cache_that_is_none(name, bad, text):
    assert refuse(kv8.StrataRangeError, text, lambda: CALLS[name](cache(**bad))) == L.ERR_RANGE


@pytest.mark.parametrize("name", sorted(CALLS))
@pytest.mark.parametrize("bad,text", [(dict(segments=0), "segments"), (dict(segments=70000), "segments"), (dict(count=0), "count"),
                                      (dict(segments=60000, count=60000), "2\\^24"), (dict(sequence=None), "null"), (dict(start=None), "null")])
def test_refuses_runs(name, bad, text):
    assert refuse(kv8.StrataRangeError, text, lambda: CALLS[name](cache(), **bad)) == L.ERR_RANGE


@pytest.mark.parametrize("name,bad,text", [("append", dict(row_stride=127), "row_stride"), ("append", dict(row_stride=1 << 50), "row_stride"),
                                           ("attend", dict(row_stride=255), "row_stride"), ("select", dict(row_stride=255), "row_stride"),
                                           ("append", dict(k=A + 2), "4-byte"), ("attend", dict(q=A + 1), "4-byte"),
                                           ("attend", dict(y=A + 3), "4-byte"), ("select", dict(picks=A + 2), "4-byte"),
                                           ("attend", dict(start=A + 2), "4-byte")])
def test_refuses_layouts(name, bad, text):
    assert refuse(kv8.StrataError, text, lambda: CALLS[name](cache(), **bad)) == L.ERR_LAYOUT


@pytest.mark.parametrize("part", ["codes", "marks", "workspace"])
def test_refuses_unaligned_parts(part):
    assert refuse(kv8.StrataError, "16-byte", lambda: CALLS["attend"](cache(**{part: A + 8}))) == L.ERR_LAYOUT


@pytest.mark.parametrize("name,bad,text", [("attend", dict(heads=0), "heads"), ("attend", dict(heads=5), "divisible"),
                                           ("select", dict(heads=3), "divisible"), ("select", dict(top=0), "top"),
                                           ("select", dict(top=40000), "top"), ("select", dict(first=3, last=2), "first"),
                                           ("select", dict(first=-1), "first"), ("attend", dict(picks=A, top=0), "top"),
                                           ("attend", dict(scale=float("nan")), "scale"), ("attend", dict(y=None), "null"),
                                           ("attend", dict(q=None), "null"), ("select", dict(picks=None), "null"),
                                           ("append", dict(k=None), "null"), ("append", dict(v=None), "null")])
def test_refuses_arguments(name, bad, text):
    assert refuse(kv8.StrataRangeError, text, lambda: CALLS[name](cache(), **bad)) == L.ERR_RANGE


def test_refuses_a_table_too_long_to_select_from():
    assert refuse(kv8.StrataRangeError, "32768", lambda: CALLS["select"](cache(blocks=32769))) == L.ERR_RANGE


def test_null_cache_and_context():
    lib = L.load()
    msg = C.create_string_buffer(64)
    assert lib.strata_kv8_append_dev(None, A, A, 0, 1, 1, A, A, None, msg, 64) == L.ERR_RANGE and b"null cache" in msg.value
    assert lib.strata_kv8_attend_dev(None, A, 0, 1, 1, 1, A, A, None, 0, 1.0, A, None, None, 0) == L.ERR_RANGE
    assert lib.strata_kv8_append(None, None, 0, 0, 0, 1, 1, 0, 0) == L.ERR_RANGE
    assert lib.strata_kv8_select(None, None, 0, 0, 1, 1, 1, 0, 0, 1, 0, 0, 0) == L.ERR_RANGE
    assert lib.strata_kv8_attend(None, None, 0, 0, 1, 1, 1, 0, 0, 0, 0, 1.0, 0) == L.ERR_RANGE


def test_sizes_and_structures():
    assert [kv8.padded(d) for d in (1, 64, 65, 128, 129, 256)] == [64, 64, 128, 128, 256, 256]
    assert kv8.sizes(2, 80, 3, 5, 7) == dict(codes=3 * 2 * 2 * 128 * 64, marks=3 * 2 * 2 * 128, scales=12, open=5 * 2 * 64 * 2 * 80, table=35,
                                             workspace=(32 << 20) // 4)
    assert C.sizeof(L.StrataKv8Cache) == 72 and C.sizeof(L.StrataKv8CacheDev) == 80


def test_reference_quantisation():
    """The tests' own quantisation: half a step at most from the value, whole for its largest."""
    rng = np.random.default_rng(0)
    x = rng.normal(0, 3, (64, 40)).astype(np.float32)
    codes, scale = R.quantise(x)
    assert np.abs(codes).max() == 127 and np.abs(codes * np.float64(scale) - x).max() <= 0.5001 * scale
    assert R.quantise(np.zeros((3, 4), np.float32))[1] == 0


def test_sequence_batch_refuses_what_an_8_bit_cache_cannot_do():
    from oracle.backend import OracleBackend
    from oracle.oracle import Oracle
    from stratacuda_b200.engine import SequenceBatch, StrataEngine
    from stratacuda_b200.model import create_fixture
    engine = StrataEngine.create(create_fixture(), OracleBackend(Oracle("port")))
    with pytest.raises(ValueError, match="top needs kv8"):
        SequenceBatch(engine, 2, top=8)
    with pytest.raises(ValueError, match="at least 3"):
        SequenceBatch(engine, 2, kv8=True, top=2)
    with pytest.raises((TypeError, ValueError, RuntimeError)):
        SequenceBatch(engine, 2, kv8=True, top=1.5)
