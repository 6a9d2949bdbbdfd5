"""Refusals of the token mixers' pointer entries and host-side sizes: no GPU is touched."""
import ctypes as C

import pytest

from stratacuda_b200 import _lib as L
from stratacuda_b200 import mixers
from stratacuda_b200.backend import StrataError, StrataRangeError

A = 0x1000  # an aligned address that is never followed


def net(**kw):
    return mixers.DeviceDeltaNet(**{**dict(key_heads=2, value_heads=4, dim=64, sequences=3, state=A, history=A, weight=A, workspace=A), **kw})


def rope(**kw):
    return mixers.DeviceQkRope(**{**dict(heads=4, kv_heads=2, dim=64, rotary=32, cells=10, q_weight=A, k_weight=A, cos=A, sin=A), **kw})


def inputs(n, **kw):
    n.inputs(**{**dict(x=A, q=A, k=A, v=A, sequence=A), **kw})


def rule(n, **kw):
    n.rule(**{**dict(q=A, k=A, v=A, decay=A, beta=A, y=A, sequence=A), **kw})


def apply(n, **kw):
    n.apply(**{**dict(q=A, k=A, yq=A, yk=A, start=A), **kw})


def refuse(kind, text, call):
    with pytest.raises(kind, match=text) as e:
        call()
    return e.value.code


@pytest.mark.parametrize("call", [inputs, rule])
@pytest.mark.parametrize("bad,text", [(dict(key_heads=0), "key_heads"), (dict(key_heads=5000, value_heads=5000), "key_heads"),
                                      (dict(value_heads=5), "multiple"), (dict(value_heads=0), "value_heads"), (dict(value_heads=8192), "value_heads"),
                                      (dict(dim=0), "dim"), (dict(dim=257), "dim"), (dict(taps=0), "taps"), (dict(taps=9), "taps"),
                                      (dict(sequences=0), "sequences")])
def test_refuses_a_net_that_is_none(call, bad, text):
    assert refuse(StrataRangeError, text, lambda: call(net(**bad))) == L.ERR_RANGE


@pytest.mark.parametrize("call,make", [(inputs, net), (rule, net), (apply, rope)])
@pytest.mark.parametrize("bad,text", [(dict(segments=0), "segments"), (dict(segments=65536), "segments"), (dict(count=0), "count"),
                                      (dict(segments=60000, count=60000), "2\\^24")])
def test_refuses_runs(call, make, bad, text):
    assert refuse(StrataRangeError, text, lambda: call(make(), **bad)) == L.ERR_RANGE


@pytest.mark.parametrize("call,make,parts", [(inputs, net, ["x", "q", "k", "v", "sequence"]),
                                             (rule, net, ["q", "k", "v", "decay", "beta", "y", "sequence"]),
                                             (apply, rope, ["q", "k", "yq", "yk", "start"])])
def test_refuses_null_and_odd_addresses(call, make, parts):
    for p in parts:
        assert refuse(StrataRangeError, "null", lambda: call(make(), **{p: 0})) == L.ERR_RANGE
        assert refuse(StrataError, "4-byte", lambda: call(make(), **{p: A + 2})) == L.ERR_LAYOUT
    assert refuse(StrataError, "4-byte", lambda: call(make(), lengths=A + 2)) == L.ERR_LAYOUT
    assert refuse(StrataError, "4-byte", lambda: call(make(status=A + 1))) == L.ERR_LAYOUT


def test_refuses_parts_that_an_operator_needs():
    for bad in (dict(weight=None), dict(history=None)):
        assert refuse(StrataRangeError, "null", lambda: inputs(net(**bad))) == L.ERR_RANGE
    for bad in (dict(state=None), dict(workspace=None)):
        assert refuse(StrataRangeError, "null", lambda: rule(net(**bad))) == L.ERR_RANGE
    assert refuse(StrataError, "128-byte", lambda: rule(net(workspace=A + 64))) == L.ERR_LAYOUT
    for bad in (dict(q_weight=0), dict(k_weight=0), dict(cos=None), dict(sin=None)):
        assert refuse(StrataRangeError, "null", lambda: apply(rope(**bad))) == L.ERR_RANGE


@pytest.mark.parametrize("call,make,bad", [(inputs, net, dict(row_stride=511)), (rule, net, dict(q_stride=127)), (rule, net, dict(k_stride=1)),
                                           (rule, net, dict(v_stride=255)), (rule, net, dict(v_stride=1 << 50)), (apply, rope, dict(q_stride=255)),
                                           (apply, rope, dict(q_head_stride=63)), (apply, rope, dict(q_head_stride=1 << 30)),
                                           (apply, rope, dict(q_head_stride=128, q_stride=447)), (apply, rope, dict(k_stride=127))])
def test_refuses_strides(call, make, bad):
    assert refuse(StrataError, "stride", lambda: call(make(), **bad)) == L.ERR_LAYOUT


@pytest.mark.parametrize("bad", [dict(q_scale=float("inf")), dict(q_scale=float("nan")), dict(epsilon=-1.0), dict(epsilon=float("nan"))])
def test_refuses_numbers(bad):
    assert refuse(StrataRangeError, "finite", lambda: inputs(net(), **bad)) == L.ERR_RANGE
    if "epsilon" in bad:
        assert refuse(StrataRangeError, "finite", lambda: apply(rope(), **bad)) == L.ERR_RANGE


@pytest.mark.parametrize("bad,text", [(dict(heads=0), "heads"), (dict(kv_heads=0), "kv_heads"), (dict(dim=0, rotary=0), "dim"), (dict(dim=300), "dim"),
                                      (dict(rotary=3), "rotary"), (dict(rotary=66), "rotary"), (dict(rotary=-2), "rotary"), (dict(cells=0), "cells")])
def test_refuses_weights(bad, text):
    assert refuse(StrataRangeError, text, lambda: apply(rope(**bad))) == L.ERR_RANGE


def test_refuses_integers_past_32_bits():
    for bad in (dict(segments=1 << 32), dict(count=(1 << 32) + 1)):
        for call, make in ((inputs, net), (rule, net), (apply, rope)):
            assert refuse(StrataRangeError, "not a number of its type", lambda: call(make(), **bad)) == L.ERR_RANGE
    assert refuse(StrataRangeError, "32-bit", lambda: net(dim=(1 << 32) + 64)) == L.ERR_RANGE
    assert refuse(StrataRangeError, "32-bit", lambda: rope(cells=1 << 31)) == L.ERR_RANGE


def test_refuses_null_calls():
    lib = L.load()
    for entry in (lib.strata_delta_inputs_dev, lib.strata_delta_rule_dev, lib.strata_qk_rope_dev):
        assert entry(None) == L.ERR_RANGE
    for pack, entry, n in ((L.DELTA_INPUTS_CALL, lib.strata_delta_inputs_dev, 11), (L.DELTA_RULE_CALL, lib.strata_delta_rule_dev, 15),
                           (L.QK_ROPE_CALL, lib.strata_qk_rope_dev, 14)):
        tail = {L.DELTA_INPUTS_CALL: (1, 1, 0.0, 0.0), L.DELTA_RULE_CALL: (1, 1), L.QK_ROPE_CALL: (1, 1, 0.0)}[pack]
        assert entry(pack.pack(*[0] * n, *tail)) == L.ERR_RANGE  # no message wanted, no net or weights


def test_refuses_tensors_that_are_not_as_they_should_be():
    torch = pytest.importorskip("torch")
    x = torch.zeros(64, 512)
    assert refuse(StrataError, "CUDA device", lambda: inputs(net(), x=x)) == L.ERR_LAYOUT
    assert refuse(StrataError, "float32", lambda: rule(net(), q=x.double())) == L.ERR_LAYOUT
    assert refuse(StrataError, "int32", lambda: rule(net(), sequence=x)) == L.ERR_LAYOUT
    assert refuse(StrataError, "CUDA device", lambda: net(state=torch.zeros(3 * 64 * 4 * 64))) == L.ERR_LAYOUT


def test_refuses_the_default_stream_of_another_device(monkeypatch):
    torch = pytest.importorskip("torch")

    class Elsewhere:  # what is looked at of a tensor on device 1
        def __init__(self, dtype=torch.float32):
            self.dtype = dtype
        get_device, numel, is_contiguous, data_ptr = lambda _: 1, lambda _: 1 << 40, lambda _: True, lambda _: A
        element_size = lambda _: 4  # noqa: E731

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    x = Elsewhere()
    for call, make in ((inputs, lambda: net(state=x, history=x, weight=x)), (rule, lambda: net(state=x, history=x, weight=x)),
                       (apply, lambda: rope(q_weight=x, k_weight=x, cos=x, sin=x))):
        assert refuse(StrataError, "default stream", lambda: call(make())) == L.ERR_LAYOUT


@pytest.mark.parametrize("stream", [0, 0x7000])
def test_refuses_streams_of_a_device_that_is_not_the_parts(monkeypatch, stream):
    """A stream goes with the current device (the launch refuses others), so that is the one that has to hold the parts."""
    torch = pytest.importorskip("torch")

    class There:  # what is looked at of a tensor on device 1
        dtype = torch.float32
        get_device, numel, is_contiguous, data_ptr, element_size = lambda _: 1, lambda _: 1 << 40, lambda _: True, lambda _: A, lambda _: 4

    x = There()
    for call, make in ((inputs, lambda: net(state=x, history=x, weight=x)), (rule, lambda: net(state=x, history=x, weight=x)),
                       (apply, lambda: rope(q_weight=x, k_weight=x, cos=x, sin=x))):
        monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
        assert refuse(StrataError, "default stream", lambda: call(make(), stream=stream)) == L.ERR_LAYOUT
        monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
        assert refuse(StrataRangeError, "segments", lambda: call(make(), segments=0, stream=stream)) == L.ERR_RANGE  # past that check


def test_other_backends_are_refused():
    class Other:
        kind = "other"
    for make in (lambda: mixers.DeltaNet(Other(), 1, 1, 64, 1), lambda: mixers.QkRope(Other(), 1, 1, 64, 32, 8, None, None)):
        assert refuse(StrataRangeError, "CUDA backend", make) == L.ERR_RANGE


def test_a_net_gives_its_buffers_back_when_a_later_one_fails():
    class Failing:
        kind = "cuda"

        def __init__(self):
            self.live = set()

        def alloc(self, length, type="f32", zero=True):
            if len(self.live) == 2:
                raise MemoryError("no more")
            buf = object()
            self.live.add(buf)
            return buf

        def free(self, buf):
            self.live.remove(buf)

    b = Failing()
    with pytest.raises(MemoryError):
        mixers.DeltaNet(b, 1, 1, 64, 1)
    assert not b.live


def test_sizes():
    assert mixers.sizes(16, 32, 128, 3) == dict(state=3 * 128 * 32 * 128, history=3 * 64 * 128 * 3, weight=64 * 128 * 4, workspace=32 << 20)
    assert C.sizeof(L.StrataDeltaNetDev) == 64 and C.sizeof(L.StrataQkRopeWeightsDev) == 64


def test_handles_refuse_strides_that_64_bits_do_not_hold():
    """ctypes cuts integers down to 64 bits without a word: 2^64 + 512 would pass for rows 512 floats apart."""
    class Lib:
        def __getattr__(self, name):
            def entry(*args):
                raise AssertionError(f"{name} was reached")
            return entry

    class Buf:
        handle = 1

    class Backend:
        kind, lib, ctx = "cuda", Lib(), None
        alloc = lambda *_, **__: Buf()  # noqa: E731

    x = Buf()
    delta, qk = mixers.DeltaNet(Backend(), 2, 4, 64, 3, weight=x), mixers.QkRope(Backend(), 4, 2, 64, 32, 10, x, x, x, x)
    for bad in ((1 << 64) + 512, -1, -(1 << 64) + 512, 1 << 64, 512.0):
        calls = [lambda: delta.inputs(x, x, x, x, x, row_stride=bad)]
        calls += [lambda n=n: delta.rule(x, x, x, x, x, x, x, **{n: bad}) for n in ("q_stride", "k_stride", "v_stride")]
        calls += [lambda n=n: qk.apply(x, x, x, x, x, **{n: bad}) for n in ("q_stride", "q_head_stride", "k_stride")]
        for call in calls:
            assert refuse(StrataRangeError, "stride", call) == L.ERR_RANGE


class Counting:
    """A backend that only counts what it has handed out; `room` allocations of any size."""
    kind = "cuda"

    def __init__(self, room=1 << 30):
        self.live, self.room = {}, room

    def alloc(self, length, type="f32", zero=True):
        if not self.room:
            raise MemoryError("no more")
        self.room -= 1
        buf = object()
        self.live[id(buf)] = (buf, length)
        return buf

    def write(self, buf, data):
        assert id(buf) in self.live

    def free(self, buf):
        del self.live[id(buf)]

    def words(self):
        return sum(n for _, n in self.live.values())


def run_mixers(b, sequences=1):
    from types import SimpleNamespace

    from stratacuda_b200.engine import RunMixers
    return RunMixers(SimpleNamespace(b=b, g={}), [], sequences)


def test_sessions_of_a_backend_share_a_workspace():
    """Engines and batches of one backend follow one another on its stream: 64 sessions need one workspace, not 8 GB of them."""
    b, other = Counting(), Counting()
    held = [run_mixers(b) for _ in range(64)]
    apart = run_mixers(other)
    assert b.words() == L.DELTA_WORKSPACE_BYTES // 4 + 64
    assert len({id(r.workspace) for r in held}) == 1 and apart.workspace is not held[0].workspace
    for r in held[:-1]:
        r.free()
        r.free()  # twice: as once
    assert b.words() == L.DELTA_WORKSPACE_BYTES // 4 + 1
    again = run_mixers(b)
    assert again.workspace is held[-1].workspace
    held[-1].free(), again.free()
    assert not b.live
    new = run_mixers(b)  # the last one's is gone
    assert id(new.workspace) in b.live
    new.free(), apart.free()
    assert not b.live and not other.live


def test_a_session_that_cannot_be_made_leaves_the_workspace_to_the_others():
    b = Counting(room=2)
    first = run_mixers(b)
    with pytest.raises(MemoryError):
        run_mixers(b)
    assert id(first.workspace) in b.live
    first.free()
    assert not b.live
    b.room = 1  # the workspace, and then nothing
    with pytest.raises(MemoryError):
        run_mixers(b)
    assert not b.live
