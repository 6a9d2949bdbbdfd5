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


# ---------------------------------------------------------------- tensors

class Calls:
    """Stands in for the library: keeps the calls that would have gone through."""

    def __init__(self):
        self.made = []

    def strata_kv8_call_dev(self, call):
        self.made.append(L.KV8_CALL.unpack(call))
        return L.OK


def tensors(device=0, **kw):
    """A DeviceCache of tensors (2 heads of 72, 3 sequences of 5 blocks, 17 pages) that say they are on `device`, and the
    arguments of a call on 3 runs of 4 tokens, by name; `kw` changes some of either."""
    import torch

    class On(torch.Tensor):
        def get_device(self):
            return getattr(self, "claimed", device)

    def make(shape, dtype=torch.float32):
        return torch.zeros(shape, dtype=dtype).as_subclass(On)

    parts = dict(codes=make((17, 2, 2, 128 * 64), torch.int8), marks=make((17, 2, 2, 128), torch.int8), scales=make((17, 2, 2)),
                 open=make((3, 2, 64, 2, 72)), table=make((3, 5), torch.int32), workspace=make(L.KV8_WORKSPACE_BYTES, torch.uint8),
                 status=make(1, torch.int32))
    arguments = dict(k=make((12, 144)), v=make((12, 144)), q=make((12, 6 * 72)), y=make((12, 6 * 72)), sequence=make(3, torch.int32),
                     start=make(3, torch.int32), picks=make((12, 2, 4), torch.int32))
    for name, change in kw.items():
        where = parts if name in parts else arguments
        where[name] = change(where[name])
    c = kv8.DeviceCache(2, 72, 17, 3, 5, **parts)
    c.lib = Calls()
    return c, arguments


def every_call(c, a, **kw):
    common = dict(sequence=a["sequence"], start=a["start"], segments=3, count=4, **kw)
    return {"append": lambda: c.append(a["k"], a["v"], **common), "select": lambda: c.select(a["q"], 6, a["picks"], top=4, **common),
            "attend": lambda: c.attend(a["q"], 6, a["y"], **common), "sparse": lambda: c.attend(a["q"], 6, a["y"], picks=a["picks"], top=4, **common)}


def elsewhere(where):
    def change(t):
        t.claimed = where
        return t
    return change


def test_tensors_as_they_should_be_go_through():
    c, a = tensors()
    for call in every_call(c, a).values():
        call()
    assert len(c.lib.made) == 4
    made = c.lib.made[0]
    assert made[1:3] == (a["k"].data_ptr(), a["v"].data_ptr()) and made[4:6] == (a["sequence"].data_ptr(), a["start"].data_ptr())
    assert c.lib.made[3][6:8] == (a["picks"].data_ptr(), a["y"].data_ptr()) and c.lib.made[2][6] == 0


@pytest.mark.parametrize("part", ["codes", "marks", "scales", "open", "table", "workspace", "status"])
def test_a_cache_of_tensors_refuses_parts_that_are_none(part):
    import torch
    cut = dict(codes=lambda t: t[:-1], marks=lambda t: t[:-1], scales=lambda t: t[1:], open=lambda t: t[:2], table=lambda t: t[:, :4].contiguous(),
               workspace=lambda t: t[1:], status=lambda t: t[:0])
    changes = [("needs", cut[part]), ("CUDA device", elsewhere(-1)), ("CUDA device", elsewhere(1))]
    if part not in ("workspace", "status"):
        changes += [("torch", lambda t: t.to(torch.float64)), ("torch", lambda t: t.to(torch.int16))]
        changes += [("contiguous", lambda t: t.transpose(0, 1))]
    for text, change in changes:
        assert refuse(kv8.StrataError, text, lambda: tensors(**{part: change})) == L.ERR_LAYOUT, text


def test_tensors_on_the_host_are_refused():
    for where in (-1, None):
        kw = dict(device=-1) if where else {n: elsewhere(-1) for n in ("codes",)}
        assert refuse(kv8.StrataError, "CUDA device", lambda: tensors(**kw)) == L.ERR_LAYOUT


@pytest.mark.parametrize("name,calls", [("k", ["append"]), ("v", ["append"]), ("q", ["select", "attend", "sparse"]), ("y", ["attend", "sparse"]),
                                        ("picks", ["select", "sparse"]), ("sequence", None), ("start", None)])
def test_calls_refuse_tensors_that_do_not_hold_their_argument(name, calls):
    import torch
    changes = [("needs", lambda t: t[:-1]), ("CUDA device", elsewhere(-1)), ("CUDA device", elsewhere(1)), ("torch", lambda t: t.to(torch.float16)),
               ("torch", lambda t: t.to(torch.int64)), ("torch", lambda t: t.double()),
               ("contiguous", lambda t: t.repeat(*[1] * (t.dim() - 1), 2)[..., ::2])]
    for text, change in changes:
        c, a = tensors(**{name: change})
        for which, call in every_call(c, a).items():
            if calls is None or which in calls:
                assert refuse(kv8.StrataError, text, call) == L.ERR_LAYOUT, (which, text)
            else:
                call()
        assert len(c.lib.made) == (4 - len(calls) if calls else 0)


def test_rows_some_way_apart():
    """row_stride says how far: of a view of longer rows, or of a tensor that has them whole; of nothing else."""
    import torch
    for change, stride, text in ((lambda t: t.repeat(1, 3)[:, 5:149], 432, None), (lambda t: t.repeat(1, 3), 432, None),
                                 (lambda t: t.repeat(1, 3)[:, 5:149], 431, "apart"), (lambda t: t.repeat(1, 3)[:, 5:148], 432, "apart"),
                                 (lambda t: t.repeat(1, 3)[:11, 5:149], 432, "apart"), (lambda t: t.repeat(3, 1)[::3], 432, None),
                                 (lambda t: t.repeat(1, 2)[:, ::2], 288, "apart"), (lambda t: t.repeat(1, 3)[:11], 432, "needs"),
                                 (lambda t: t, 145, "needs"), (lambda t: t.half().repeat(1, 3)[:, 5:149], 432, "torch"),
                                 (lambda t: t.repeat(1, 3)[:, 5:149].unsqueeze(0), 432, "apart")):
        c, a = tensors(k=change, v=change)
        call = every_call(c, a, row_stride=stride)["append"]
        if text is None:
            call()
            assert c.lib.made[0][1] == a["k"].data_ptr() and c.lib.made[0][3] == stride
        else:
            assert refuse(kv8.StrataError, text, call) == L.ERR_LAYOUT
            assert not c.lib.made


def test_addresses_and_tensors_mix():
    """Addresses are the caller's word; tensors beside them are still looked at."""
    c, a = tensors()
    d = cache(kv_heads=2, dim=72, pages=17, sequences=3, blocks=5)
    d.lib = Calls()
    for call in every_call(d, a).values():
        call()
    every_call(c, dict.fromkeys(a, A))["sparse"]()
    assert len(d.lib.made) == 4 and len(c.lib.made) == 1
    a["q"] = a["q"].half()
    assert refuse(kv8.StrataError, "torch", every_call(d, a)["attend"]) == L.ERR_LAYOUT


# ---------------------------------------------------------------- the selection's rounding

@pytest.mark.parametrize("dim,group,blocks,top", [(256, 12, 1024, 32), (128, 4, 512, 16), (64, 1, 300, 8)])
def test_rounded_scores_pick_what_the_marks_bound_picks(dim, group, blocks, top):
    """Queries rounded to 8 bits choose at least 15 of 16 blocks that the bound itself would choose, with keys some of whose channels
    are loud; and the bound is one: no block's summed logits pass it."""
    import numpy as np

    import kv8_reference as R
    rng = np.random.default_rng(1)
    loud, size = 1 + 3 * (rng.random(dim) < 0.06), np.exp(0.3 * rng.normal(size=(blocks, 1, 1)))
    keys = (rng.normal(size=(blocks, 64, dim)) + rng.normal(size=(blocks, 1, dim))) * size * loud
    scales = (np.abs(keys).max((1, 2)) / 127).astype(np.float32)
    codes = np.clip(np.rint(keys / scales[:, None, None]), -127, 127)
    lo, hi = codes.min(1), codes.max(1)
    same = []
    for _ in range(16):
        q = rng.normal(size=(group, dim)).astype(np.float32)
        bound = (hi @ np.maximum(q, 0).sum(0) + lo @ np.minimum(q, 0).sum(0)) * scales
        logits = ((codes * scales[:, None, None]) @ q.T.astype(np.float64)).sum(-1)
        assert (logits.max(1) <= bound * (1 + 1e-6) + 1e-6).all()
        order = bound.copy()
        order[:1] = order[-2:] = np.inf
        want = np.argsort(-order, kind="stable")[:top]
        same.append(np.isin(want, R.select(q, (lo, hi), scales, blocks, top, 1, 2)).mean())
    assert np.mean(same) >= 15 / 16
