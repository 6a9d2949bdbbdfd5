"""Token mixers over runs of many sequences on a B200, against their definitions in 64 bits.

Tolerances. u = 2^-24 is half a step of F32. An output of `inputs` or `qk_rope` goes through 4 products and sums of the
convolution or the norm (each u), an exponential and a division or square root (2 u each), and a rotation's two products and sum: at
most 16 roundings that matter to one element, 2^-20 of the magnitudes that its last sum adds. `rule`: the factors of a product keep
22 bits or more (2^-23 each, two of them), and five products follow one another (the system's inverse, differences from the state,
their correction, result, new state); |k| <= 1, beta <= 1 and decay <= 1 keep earlier errors from growing. Roundings are independent of
one another, so an output's error in the 2-norm is about sqrt(10) 2^-23 = 2^-21.3 of its norm: the bound is 2^-20. One element may
be 2^-14.5 of the root mean square of its head off, 45 times that: a Gaussian's tail, and rows that see more than the average.
"""
import numpy as np
import pytest

import mixers_reference as R
from stratacuda_b200 import _lib as L

pytestmark = pytest.mark.gpu
REL, ONE = 2.0 ** -20, 2.0 ** -14.5


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def near(got, want, heads=1, rel=REL, one=ONE):
    """got against want in the 2-norm, and each element against the root mean square of its head.

    Below 2^-126, F32's smallest normal number, there are no 24 bits to be right in: a state of 900 decays without any strength is
    1e-160 by the definition, which F32 does not have. An error of 2^-126 counts as none there."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape
    assert np.isfinite(got).all()
    norm = np.linalg.norm(want)
    assert np.linalg.norm(got - want) <= rel * norm, np.linalg.norm(got - want) / max(norm, 1e-300)
    g, w = got.reshape(-1, heads, got.shape[-1] // heads), want.reshape(-1, heads, want.shape[-1] // heads)
    rms = np.sqrt((w * w).mean((0, 2), keepdims=True))
    off = np.abs(g - w) / np.maximum(np.maximum(rms, np.abs(w)), 2.0 ** -126 / one)
    assert off.max() <= one, off.max()


class Net:
    """A rule call's tensors, and what it leaves."""

    def __init__(self, torch, kh, vh, dim, sequences, c, workspace=None, status=True):
        from stratacuda_b200.mixers import DeviceDeltaNet
        self.torch, self.kh, self.vh, self.dim = torch, kh, vh, dim
        self.t = {n: torch.tensor(a, device="cuda") for n, a in c.items()}
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.workspace = torch.zeros(L.DELTA_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda") if workspace is None else workspace
        self.net = DeviceDeltaNet(kh, vh, dim, sequences, state=self.t["state"], workspace=self.workspace, status=self.status)

    def ints(self, x):
        return None if x is None else self.torch.tensor(x, dtype=self.torch.int32, device="cuda")

    def rule(self, sequence, segments, count, lengths=None, y=None, **kw):
        t = self.t
        y = self.torch.full((segments * count, self.vh * self.dim), 7.0, device="cuda") if y is None else y
        self.net.rule(t["q"], t["k"], t["v"], t["decay"], t["beta"], y, self.ints(sequence), segments, count, self.ints(lengths),
                      stream=self.torch.cuda.current_stream().cuda_stream, **kw)
        self.torch.cuda.synchronize()
        return y.cpu().numpy()

    def state(self):
        return self.t["state"].cpu().numpy()


def check_rule(torch, kh, vh, dim, segments, count, sequence=None, lengths=None, sequences=None, edit=None, keys="mixed", seed=1, status=0, **tol):
    sequence = list(range(segments)) if sequence is None else sequence
    sequences = sequences or segments
    c = R.rule_case(np.random.default_rng(seed), kh, vh, dim, sequences, segments, count, keys)
    if edit:
        edit(c)
    net = Net(torch, kh, vh, dim, sequences, c)
    y = net.rule(sequence, segments, count, lengths)
    want, state = R.rule(c["q"], c["k"], c["v"], c["decay"], c["beta"], c["state"], kh, vh, dim, sequence, lengths, segments, count,
                         np.full((segments * count, vh * dim), 7.0))
    near(y, want, vh, **tol)
    near(net.state().reshape(-1, vh * dim), state.reshape(-1, vh * dim), vh, **tol)
    assert int(net.status.item()) == status
    # what the call leaves alone keeps its bits
    for i, s, n in R.runs(sequence, lengths, segments, count, sequences):
        if s >= 0:
            assert (y[i * count + n:(i + 1) * count] == 7.0).all()
        else:
            assert (y[i * count:(i + 1) * count] == 0.0).all()
    for s in set(range(sequences)) - {s for _, s, n in R.runs(sequence, lengths, segments, count, sequences) if n}:
        assert np.array_equal(net.state()[s], c["state"][s])
    return net, c, y


@pytest.mark.parametrize("count", [1, 2, 7, 63, 64, 65, 128, 129, 200])
@pytest.mark.parametrize("kh,vh,dim", [(2, 4, 128), (1, 3, 64)])
def test_rule_lengths_of_runs(torch, kh, vh, dim, count):
    check_rule(torch, kh, vh, dim, 1, count)


@pytest.mark.parametrize("dim", [1, 2, 3, 16, 31, 40, 63, 65, 80, 100, 127, 192, 255, 256])
@pytest.mark.parametrize("count", [3, 150])
def test_rule_head_sizes(torch, dim, count):
    check_rule(torch, 2, 4, dim, 2, count, seed=dim)


@pytest.mark.parametrize("kh,vh", [(1, 1), (3, 3), (5, 5), (1, 4), (3, 9), (2, 10)])
@pytest.mark.parametrize("count", [1, 70])
def test_rule_heads(torch, kh, vh, count):
    check_rule(torch, kh, vh, 64, 2, count, seed=vh)


@pytest.mark.parametrize("count", [1, 5, 130])
@pytest.mark.parametrize("dim", [64, 128])
def test_rule_ragged_runs(torch, count, dim):
    """Runs in another order than their sequences, with idle slots, lengths of zero, one and all, and sequences that have no run."""
    sequence = [6, -1, 2, 0, 7, 3, 4]
    lengths = [count, count, 0, 1, max(1, count // 2), max(1, count - 1), min(count, 64)]
    check_rule(torch, 2, 4, dim, 7, count, sequence, lengths, 9)


@pytest.mark.parametrize("count", [1, 100])
def test_rule_reports_what_is_outside(torch, count):
    """A sequence outside, one that an earlier run has, lengths outside: reported, left out or cut."""
    check_rule(torch, 1, 2, 64, 4, count, [1, 5, 2, 0], None, 3, status=1)
    check_rule(torch, 1, 2, 64, 4, count, [1, 2, 1, 0], None, 3, status=1)
    check_rule(torch, 1, 2, 64, 3, count, [1, -7, 0], None, 3, status=1)
    check_rule(torch, 1, 2, 64, 3, count, [1, 2, 0], [-4, count, count + 9], 3, status=1)


@pytest.mark.parametrize("count", [4, 64, 190, 900])
@pytest.mark.parametrize("what", ["zero decay", "some zero decays", "tiny decays", "ones", "no strength", "strength one, one key", "zero keys", "zero state"])
def test_rule_borders(torch, what, count):
    def edit(c):
        if what == "zero decay":
            c["decay"][:] = 0
        elif what == "some zero decays":
            c["decay"][::7] = 0
        elif what == "tiny decays":
            c["decay"][::5] = 1e-30
        elif what == "ones":
            c["decay"][:] = 1
        elif what == "no strength":
            c["beta"][:] = 0
        elif what == "strength one, one key":
            c["beta"][:] = 1
            c["decay"][:] = 1
        elif what == "zero keys":
            c["k"][::3] = 0
            c["q"][1::3] = 0
        else:
            c["state"][:] = 0
    check_rule(torch, 1, 2, 128, 2, count, edit=edit, keys="same" if "one key" in what else "mixed")


@pytest.mark.parametrize("count", [3, 140, 900])
@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e12, 1e17])
def test_rule_magnitudes(torch, count, scale):
    """Values and states of any size, and channels of one head that are far apart: each channel's error goes by its own."""
    def edit(c):
        c["v"] *= np.float32(scale)
        c["state"] *= np.float32(scale)
    check_rule(torch, 1, 2, 64, 1, count, edit=edit)

    def spread(c):
        by = (10.0 ** np.linspace(-12, 12, 128)).astype(np.float32)
        c["v"] *= by
        c["state"] *= by.reshape(2, 64)
    sequence = [0]
    c = R.rule_case(np.random.default_rng(4), 1, 2, 64, 1, 1, count)
    spread(c)
    net = Net(torch, 1, 2, 64, 1, c)
    y = net.rule(sequence, 1, count)
    want, state = R.rule(c["q"], c["k"], c["v"], c["decay"], c["beta"], c["state"], 1, 2, 64, sequence, None, 1, count, np.zeros((count, 128)))
    near(y, want, 128, rel=1.0, one=4 * ONE)  # heads of one channel each
    near(net.state().reshape(64, 128), state.reshape(64, 128), 128, rel=1.0, one=4 * ONE)


@pytest.mark.parametrize("count", [5, 150, 900])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("where", ["v", "k", "q", "decay", "beta"])
def test_rule_values_that_are_not_finite_stay_behind_their_token(torch, count, bad, where):
    """Tokens before one with a value that is not finite, other runs, heads that do not read it and rows behind a run's end do not
    see it; what follows is NaN or infinite where the definition says so."""
    kh, vh, dim, at = 2, 4, 64, count // 2
    c = R.rule_case(np.random.default_rng(8), kh, vh, dim, 2, 2, count)
    want, state = R.rule(c["q"], c["k"], c["v"], c["decay"], c["beta"], c["state"], kh, vh, dim, [0, 1], [count, count - 2], 2, count,
                         np.full((2 * count, vh * dim), 7.0))
    c[where][at, 1] = bad           # key head 0, or value head 1 of decay and beta, or channel 1 of value head 0
    c["v"][2 * count - 1] = np.nan  # behind the second run's end
    net = Net(torch, kh, vh, dim, 2, c)
    y = net.rule([0, 1], 2, count, [count, count - 2])
    near(y[:at], want[:at], vh)
    near(y[count:], want[count:], vh)
    clean = [h for h in range(vh) if h not in {"v": [0], "k": [0, 2], "q": [0, 2], "decay": [1], "beta": [1]}[where]]
    pick = lambda a: a.reshape(count, vh, dim)[:, clean].reshape(count, -1)  # noqa: E731
    near(pick(y[:count]), pick(want[:count]), len(clean))
    near(net.state()[1].reshape(dim, -1), state[1].reshape(dim, -1), vh)
    bad_y, bad_state = R.rule(c["q"], c["k"], c["v"], c["decay"], c["beta"], c["state"], kh, vh, dim, [0, 1], [count, count - 2], 2, count,
                              np.full((2 * count, vh * dim), 7.0))
    assert np.array_equal(np.isfinite(y), np.isfinite(bad_y))
    assert np.array_equal(np.isfinite(net.state()), np.isfinite(bad_state))


@pytest.mark.parametrize("cut", [1, 37, 64, 128])
def test_rule_in_two_calls(torch, cut):
    """A run that is split over calls ends where one call does."""
    kh, vh, dim, count = 2, 4, 128, 201
    c = R.rule_case(np.random.default_rng(9), kh, vh, dim, 1, 1, count)
    want, state = R.rule(c["q"], c["k"], c["v"], c["decay"], c["beta"], c["state"], kh, vh, dim, [0], None, 1, count, np.zeros((count, vh * dim)))
    net = Net(torch, kh, vh, dim, 1, c)
    whole = dict(net.t)
    got = []
    for a, b in ((0, cut), (cut, count)):
        net.t.update({n: whole[n][a:b].contiguous() for n in ("q", "k", "v", "decay", "beta")})
        got.append(net.rule([0], 1, b - a))
    near(np.concatenate(got), want, vh)
    near(net.state().reshape(dim, -1), state.reshape(dim, -1), vh)


@pytest.mark.parametrize("count", [2, 90])
@pytest.mark.parametrize("extra", [0, 1, 4])
def test_rule_reads_strided_rows(torch, count, extra):
    """q, k and v as columns of longer rows, on and off the 16-byte grid."""
    kh, vh, dim = 2, 4, 64
    c = R.rule_case(np.random.default_rng(10), kh, vh, dim, 1, 1, count)
    want, state = R.rule(c["q"], c["k"], c["v"], c["decay"], c["beta"], c["state"], kh, vh, dim, [0], None, 1, count, np.zeros((count, vh * dim)))
    net = Net(torch, kh, vh, dim, 1, c)
    wide = torch.full((count, 2 * kh * dim + vh * dim + 3 * extra), float("nan"), device="cuda")
    at = {"q": extra, "k": kh * dim + extra, "v": 2 * kh * dim + extra}
    for n, width in (("q", kh * dim), ("k", kh * dim), ("v", vh * dim)):
        wide[:, at[n]:at[n] + width] = net.t[n]
        net.t[n] = wide[:, at[n]:at[n] + width]
    y = net.rule([0], 1, count, q_stride=wide.shape[1], k_stride=wide.shape[1], v_stride=wide.shape[1])
    near(y, want, vh)
    near(net.state().reshape(dim, -1), state.reshape(dim, -1), vh)


@pytest.mark.parametrize("count", [1, 100])
def test_rule_off_the_16_byte_grid(torch, count):
    """State and result that start on odd floats."""
    kh, vh, dim = 1, 2, 64
    c = R.rule_case(np.random.default_rng(11), kh, vh, dim, 2, 2, count)
    want, state = R.rule(c["q"], c["k"], c["v"], c["decay"], c["beta"], c["state"], kh, vh, dim, [0, 1], None, 2, count, np.zeros((2 * count, vh * dim)))
    shifted = torch.zeros(c["state"].size + 1, device="cuda")[1:]
    shifted.copy_(torch.tensor(c["state"]).reshape(-1))
    net = Net(torch, kh, vh, dim, 2, c)
    from stratacuda_b200.mixers import DeviceDeltaNet
    net.net = DeviceDeltaNet(kh, vh, dim, 2, state=shifted, workspace=net.workspace)
    y = torch.zeros(2 * count * vh * dim + 3, device="cuda")[3:].reshape(2 * count, -1)
    near(net.rule([0, 1], 2, count, y=y), want, vh)
    near(shifted.cpu().numpy().reshape(-1, vh * dim), state.reshape(-1, vh * dim), vh)


@pytest.mark.parametrize("count", [1, 150, 900])
def test_rule_repeats_bit_for_bit_and_replays(torch, count):
    """The same call gives the same bits, eagerly, from a captured graph and on another stream."""
    kh, vh, dim = 2, 4, 128
    c = R.rule_case(np.random.default_rng(12), kh, vh, dim, 3, 3, count)
    net = Net(torch, kh, vh, dim, 3, c)
    first, after = net.rule([2, 0, 1], 3, count), net.state()
    start = torch.tensor(c["state"], device="cuda")
    y, sequence = torch.zeros(3 * count, vh * dim, device="cuda"), net.ints([2, 0, 1])
    side = torch.cuda.Stream()
    args = [net.t[n] for n in ("q", "k", "v", "decay", "beta")]
    net.t["state"].copy_(start)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        net.net.rule(*args, y, sequence, 3, count, stream=side.cuda_stream)
    torch.cuda.synchronize()
    assert np.array_equal(y.cpu().numpy(), first) and np.array_equal(net.state(), after)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        net.net.rule(*args, y, sequence, 3, count, stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(2):
        net.t["state"].copy_(start)
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(y.cpu().numpy(), first) and np.array_equal(net.state(), after)
    # other sequences and lengths under the same graph: both are read on the device
    sequence.copy_(net.ints([0, -1, 1]))
    net.t["state"].copy_(start)
    graph.replay()
    torch.cuda.synchronize()
    want, state = R.rule(c["q"], c["k"], c["v"], c["decay"], c["beta"], c["state"], kh, vh, dim, [0, -1, 1], None, 3, count,
                         np.zeros((3 * count, vh * dim)))
    near(y.cpu().numpy(), want, vh)
    near(net.state().reshape(-1, vh * dim), state.reshape(-1, vh * dim), vh)


def test_rule_of_more_chunks_than_the_workspace_holds(torch):
    """Many sequences with prompts: the work is taken in parts."""
    check_rule(torch, 8, 8, 128, 40, 321, lengths=[321 - 7 * i for i in range(40)])


@pytest.mark.parametrize("kh,vh,dim,segments,count,sequence,lengths", [
    (1, 2, 128, 1, 700, None, None), (2, 4, 64, 2, 1100, [1, 0], [1100, 641]), (1, 3, 40, 2, 800, None, [1, 800]), (1, 2, 65, 1, 900, None, None),
    (2, 2, 100, 3, 1000, [2, -1, 0], [999, 1000, 577]), (1, 1, 1, 2, 1500, None, None), (1, 1, 17, 4, 1500, [3, 1, 0, 2], [0, 64, 65, 1499]),
    (1, 1, 63, 1, 4097, None, None), (1, 1, 128, 1, 9001, None, None), (8, 24, 128, 1, 1100, None, None), (6, 24, 32, 1, 1030, None, None)])
def test_rule_in_parts(torch, kh, vh, dim, segments, count, sequence, lengths):
    """Runs of few states: parts at once, from the states that their ends and transitions give."""
    check_rule(torch, kh, vh, dim, segments, count, sequence, lengths, segments + 1, seed=count)


def test_rule_in_parts_of_more_than_the_workspace_holds(torch):
    check_rule(torch, 16, 16, 128, 1, 4000)


def test_rule_in_parts_that_would_blow_up(torch):
    """Keys of length 3: a state that is not zero grows past all bounds, one that is zero stays; one head of two."""
    def edit(c):
        c["k"][:, :64] = 3 * c["k"][:1, :64] / np.linalg.norm(c["k"][0, :64])
        c["v"][:, :64] = 0
        c["state"][:, :, 0] = 0
        c["beta"][:, 0] = 1
    _, _, y = check_rule(torch, 2, 2, 64, 1, 1000, edit=edit)
    assert (y[:, :64] == 0).all()


@pytest.mark.parametrize("lengths,sequence", [(None, None), ([1250, 1250], [1, 0]), ([1200, 3], None), ([700, 1250], [2, -1]), ([0, 64 * 9], None)])
def test_rule_of_few_long_runs(torch, lengths, sequence):
    """Parts of a prompt follow one another, the next one's first kernel beside the last one's second; runs end in all of them."""
    check_rule(torch, 16, 32, 64, 2, 1250, sequence, lengths, 3)


def test_rule_of_few_long_runs_repeats_and_replays(torch):
    """Two calls in a row, eagerly and from a graph: bit for bit the same, on one workspace."""
    kh, vh, dim, count = 16, 32, 128, 2500
    c = R.rule_case(np.random.default_rng(3), kh, vh, dim, 1, 1, count)
    net = Net(torch, kh, vh, dim, 1, c)
    start = torch.tensor(c["state"], device="cuda")
    args = [net.t[n] for n in ("q", "k", "v", "decay", "beta")]
    ys, sequence = [torch.zeros(count, vh * dim, device="cuda") for _ in range(2)], net.ints([0])

    def twice():
        for y in ys:
            net.net.rule(*args, y, sequence, 1, count, stream=torch.cuda.current_stream().cuda_stream)

    twice()
    torch.cuda.synchronize()
    first, after = [y.cpu().numpy() for y in ys], net.state()
    assert not np.array_equal(first[0], first[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        twice()
    for again in (twice, graph.replay, graph.replay):
        net.t["state"].copy_(start)
        again()
        torch.cuda.synchronize()
        assert all(np.array_equal(y.cpu().numpy(), f) for y, f in zip(ys, first)) and np.array_equal(net.state(), after)


@pytest.mark.parametrize("dim,count", [(64, 200), (128, 131)])
def test_rule_takes_long_runs_first(torch, dim, count):
    """More states than multiprocessors, runs of all lengths and of equal ones, idle ones, numbers outside and one sequence twice."""
    sequence = [(7 * i + 3) % 24 for i in range(24)]
    lengths = [(37 * i) % (count + 1) for i in range(24)]
    lengths[5] = lengths[6] = lengths[20] = count
    lengths[9] = 0
    sequence[11] = -1
    check_rule(torch, 4, 8, dim, 24, count, sequence, lengths, 24)
    sequence[3] = sequence[1]
    sequence[17], lengths[2], lengths[4] = 99, -5, count + 7
    check_rule(torch, 4, 8, dim, 24, count, sequence, lengths, 24, status=1)


# ---------------------------------------------------------------- inputs

@pytest.mark.parametrize("count", [1, 2, 3, 4, 15, 16, 17, 100])
@pytest.mark.parametrize("kh,vh,dim,taps", [(2, 4, 128, 4), (1, 3, 64, 4), (3, 3, 37, 4), (2, 2, 256, 3), (1, 2, 20, 8), (2, 2, 32, 1), (1, 1, 200, 2)])
def test_inputs(torch, kh, vh, dim, taps, count):
    from stratacuda_b200.mixers import DeviceDeltaNet
    rng = np.random.default_rng(count)
    sequence, lengths = [4, -1, 0, 2, 1], [count, count, 0, max(1, count - 1), (count + 1) // 2]
    channels = (2 * kh + vh) * dim
    x, w = rng.standard_normal((5 * count, channels)).astype(np.float32), rng.standard_normal((channels, taps)).astype(np.float32)
    history = rng.standard_normal((5, channels, taps - 1)).astype(np.float32)
    widths = (kh * dim, kh * dim, vh * dim)
    want = R.inputs(x, history, w, kh, vh, dim, sequence, lengths, 5, count, [np.full((5 * count, d), 7.0) for d in widths])
    dev = lambda a, t=None: torch.tensor(a, device="cuda", dtype=t)  # noqa: E731
    h, status = dev(history), torch.zeros(1, dtype=torch.int32, device="cuda")
    net = DeviceDeltaNet(kh, vh, dim, 5, taps, history=h, weight=dev(w), status=status)
    outs = [torch.full((5 * count, d), 7.0, device="cuda") for d in widths]
    net.inputs(dev(x), *outs, dev(sequence, torch.int32), 5, count, dev(lengths, torch.int32), stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for got, exact, heads in zip(outs, want, (kh, kh, vh)):
        near(got.cpu().numpy(), exact, heads, one=2.0 ** -18)
    assert np.array_equal(h.cpu().numpy(), want[3].astype(np.float32))  # inputs as they came
    assert int(status.item()) == 0
    for i, s, n in R.runs(sequence, lengths, 5, count, 5):
        for o in outs:
            rows = o[i * count:(i + 1) * count].cpu().numpy()
            assert (rows == 0).all() if s < 0 else (rows[n:] == 7.0).all()


@pytest.mark.parametrize("extra", [0, 1, 4])
def test_inputs_reads_strided_rows_and_takes_a_scale(torch, extra):
    from stratacuda_b200.mixers import DeviceDeltaNet
    rng = np.random.default_rng(3)
    kh, vh, dim, count = 2, 4, 64, 21
    channels = (2 * kh + vh) * dim
    x = rng.standard_normal((count, channels)).astype(np.float32)
    w, history = rng.standard_normal((channels, 4)).astype(np.float32), rng.standard_normal((1, channels, 3)).astype(np.float32)
    want = R.inputs(x, history, w, kh, vh, dim, [0], None, 1, count, [np.zeros((count, d)) for d in (kh * dim, kh * dim, vh * dim)], q_scale=0.25, eps=0.1)
    wide = torch.full((count, channels + 2 * extra), float("nan"), device="cuda")
    wide[:, extra:extra + channels] = torch.tensor(x, device="cuda")
    net = DeviceDeltaNet(kh, vh, dim, 1, history=torch.tensor(history, device="cuda"), weight=torch.tensor(w, device="cuda"))
    outs = [torch.zeros(count, d, device="cuda") for d in (kh * dim, kh * dim, vh * dim)]
    net.inputs(wide[:, extra:extra + channels], *outs, torch.zeros(1, dtype=torch.int32, device="cuda"), 1, count, row_stride=wide.shape[1],
               q_scale=0.25, epsilon=0.1, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for got, exact, heads in zip(outs, want, (kh, kh, vh)):
        near(got.cpu().numpy(), exact, heads, one=2.0 ** -18)


def test_inputs_reports_what_is_outside(torch):
    from stratacuda_b200.mixers import DeviceDeltaNet
    for sequence, lengths in (([0, 0], None), ([0, 2], None), ([0, -2], None), ([0, 1], [3, 9]), ([1, 0], [-1, 3])):
        rng = np.random.default_rng(5)
        x, w = rng.standard_normal((6, 64)).astype(np.float32), rng.standard_normal((64, 4)).astype(np.float32)
        history = rng.standard_normal((2, 64, 3)).astype(np.float32)
        want = R.inputs(x, history, w, 1, 2, 16, sequence, lengths, 2, 3, [np.zeros((6, d)) for d in (16, 16, 32)])
        h, status = torch.tensor(history, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        net = DeviceDeltaNet(1, 2, 16, 2, history=h, weight=torch.tensor(w, device="cuda"), status=status)
        outs = [torch.zeros(6, d, device="cuda") for d in (16, 16, 32)]
        ints = lambda a: None if a is None else torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        net.inputs(torch.tensor(x, device="cuda"), *outs, ints(sequence), 2, 3, ints(lengths), stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert int(status.item()) == 1
        for got, exact in zip(outs, want):
            near(got.cpu().numpy(), exact, one=2.0 ** -18)
        assert np.array_equal(h.cpu().numpy(), want[3].astype(np.float32))


# ---------------------------------------------------------------- qk_rope

@pytest.mark.parametrize("count", [1, 5, 33])
@pytest.mark.parametrize("heads,kv,dim,rotary,gated", [(16, 2, 256, 64, True), (4, 4, 128, 128, False), (6, 2, 64, 32, True), (3, 1, 32, 32, False),
                                                       (5, 3, 80, 48, True), (2, 2, 37, 10, False), (2, 1, 250, 250, True), (4, 2, 256, 256, False),
                                                       (3, 2, 96, 0, False), (1, 1, 256, 192, True), (2, 2, 2, 2, False), (1, 1, 1, 0, False)])
def test_qk_rope(torch, heads, kv, dim, rotary, gated, count):
    from stratacuda_b200.mixers import DeviceQkRope
    rng = np.random.default_rng(dim)
    cells, segments, apart = 50, 4, 2 * dim if gated else dim
    q, k = rng.standard_normal((segments * count, heads * apart)).astype(np.float32), rng.standard_normal((segments * count, kv * dim)).astype(np.float32)
    wq, wk = (rng.standard_normal(dim).astype(np.float32) for _ in range(2))
    angle = rng.standard_normal((cells, rotary // 2)) * 30
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    sequence, start, lengths = [9, -1, 0, 3], [0, 77, cells - count, 7], [count, count, count, count // 2]
    want = R.qk_rope(q, k, wq, wk, cos, sin, heads, kv, dim, rotary, sequence, start, lengths, segments, count,
                     np.full((segments * count, heads * dim), 7.0), np.full((segments * count, kv * dim), 7.0), apart)
    dev = lambda a, t=None: torch.tensor(a, device="cuda", dtype=t)  # noqa: E731
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    rope = DeviceQkRope(heads, kv, dim, rotary, cells, dev(wq), dev(wk), dev(cos) if rotary else None, dev(sin) if rotary else None, sequences=10, status=status)
    yq, yk = torch.full((segments * count, heads * dim), 7.0, device="cuda"), torch.full((segments * count, kv * dim), 7.0, device="cuda")
    i32 = torch.int32
    rope.apply(dev(q), dev(k), yq, yk, dev(start, i32), segments, count, dev(sequence, i32), dev(lengths, i32), q_head_stride=apart,
               stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    near(yq.cpu().numpy(), want[0], heads, one=2.0 ** -18)
    near(yk.cpu().numpy(), want[1], kv, one=2.0 ** -18)
    assert int(status.item()) == 0


def test_qk_rope_in_place_outside_and_strided(torch):
    """In place; a position outside the tables, before and behind; rows among others; epsilon; no list of sequences."""
    from stratacuda_b200.mixers import DeviceQkRope
    rng = np.random.default_rng(6)
    heads, kv, dim, rotary, cells, count = 4, 2, 64, 32, 20, 3
    cos, sin = (rng.standard_normal((cells, 16)).astype(np.float32) for _ in range(2))
    wq, wk = (rng.standard_normal(dim).astype(np.float32) for _ in range(2))
    q, k = rng.standard_normal((6, heads * dim)).astype(np.float32), rng.standard_normal((6, kv * dim)).astype(np.float32)
    dev = lambda a, t=None: torch.tensor(a, device="cuda", dtype=t)  # noqa: E731
    for start, status in (([3, 9], 0), ([-1, 4], 1), ([18, 0], 1), ([2 ** 31 - 2, 5], 1)):
        want = R.qk_rope(q, k, wq, wk, cos, sin, heads, kv, dim, rotary, None, start, None, 2, count, np.zeros(q.shape), np.zeros(k.shape), eps=0.3)
        word = torch.zeros(1, dtype=torch.int32, device="cuda")
        rope = DeviceQkRope(heads, kv, dim, rotary, cells, dev(wq), dev(wk), dev(cos), dev(sin), status=word)
        yq, yk = dev(q), dev(k)
        rope.apply(yq, yk, yq, yk, dev(start, torch.int32), 2, count, epsilon=0.3, stream=torch.cuda.current_stream().cuda_stream)
        wide = torch.full((6, (heads + kv) * dim + 1), float("nan"), device="cuda")
        wide[:, :heads * dim], wide[:, heads * dim:-1] = dev(q), dev(k)
        zq, zk = torch.zeros(6, heads * dim, device="cuda"), torch.zeros(6, kv * dim, device="cuda")
        rope.apply(wide[:, :heads * dim], wide[:, heads * dim:-1], zq, zk, dev(start, torch.int32), 2, count, q_stride=wide.shape[1],
                   k_stride=wide.shape[1], epsilon=0.3, stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert int(word.item()) == status
        for got, exact, h in ((yq, want[0], heads), (zq, want[0], heads), (yk, want[1], kv), (zk, want[1], kv)):
            near(got.cpu().numpy(), exact, h, one=2.0 ** -18)


# ---------------------------------------------------------------- together, through handles

@pytest.mark.parametrize("count", [1, 77])
def test_handles_run_a_layer(torch, count):
    """The inputs and the rule one after another on a context's buffers, twice, as a layer of a batch of sessions uses them."""
    from stratacuda_b200.backend import CudaBackend
    from stratacuda_b200.mixers import DeltaNet
    rng = np.random.default_rng(2)
    b = CudaBackend(0)
    kh, vh, dim, S = 2, 4, 64, 3
    channels, rows = (2 * kh + vh) * dim, S * count
    w = rng.standard_normal((channels, 4)).astype(np.float32)
    net = DeltaNet(b, kh, vh, dim, S, weight=b.alloc(w.ravel()))
    sequence = np.array([2, 0, -1], np.int32)
    seq = b.alloc(sequence, "i32")
    q, k, v, y = b.alloc(rows * kh * dim), b.alloc(rows * kh * dim), b.alloc(rows * vh * dim), b.alloc(rows * vh * dim)
    history, state = np.zeros((S, channels, 3)), np.zeros((S, dim, vh, dim))
    for _ in range(2):
        x = rng.standard_normal((rows, channels)).astype(np.float32)
        c = R.rule_case(rng, kh, vh, dim, S, S, count)
        net.inputs(b.alloc(x.ravel()), q, k, v, seq, S, count)
        net.rule(q, k, v, b.alloc(c["decay"].ravel()), b.alloc(c["beta"].ravel()), y, seq, S, count)
        *qkv, history = R.inputs(x, history, w, kh, vh, dim, sequence, None, S, count, [np.zeros((rows, d)) for d in (kh * dim, kh * dim, vh * dim)])
        want, state = R.rule(*qkv, c["decay"], c["beta"], state, kh, vh, dim, sequence, None, S, count, np.zeros((rows, vh * dim)))
        near(b.read(y).reshape(rows, -1), want, vh)
    near(b.read(net.state).reshape(-1, vh * dim), state.reshape(-1, vh * dim), vh)
    assert np.array_equal(b.read(net.history).reshape(history.shape), history.astype(np.float32))
    # a sequence outside is reported by the next synchronising call, and the context stays usable
    b.write(seq, np.array([2, 3, -1], np.int32))
    net.rule(q, k, v, b.alloc(c["decay"].ravel()), b.alloc(c["beta"].ravel()), y, seq, S, count)
    with pytest.raises(Exception, match="device check failed"):
        b.idle()
    b.idle()
    net.free()


def test_handles_refuse_buffers_that_are_too_short(torch):
    """Sizes are counted in 64 bits: numbers of sequences whose states would be 2^31 rows or more do not wrap round."""
    from stratacuda_b200.backend import CudaBackend, StrataError
    from stratacuda_b200.mixers import DeltaNet
    b = CudaBackend(0)
    kh, vh, dim = 1, 1, 128
    f, seq, work = b.alloc(16 * dim), b.alloc(np.zeros(1, np.int32), "i32"), b.alloc(L.DELTA_WORKSPACE_BYTES // 4, "u32", zero=False)
    state = b.alloc(dim * dim)
    for sequences in (2, 1 << 24, 1 << 25, (1 << 31) - 1):
        net = DeltaNet(b, kh, vh, dim, sequences, state=state, history=f, weight=f, workspace=work)
        with pytest.raises(StrataError, match="state needs"):
            net.rule(f, f, f, f, f, f, seq)
        with pytest.raises(StrataError, match="history needs"):
            net.inputs(f, f, f, f, seq)
    net = DeltaNet(b, kh, vh, dim, 1, state=state, history=f, weight=f, workspace=work)
    for short in ("q", "v", "y"):
        with pytest.raises(StrataError, match=short + " needs"):
            net.rule(**{**dict(q=f, k=f, v=f, decay=f, beta=f, y=f), short: seq}, sequence=seq)
    with pytest.raises(StrataError, match="workspace needs"):
        DeltaNet(b, kh, vh, dim, 1, state=state, history=f, weight=f, workspace=f).rule(f, f, f, f, f, f, seq)
