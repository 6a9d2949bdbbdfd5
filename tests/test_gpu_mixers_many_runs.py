"""Calls of thousands of runs on a B200: sequences that are outside or there twice, wherever they stand, and what a run costs."""
import numpy as np
import pytest

import mixers_reference as R
from test_gpu_mixers import Net, near

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def rule_of_many(c, kh, vh, dim, sequence, lengths, count):
    """R.rule, token by token over all runs at once; y (7 where no token is) and the states after."""
    c = {n: a.astype(np.float64) for n, a in c.items()}
    segments, of = len(sequence), np.arange(vh) % kh
    live = [(i, s, n) for i, s, n in R.runs(sequence, lengths, segments, count, len(c["state"])) if s >= 0]
    y, state = np.zeros((segments, count, vh * dim)), c["state"].copy()
    for i, s, n in live:
        y[i] = 7.0
    run, seq, length = (np.array(x) for x in zip(*live))
    S = state[seq].transpose(0, 2, 1, 3)  # [run, vh, key, value]
    row = {n: c[n].reshape(segments, count, -1) for n in ("q", "k", "v", "decay", "beta")}
    for t in range(count):
        m = length > t
        at = run[m]
        k, q = (row[n][at, t].reshape(-1, kh, dim)[:, of] for n in ("k", "q"))
        s = S[m] * row["decay"][at, t][:, :, None, None]
        d = row["beta"][at, t][:, :, None] * (row["v"][at, t].reshape(-1, vh, dim) - np.einsum("rhkv,rhk->rhv", s, k))
        s = s + k[:, :, :, None] * d[:, :, None]
        S[m] = s
        y[at, t] = np.einsum("rhkv,rhk->rhv", s, q).reshape(len(at), -1)
    state[seq] = S.transpose(0, 2, 1, 3)
    return y.reshape(segments * count, -1), state


@pytest.mark.parametrize("segments,count,dim", [(1024, 1, 16), (1025, 1, 16), (3001, 2, 16), (3001, 2, 40), (5000, 1, 8), (1100, 50, 8), (4001, 46, 8)])
@pytest.mark.parametrize("wrong", [False, True])
def test_rule_of_many_runs(torch, segments, count, dim, wrong):
    """In tokens and in chunks; idle runs, runs without tokens, and sequences twice: next to one another, far apart, first and last."""
    kh, vh, rng = 1, 2, np.random.default_rng(segments)
    sequences = segments + 3
    sequence = rng.permutation(sequences)[:segments].tolist()
    lengths = rng.integers(0, count + 1, segments).tolist()
    for i in range(5, segments, 97):
        sequence[i] = -1
    if wrong:
        sequence[segments - 1] = sequence[0]
        sequence[segments // 2] = sequence[segments // 2 - 1]
        sequence[130], sequence[131], sequence[128] = sequence[2], sequence[2], sequence[127]
        sequence[1023], sequence[700], sequence[701] = sequence[1022], sequences, -2
    c = R.rule_case(rng, kh, vh, dim, sequences, segments, count)
    net = Net(torch, kh, vh, dim, sequences, c)
    y = net.rule(sequence, segments, count, lengths)
    want, state = rule_of_many(c, kh, vh, dim, sequence, lengths, count)
    near(y, want, vh)
    near(net.state().reshape(-1, vh * dim), state.reshape(-1, vh * dim), vh)
    assert int(net.status.item()) == int(wrong)
    touched = {s for _, s, n in R.runs(sequence, lengths, segments, count, sequences) if s >= 0 and n}
    for s in set(range(sequences)) - touched:
        assert np.array_equal(net.state()[s], c["state"][s])


def test_a_run_costs_the_same_in_calls_of_many(torch):
    """The look for sequences that are there twice does not grow with the square of the runs: 65535 single tokens take at most twice as
    long for each run as 4096 do (states past L2 both times: 1.0 by their bytes; 2.7 with a look for each block)."""
    from stratacuda_b200 import _lib as L
    from stratacuda_b200.mixers import DeviceDeltaNet
    kh, vh, dim, times = 2, 4, 64, {}
    workspace = torch.zeros(L.DELTA_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    for segments in (4096, 65535):
        state = torch.zeros(segments * dim * vh * dim, device="cuda")
        net = DeviceDeltaNet(kh, vh, dim, segments, state=state, workspace=workspace)
        q, k, v, y = (torch.zeros(segments, n * dim, device="cuda") for n in (kh, kh, vh, vh))
        a = torch.ones(segments, vh, device="cuda")
        sequence = torch.randperm(segments, device="cuda").to(torch.int32)
        took = []
        for _ in range(6):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            net.rule(q, k, v, a, a, y, sequence, segments, 1, stream=torch.cuda.current_stream().cuda_stream)
            end.record()
            torch.cuda.synchronize()
            took.append(begin.elapsed_time(end))
        times[segments] = min(took) / segments
    assert times[65535] <= 2 * times[4096], times
