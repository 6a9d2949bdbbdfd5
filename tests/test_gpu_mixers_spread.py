"""The gated delta rule over runs where tokens differ in size by many powers of ten, on a B200 against its definition in 64 bits.

Tolerances. A token's result may be off by what F32 loses of the magnitudes that its state holds, and by nothing that comes later or
that a decay has taken away. With e_j = |beta_j| (|v_j| + |prediction_j|), what a difference is made from, and G_tj the product of the
decays after token j up to t, a state column holds  H_t^2 = sum_{j <= t} (G_tj |k_j| e_j)^2 + (P_t |S|)^2,  each term with independent
roundings of its own: factors of 22 bits (2^-23 each, two of them) through five products, 2^-21.3 as in the rule's other tests. A result
is then |q_t| H_t 2^-21.3 off: 2^-20 of |q_t| H_t in the 2-norm over a token's channels, 45 times the typical error, 2^-14.5, for one of
its elements. beta |k|^2 <= 1 and decays up to one keep earlier errors from growing."""
import numpy as np
import pytest

import mixers_reference as R
from test_gpu_mixers import ONE, REL, Net

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def walk(c, kh, vh, dim, segments, count, lengths=None):
    """y, states after, and what a token's results and the states' columns hold; run i is sequence i's."""
    c = {n: a.astype(np.float64) for n, a in c.items()}
    y, hold = np.zeros((segments * count, vh, dim)), np.ones((segments * count, vh, dim))
    states, holds, of = np.zeros((segments, vh, dim, dim)), np.zeros((segments, vh, dim)), np.arange(vh) % kh
    for i in range(segments):
        S = c["state"][i].transpose(1, 0, 2)  # [vh, key, value]
        H = np.sqrt((S * S).sum(1))
        for r in range(i * count, i * count + (count if lengths is None else lengths[i])):
            k, q = c["k"][r].reshape(kh, dim)[of], c["q"][r].reshape(kh, dim)[of]
            a, b, v = c["decay"][r][:, None], c["beta"][r][:, None], c["v"][r].reshape(vh, dim)
            S = S * a[:, None]
            p = np.einsum("hkv,hk->hv", S, k)
            S = S + k[:, :, None] * (b * (v - p))[:, None]
            e = np.abs(b) * (np.abs(v) + np.abs(p)) * np.linalg.norm(k, axis=1)[:, None]
            H = np.sqrt((H * a) ** 2 + e * e)
            y[r], hold[r] = np.einsum("hkv,hk->hv", S, q), H * np.linalg.norm(q, axis=1)[:, None]
        states[i], holds[i] = S, H
    return y, hold, states, holds


def close(got, want, hold):
    """[..., channels], each token's head by what it holds. Below 2^-126 F32 has no normal numbers: 2^-126 off counts as none."""
    off, floor = np.abs(got.astype(np.float64) - want), 2.0 ** -126
    one = off / np.maximum(hold, floor / ONE)
    assert one.max() <= ONE, (one.max(), np.unravel_index(one.argmax(), one.shape))
    row = np.linalg.norm(off, axis=-1) / np.maximum(np.linalg.norm(hold, axis=-1), floor / REL)
    assert row.max() <= REL, (row.max(), np.unravel_index(row.argmax(), row.shape))


def check(torch, kh, vh, dim, segments, count, edit, lengths=None, seed=1):
    c = R.rule_case(np.random.default_rng(seed), kh, vh, dim, segments, segments, count)
    edit(c)
    c = {n: np.ascontiguousarray(a, np.float32) for n, a in c.items()}
    net = Net(torch, kh, vh, dim, segments, c)
    y = net.rule(list(range(segments)), segments, count, lengths)
    want, hold, states, holds = walk(c, kh, vh, dim, segments, count, lengths)
    rows = [r for i in range(segments) for r in range(i * count, i * count + (count if lengths is None else lengths[i]))]
    y = y.reshape(-1, vh, dim)
    assert np.isfinite(y).all() and int(net.status.item()) == 0
    close(y[rows], want[rows], hold[rows])
    close(net.state().transpose(0, 2, 1, 3), states, np.broadcast_to(holds[:, :, None], states.shape))


# (heads, dim, runs, count): a few chunks; a short last chunk; parts of runs; one chain for each multiprocessor and the next slab's first
# kernel beside it; more states than multiprocessors
FORMS = [(1, 2, 64, 1, 150), (2, 4, 128, 1, 67), (1, 2, 128, 1, 900), (16, 32, 64, 1, 1250), (4, 8, 64, 24, 90)]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("size", [1e5, 1e8, 1e12, 1e17])
@pytest.mark.parametrize("what", ["token", "channel", "last token"])
def test_a_large_token_takes_nothing_from_those_before(torch, form, size, what):
    kh, vh, dim, segments, count = form

    def edit(c):
        at = count - 1 if what == "last token" else min(40, count - 2)
        for i in range(segments):
            if what == "channel":
                c["v"][i * count + at, 5] *= size
            else:
                c["v"][i * count + at] *= size
    check(torch, kh, vh, dim, segments, count, edit)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("size", [1e8, 1e17])
@pytest.mark.parametrize("decay", [0.0, 1e-20])
def test_what_a_decay_takes_away_is_gone(torch, form, size, decay):
    """A large token, or a large state, and a little later a decay that ends it."""
    kh, vh, dim, segments, count = form

    def token(c):
        for i in range(segments):
            c["v"][i * count + 20] *= size
            c["decay"][i * count + 33] = decay

    def state(c):
        c["state"] *= size
        for i in range(segments):
            c["decay"][i * count + 33] = decay
    check(torch, kh, vh, dim, segments, count, token)
    check(torch, kh, vh, dim, segments, count, state)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("what", ["tokens", "elements", "growing", "shrinking", "one small", "small decays"])
def test_tokens_of_all_sizes(torch, form, what):
    kh, vh, dim, segments, count = form
    rng = np.random.default_rng(5)

    def edit(c):
        v = c["v"]
        t = np.tile(np.arange(count), segments)[:, None]
        if what == "tokens":
            v *= 10.0 ** rng.uniform(-12, 12, (len(v), 1))
        elif what == "elements":
            v *= 10.0 ** rng.uniform(-12, 12, v.shape)
        elif what == "growing":
            v *= 10.0 ** (t % 64 / 4 - 8)
        elif what == "shrinking":
            v *= 10.0 ** (8 - t % 64 / 4)
        elif what == "one small":
            v[t[:, 0] == 3] *= 1e-13
        else:
            v *= 10.0 ** rng.uniform(-9, 9, (len(v), 1))
            c["decay"][:] = 10.0 ** rng.uniform(-12, 0, c["decay"].shape)
    check(torch, kh, vh, dim, segments, count, edit, seed=2)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 24, 2.0 ** 40])
def test_strengths_and_keys_of_all_sizes(torch, form, size):
    """A token whose key is `size` times shorter, its strength size^2 larger: its difference is larger than all others'. One the other way."""
    kh, vh, dim, segments, count = form

    def edit(c):
        for i in range(segments):
            for at, by in ((30, 1 / size), (45, size)):
                c["k"][i * count + at] *= by
                c["beta"][i * count + at] /= by * by
                c["v"][i * count + at] *= by  # (as large as what the state says of that key)
    check(torch, kh, vh, dim, segments, count, edit)


@pytest.mark.parametrize("form", FORMS)
def test_runs_that_begin_from_nothing(torch, form):
    """No state, no first strength, tokens of zeros, and lengths that end inside a chunk."""
    kh, vh, dim, segments, count = form

    def edit(c):
        c["state"][:] = 0
        c["v"][::5] = 0
        c["beta"][::count] = 0
        for i in range(segments):
            c["v"][i * count + 1] *= 1e-14
    check(torch, kh, vh, dim, segments, count, edit, [count - i % 7 for i in range(segments)])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("growing", [36, 40, 60])
def test_growth_that_only_queries_see(torch, dim, growing):
    """Keys that do not meet, and a value of 2^-100 that decays of 8 bring back: what a token weighs it by, 8^40 and more times a query's
    and a key's factors, passes F32's range, the result does not."""
    kh, vh, count = 1, 2, 64

    def edit(c):
        c["state"][:] = 0
        c["decay"][:] = 1
        c["decay"][0] = 0
        c["decay"][1:growing] = 8
        c["k"][:] = np.eye(dim)[np.arange(count) % dim]
        c["q"][:] = c["k"][:1] / 8
        c["beta"][:] = 1
        c["v"] *= 2.0 ** -100
        c["v"][1:] = 0
    check(torch, kh, vh, dim, 1, count, edit)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("where", ["behind", "before", "between", "keys alone", "queries alone"])
def test_rows_of_zeros(torch, form, where):
    """Rows that fill up a batch without lengths: no key, query and value (or one of the first two), beside tokens that are large."""
    kh, vh, dim, segments, count = form
    t = np.tile(np.arange(count), segments)
    rows = {"behind": t >= count - count // 3, "before": t < count // 3, "between": (t % 7 == 3) | ((t > 20) & (t < 40))}.get(where, t % 5 == 2)

    def edit(c):
        c["v"][t == 50 % count] *= 1e10
        for n in {"keys alone": "k", "queries alone": "q"}.get(where, "qkv"):  # (each letter a name)
            c[n][rows] = 0
        if where == "keys alone":  # what such a token is given goes nowhere
            c["v"][rows] *= (10.0 ** np.random.default_rng(1).uniform(-12, 12, (rows.sum(), 1))).astype(np.float32)
    check(torch, kh, vh, dim, segments, count, edit)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("what", ["keys", "short keys", "short keys, large values"])
def test_keys_of_all_sizes(torch, form, what):
    """Every token's key of a size of its own: with a strength that goes with it (beta |k|^2 as before), or shorter alone."""
    kh, vh, dim, segments, count = form
    rng = np.random.default_rng(7)

    def edit(c):
        by = 10.0 ** rng.uniform(-6, 6 if what == "keys" else 0, (len(c["k"]), 1))
        c["k"] *= by
        if what == "keys":
            c["beta"] /= by * by
            c["v"] *= by
        elif what != "short keys":
            c["v"] /= by * by
    check(torch, kh, vh, dim, segments, count, edit)
