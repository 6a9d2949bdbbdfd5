"""The token mixers of the hybrid model over runs of many sequences: the plain forms of the operators, and the cases on which
the CUDA kernels are measured.

A call works on `segments` runs of `count` rows; run i belongs to sequence[i] (-1: an idle slot, whose rows become zero and
whose state stays). With `lengths`, run i has lengths[i] tokens and its rows behind them are left as they were.

inputs:  the delta-rule layer's inputs from its [q | k | v] projection x: a causal convolution of `taps` taps over each channel,
         which goes on from the sequence's last taps - 1 inputs (`history` [sequences][channels][taps - 1]), SiLU, and for each
         head of q and k the L2 norm: s / sqrt(sum s^2 + 1e-6), q's times 1 / sqrt(dim).
rule:    the gated delta rule, for each value head with a state S [dim][dim] of its sequence (`state` [sequences][dim][value
         heads][dim]); value head h reads key head h % key heads:
             S <- decay_t S;  d = beta_t (v_t - S^T k_t);  S <- S + k_t d^T;  y_t = S^T q_t
qk_rope: for each head of q and k the RMS norm times a weight of each channel, and the rotation of the first `rotary` channels
         (pairs are half of them apart) by row start[i] + j of the tables cos and sin [cells][rotary / 2]. Head rows of q may
         lie apart, as in a projection of [q | gate] for each head.
"""
import math
import random

import torch

own = False
CHUNK = 64
EPS = 1e-6
WORKSPACE = 128 << 20


# ---------------------------------------------------------------- cases

def _delta(name, op, kh, vh, dim, segments, count, ragged=False, taps=4):
    c = dict(op=op, kh=kh, vh=vh, dim=dim, segments=segments, count=count, ragged=ragged, taps=taps)
    if name:
        c["name"] = name
    return c


def _rope(name, heads, kv, dim, rotary, segments, count, cells, ragged=False, gated=True):
    c = dict(op="qk_rope", heads=heads, kv=kv, dim=dim, rotary=rotary, segments=segments, count=count, cells=cells, ragged=ragged, gated=gated)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # the token step of one session of the 48-layer model: latency
        _delta("rule, one token", "rule", 16, 32, 128, 1, 1),
        # the token step of a batch of 64 sessions, one slot idle: the states' bytes
        _delta("rule, 64 sessions", "rule", 16, 32, 128, 64, 1, ragged=True),
        # a few tokens of each of 16 sessions (drafted tokens that are checked, short turns), of their own number
        _delta("rule, up to 7 tokens of 16", "rule", 16, 32, 128, 16, 7, ragged=True),
        # a prompt of one session
        _delta("rule, prompt of 2048", "rule", 16, 32, 128, 1, 2048),
        # prompts of many sessions of a small model, of all lengths
        _delta("rule, 24 prompts up to 531", "rule", 4, 8, 64, 24, 531, ragged=True),
        # a long odd prompt in the full model's geometry
        _delta("rule, prompt of 8191", "rule", 16, 48, 128, 1, 8191),
        # the inputs of the same layers: the token step of one session
        _delta("inputs, one token", "inputs", 16, 32, 128, 1, 1),
        # of 64 sessions
        _delta("inputs, 64 sessions", "inputs", 16, 32, 128, 64, 1, ragged=True),
        # and of a long odd prompt
        _delta("inputs, prompt of 8191", "inputs", 16, 48, 128, 1, 8191),
        # queries and keys of a full-attention layer with gates beside the queries: the token step of one session
        _rope("qk_rope, one token", 16, 2, 256, 64, 1, 1, 2048),
        # of 64 sessions, one slot idle
        _rope("qk_rope, 64 sessions", 16, 2, 256, 64, 64, 1, 2048, ragged=True),
        # and of a long odd prompt
        _rope("qk_rope, prompt of 8191", 24, 2, 256, 64, 1, 8191, 16384),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["rule", "rule", "rule", "inputs", "qk_rope"])
    prompt = rng.random() < 0.6
    segments = 1 if prompt and rng.random() < 0.5 else _log(rng, 1, 24 if prompt else 96)
    ragged = segments > 1 and rng.random() < 0.8
    if op == "qk_rope":
        dim = rng.choice([32, 64, 80, 96, 128, 128, 256, 256])
        kv = rng.choice([1, 2, 3, 4, 8])
        heads = kv * rng.choice([1, 2, 3, 8, 12])
        while heads * dim > 6144:
            heads -= kv
        count = _log(rng, 2, 8191 // segments) if prompt else _log(rng, 1, 4)
        return _rope("", heads, kv, dim, rng.choice([dim, dim // 2, 16]), segments, count, count + _log(rng, 1, 8192), ragged=ragged, gated=rng.random() < 0.6)
    dim = rng.choice([16, 32, 40, 64, 64, 80, 96, 128, 128, 128, 128, 192, 256])
    kh = rng.choice([1, 2, 4, 6, 8, 16])
    vh = kh * rng.choice([1, 2, 2, 3, 4])
    while (2 * kh + vh) * dim > 10240 or vh * dim > 6144:
        kh, vh = (kh, vh - kh) if vh > kh else (kh // 2, kh // 2)
    most = max(2, 8191 // segments) if dim <= 128 else max(2, 512 // segments)
    count = _log(rng, 2, most) if prompt else _log(rng, 1, 8)
    return _delta("", op, kh, vh, dim, segments, count, ragged=ragged, taps=rng.choice([4, 4, 4, 2, 3]) if op == "inputs" else 4)


def _lengths(case):
    """Tokens of each run, one of many without any; -1 for an idle slot."""
    s, n = case["segments"], case["count"]
    if not case["ragged"]:
        return [n] * s
    got = [1 + int(n * ((0.37 + 0.6180339887 * i) % 1.0)) for i in range(s)]
    got[s // 2] = n
    if s >= 8:
        got[s // 3] = -1
        got[s // 4] = 0
    return got


# ---------------------------------------------------------------- the operators, plainly

def _valid(st):
    """Rows that hold a token, rows of idle slots: [segments, count]"""
    c = st["case"]
    j = torch.arange(c["count"], device="cuda")[None]
    live = st["sequence"][:, None] >= 0
    there = live if st["lengths"] is None else live & (j < st["lengths"][:, None])
    return there.expand(c["segments"], c["count"]), ~live.expand(c["segments"], c["count"])


def _put(old, rows, there, idle):
    """Rows with a token, zeros for idle slots, what was there before elsewhere."""
    shape = (-1,) + (1,) * (old.dim() - 1)
    zero = torch.zeros((), device=old.device)
    old.copy_(torch.where(there.reshape(shape), rows, torch.where(idle.reshape(shape), zero, old)))
    return old


def _inputs(st):
    c = st["case"]
    S, n, taps, dim = c["segments"], c["count"], c["taps"], c["dim"]
    kd, vd = c["kh"] * dim, c["vh"] * dim
    there, idle = _valid(st)
    seq = st["sequence"].clamp(min=0).long()
    rows = torch.cat([st["history"][seq].transpose(1, 2), st["x"].reshape(S, n, -1)], 1)      # [S, taps - 1 + n, channels]
    s = (rows.unfold(1, taps, 1) * st["w"]).sum(-1)
    s = s / (1 + torch.exp(-s))
    q, k, v = s.reshape(S * n, -1).split([kd, kd, vd], -1)
    q, k = (t.reshape(S * n, c["kh"], dim) for t in (q, k))
    q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + EPS) * (1 / math.sqrt(dim))
    k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + EPS)
    last = there.sum(1)[:, None] + torch.arange(taps - 1, device="cuda")                      # the last taps - 1 rows of each run
    new = rows[torch.arange(S, device="cuda")[:, None], last].transpose(1, 2)
    live = st["sequence"] >= 0
    st["history"][seq[live]] = new[live]
    return [_put(st[o], t.reshape(S * n, -1), there, idle) for o, t in (("q", q), ("k", k), ("v", v))] + [st["history"]]


def _triangular_inverse(a):
    """(I + a)^-1 of strictly lower triangular matrices [.., n, n], n a power of two: from the inverses of diagonal blocks to
    those of blocks twice as large."""
    n = a.shape[-1]
    i = torch.arange(n, device=a.device)
    t = torch.eye(n, device=a.device).expand(a.shape)
    size = 1
    while size < n:
        below = (i[:, None] // (2 * size) == i // (2 * size)) & (i[:, None] // size > i // size)
        t = t - t @ torch.where(below, a, torch.zeros((), device=a.device)) @ t
        size *= 2
    return t


def _rule(st):
    """In chunks: a chunk's differences from the state before it by one triangular system, the state from chunk to chunk."""
    c = st["case"]
    S, n, kh, vh, dim = c["segments"], c["count"], c["kh"], c["vh"], c["dim"]
    there, idle = _valid(st)
    C = min(CHUNK, 1 << (n - 1).bit_length())
    N = (n + C - 1) // C
    zero, one = torch.zeros((), device="cuda"), torch.ones((), device="cuda")

    def chunks(x, heads, width, fill=zero):
        x = torch.where(there[..., None, None], x.reshape(S, n, heads, width), fill)
        x = torch.cat([x, fill.expand(S, N * C - n, heads, width)], 1)
        x = x.reshape(S, N, C, heads, width).permute(1, 0, 3, 2, 4)                            # [N, S, heads, C, width]
        return x.repeat(1, 1, vh // heads, 1, 1) if heads < vh else x

    q, k, v = chunks(st["q"], kh, dim), chunks(st["k"], kh, dim), chunks(st["v"], vh, dim)
    beta, a = chunks(st["beta"], vh, 1), chunks(st["decay"], vh, 1, one)
    g = torch.log(a.double()).clamp(min=-1000.0).cumsum(-2)                                    # [N, S, vh, C, 1]
    i = torch.arange(C, device="cuda")
    upto = i[:, None] >= i
    gamma = torch.exp(torch.where(upto, g - g.transpose(-1, -2), zero.double())).float()
    kk = k @ k.transpose(-1, -2)
    t = _triangular_inverse(torch.where(i[:, None] > i, beta * gamma * kk, zero))
    first = torch.exp(g).float()                                                               # decay from the chunk's beginning
    u, w = t @ (beta * v), t @ (beta * first * k)
    attn = torch.where(upto, gamma * (q @ k.transpose(-1, -2)), zero)
    to_end = (torch.exp(g[..., -1:, :] - g).float() * k).transpose(-1, -2)
    q = q * first
    end = first[..., -1:, :]
    seq = st["sequence"].clamp(min=0).long()
    state = st["state"][seq].transpose(1, 2)                                                   # [S, vh, dim, dim]
    y = torch.empty(N, S, vh, C, dim, device="cuda")
    for m in range(N):
        d = u[m] - w[m] @ state
        y[m] = q[m] @ state + attn[m] @ d
        state = end[m] * state + to_end[m] @ d
    live = st["sequence"] >= 0
    st["state"][seq[live]] = state.transpose(1, 2)[live]
    y = y.permute(1, 0, 3, 2, 4).reshape(S, N * C, vh * dim)[:, :n].reshape(S * n, vh * dim)
    return _put(st["y"], y, there, idle), st["state"]


def _q_heads(st):
    """q's head rows, which may lie among gates: [segments * count, heads, dim]"""
    c = st["case"]
    return st["q"].reshape(-1, c["heads"], c["dim"] * (2 if c["gated"] else 1))[..., : c["dim"]]


def _qk_rope(st):
    c = st["case"]
    S, n, dim, half = c["segments"], c["count"], c["dim"], c["rotary"] // 2
    there, idle = _valid(st)
    at = (st["start"].long()[:, None] + torch.arange(n, device="cuda")).clamp(0, c["cells"] - 1).reshape(-1)
    cos, sin = st["cos"][at][:, None], st["sin"][at][:, None]

    def one(x, w):
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1).reshape(S * n, -1)

    return _put(st["yq"], one(_q_heads(st), st["wq"]), there, idle), _put(st["yk"], one(st["k"].reshape(S * n, c["kv"], dim), st["wk"]), there, idle)


# ---------------------------------------------------------------- the framework's calls

def _handle(st):
    """The object that a program holds for as long as it has the state or the weights."""
    from stratacuda_b200.mixers import DeviceDeltaNet, DeviceQkRope

    c = st["case"]
    if c["op"] == "qk_rope":
        st["handle"] = DeviceQkRope(heads=c["heads"], kv_heads=c["kv"], dim=c["dim"], rotary=c["rotary"], cells=c["cells"], q_weight=st["wq"],
                                    k_weight=st["wk"], cos=st["cos"], sin=st["sin"])
    else:
        st["handle"] = DeviceDeltaNet(key_heads=c["kh"], value_heads=c["vh"], dim=c["dim"], sequences=c["segments"], taps=c["taps"],
                                      state=st.get("state"), history=st.get("history"), weight=st.get("w"), workspace=st.get("workspace"))
    return st["handle"]


def _run_own(st):
    c, h = st["case"], st.get("handle") or _handle(st)
    runs = dict(sequence=st["sequence"], segments=c["segments"], count=c["count"], lengths=st["lengths"], stream=torch.cuda.current_stream().cuda_stream)
    if c["op"] == "inputs":
        h.inputs(st["x"], st["q"], st["k"], st["v"], **runs)
        return [st["q"], st["k"], st["v"], st["history"]]
    if c["op"] == "rule":
        h.rule(st["q"], st["k"], st["v"], st["decay"], st["beta"], st["y"], **runs)
        return st["y"], st["state"]
    h.apply(st["q"], st["k"], st["yq"], st["yk"], start=st["start"], q_head_stride=c["dim"] * (2 if c["gated"] else 1), **runs)
    return st["yq"], st["yk"]


# ---------------------------------------------------------------- what the measurement asks for

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    S, n, dim, op = case["segments"], case["count"], case["dim"], case["op"]
    T = S * n
    lens = _lengths(case)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    st = dict(case=dict(case))
    order = torch.randperm(S, generator=g, device="cuda").tolist()
    st["sequence"] = torch.tensor([s if L >= 0 else -1 for s, L in zip(order, lens)], dtype=torch.int32, device="cuda")
    st["lengths"] = torch.tensor([max(L, 0) for L in lens], dtype=torch.int32, device="cuda") if case["ragged"] else None
    if op == "qk_rope":
        cells, half = case["cells"], case["rotary"] // 2
        st["start"] = (torch.rand(S, generator=g, device="cuda") * (cells - n + 1)).to(torch.int32).clamp(0, cells - n)
        angle = torch.arange(cells, device="cuda", dtype=torch.float64)[:, None] * 1e7 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        st["cos"], st["sin"] = torch.cos(angle).float(), torch.sin(angle).float()
        st["wq"], st["wk"] = 1 + 0.05 * normal(dim), 1 + 0.05 * normal(dim)
        st["q"] = normal(T, case["heads"] * dim * (2 if case["gated"] else 1))
        st["k"] = normal(T, case["kv"] * dim)
        st["yq"], st["yk"] = torch.zeros(T, case["heads"] * dim, device="cuda"), torch.zeros(T, case["kv"] * dim, device="cuda")
        return st
    kh, vh, taps = case["kh"], case["vh"], case["taps"]
    kd, vd = kh * dim, vh * dim
    if op == "inputs":
        st["x"], st["w"] = normal(T, 2 * kd + vd), normal(2 * kd + vd, taps) / math.sqrt(taps)
        st["history"] = normal(S, 2 * kd + vd, taps - 1)
        st["q"], st["k"], st["v"] = (torch.zeros(T, d, device="cuda") for d in (kd, kd, vd))
        return st
    # what the inputs look like after the convolution's SiLU and the norms: keys have a common part
    q, k, v = (t / (1 + torch.exp(-t)) for t in (normal(T, kh, dim), normal(T, kh, dim), normal(T, vd)))
    st["q"] = (q / torch.sqrt((q * q).sum(-1, keepdim=True) + EPS) / math.sqrt(dim)).reshape(T, kd)
    st["k"] = (k / torch.sqrt((k * k).sum(-1, keepdim=True) + EPS)).reshape(T, kd)
    st["v"] = v
    # heads that remember for a few tokens and for hundreds
    rate = torch.exp(torch.rand(vh, generator=g, device="cuda") * math.log(400.0)) * 0.005
    st["decay"] = torch.exp(-rate * torch.log(1 + torch.exp(normal(T, vh))))
    st["beta"] = 1 / (1 + torch.exp(-normal(T, vh)))
    st["state"] = 0.2 * normal(S, dim, vh, dim)
    st["y"] = torch.zeros(T, vd, device="cuda")
    st["workspace"] = torch.zeros(WORKSPACE, dtype=torch.uint8, device="cuda")
    return st


def run(state):
    if own:
        return _run_own(state)
    return {"inputs": _inputs, "rule": _rule, "qk_rope": _qk_rope}[state["case"]["op"]](state)


def work(case):
    live = [L for L in _lengths(case) if L > 0]
    tokens, dim = sum(live), case["dim"]
    if case["op"] == "qk_rope":
        width = (case["heads"] + case["kv"]) * dim
        return dict(bytes=tokens * width * 8 + tokens * case["rotary"] * 4 + 8 * dim, flops=tokens * width * 7)
    kd, vd = case["kh"] * dim, case["vh"] * dim
    if case["op"] == "inputs":
        channels = 2 * kd + vd
        return dict(bytes=tokens * channels * 8 + channels * 4 * case["taps"] + len(live) * channels * (case["taps"] - 1) * 8,
                    flops=tokens * channels * (2 * case["taps"] + 6))
    # three products of a token with the state of each value head: prediction, update, result
    return dict(bytes=tokens * (2 * kd + 2 * vd + 2 * case["vh"]) * 4 + len(live) * vd * dim * 8, flops=6 * tokens * vd * dim)


def exact(case, seed):
    """Token by token, from the definitions, in 64 bits."""
    st = prepare(case, seed)
    S, n, dim = case["segments"], case["count"], case["dim"]
    lens, seqs = _lengths(case), st["sequence"].tolist()
    if case["op"] == "qk_rope":
        out = []
        half = case["rotary"] // 2
        for x, w, heads, put in ((_q_heads(st), st["wq"], case["heads"], st["yq"]), (st["k"], st["wk"], case["kv"], st["yk"])):
            y = put.double()
            x = x.double().reshape(S, n, heads, dim)
            for i, L in enumerate(lens):
                if L > 0:
                    r = x[i, :L] * torch.rsqrt(x[i, :L].pow(2).mean(-1, keepdim=True) + EPS) * w.double()
                    p = int(st["start"][i])
                    z = torch.complex(st["cos"][p:p + L].double(), st["sin"][p:p + L].double())
                    turned = torch.complex(r[..., :half], r[..., half:2 * half]) * z[:, None]
                    r[..., :half], r[..., half:2 * half] = turned.real, turned.imag
                    y[i * n:i * n + L] = r.reshape(L, -1)
            out.append(y)
        return out[0], out[1]
    kh, vh = case["kh"], case["vh"]
    if case["op"] == "inputs":
        out = [st[o].double() for o in "qkv"]
        history, w, taps = st["history"].double(), st["w"].double(), case["taps"]
        for i, L in enumerate(lens):
            if L <= 0:
                continue
            x = torch.cat([history[seqs[i]], st["x"][i * n:i * n + L].double().T], 1)          # [channels, taps - 1 + L]
            s = torch.nn.functional.conv1d(x[None], w[:, None], groups=x.shape[0])[0].T
            s = s * torch.sigmoid(s)
            history[seqs[i]] = x[:, L:]
            for o, part, scale in zip(out, s.split([kh * dim, kh * dim, vh * dim], 1), (dim ** -0.5, 1.0, None)):
                if scale is not None:
                    heads = part.reshape(L, kh, dim)
                    part = (heads * (scale * torch.rsqrt(heads.square().sum(-1, keepdim=True) + EPS))).reshape(L, -1)
                o[i * n:i * n + L] = part
        return out + [history]
    state, y = st["state"].double(), st["y"].double()
    of = torch.arange(vh, device="cuda") % kh
    at = torch.tensor([i for i in range(S) if seqs[i] >= 0], device="cuda")
    where = torch.tensor([seqs[i] for i in at.tolist()], device="cuda")
    M = state[where].permute(0, 2, 3, 1).contiguous()                                          # [runs, vh, value, key]
    q, k = (st[x].double().reshape(S, n, kh, dim)[at][:, :, of] for x in "qk")
    v = st["v"].double().reshape(S, n, vh, dim)[at]
    a, b = (st[x].double().reshape(S, n, vh, 1)[at] for x in ("decay", "beta"))
    long = torch.tensor([max(L, 0) for L in lens], device="cuda")[at]
    ys = y.reshape(S, n, vh, dim)
    for t in range(n):
        on = (t < long)[:, None, None]
        N = M * a[:, t, ..., None]
        d = (v[:, t] - torch.einsum("shvk,shk->shv", N, k[:, t])) * b[:, t]
        N = N + d[..., None] * k[:, t, :, None]
        ys[at, t] = torch.where(on, torch.einsum("shvk,shk->shv", N, q[:, t]), ys[at, t])
        M = torch.where(on[..., None], N, M)
    state[where] = M.permute(0, 3, 1, 2)
    return y, state
