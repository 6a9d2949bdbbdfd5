"""The token mixers over runs of many sequences from their definitions, in 64 bits, and cases for their tests."""
import numpy as np


def runs(sequence, lengths, segments, count, sequences):
    """(run, sequence, tokens) of each run; sequence -1 where it is idle, outside, or an earlier run has it."""
    seen, out = set(), []
    for i in range(segments):
        s = -1 if sequence is None else int(sequence[i])
        s = 0 if sequence is None else s
        n = count if lengths is None else min(max(int(lengths[i]), 0), count)
        if sequence is not None and (s < 0 or s >= sequences or s in seen):
            s = -1
        seen.add(s)
        out.append((i, s, n))
    return out


def inputs(x, history, weight, kh, vh, dim, sequence, lengths, segments, count, outs, q_scale=None, eps=1e-6):
    """q, k, v, history after; `outs` are what q, k and v held before."""
    taps = weight.shape[1]
    q, k, v = (o.astype(np.float64).copy() for o in outs)
    history, x, w = history.astype(np.float64).copy(), x.astype(np.float64), weight.astype(np.float64)
    kd = kh * dim
    for i, s, n in runs(sequence, lengths, segments, count, history.shape[0]):
        rows = slice(i * count, (i + 1) * count)
        if s < 0:
            q[rows] = k[rows] = v[rows] = 0
            continue
        got = np.concatenate([history[s], x[i * count:i * count + n].T], 1)      # [channels, taps - 1 + n]
        c = sum(w[:, m:m + 1] * got[:, m:m + n] for m in range(taps)).T           # [n, channels]
        c = c / (1 + np.exp(-c))
        a, b = c[:, :kd].reshape(n, kh, dim), c[:, kd:2 * kd].reshape(n, kh, dim)
        scale = 1 / np.sqrt(dim) if q_scale is None else q_scale
        q[i * count:i * count + n] = (a / np.sqrt((a * a).sum(-1, keepdims=True) + eps) * scale).reshape(n, kd)
        k[i * count:i * count + n] = (b / np.sqrt((b * b).sum(-1, keepdims=True) + eps)).reshape(n, kd)
        v[i * count:i * count + n] = c[:, 2 * kd:]
        history[s] = got[:, n:]
    return q, k, v, history


def rule(q, k, v, decay, beta, state, kh, vh, dim, sequence, lengths, segments, count, y):
    """y and the states after; `state` [sequences][dim key][vh][dim value]."""
    q, k, v, decay, beta, state, y = (t.astype(np.float64) for t in (q, k, v, decay, beta, state, y))
    state, y = state.copy(), y.copy()
    of = np.arange(vh) % kh
    with np.errstate(all="ignore"):
        for i, s, n in runs(sequence, lengths, segments, count, state.shape[0]):
            if s < 0:
                y[i * count:(i + 1) * count] = 0
                continue
            S = state[s].transpose(1, 0, 2)                                          # [vh, key, value]
            for r in range(i * count, i * count + n):
                kr, qr = k[r].reshape(kh, dim)[of], q[r].reshape(kh, dim)[of]
                S = S * decay[r][:, None, None]
                d = beta[r][:, None] * (v[r].reshape(vh, dim) - np.einsum("hkv,hk->hv", S, kr))
                S = S + kr[:, :, None] * d[:, None]
                y[r] = np.einsum("hkv,hk->hv", S, qr).reshape(-1)
            state[s] = S.transpose(1, 0, 2)
    return y, state


def qk_rope(q, k, wq, wk, cos, sin, heads, kv, dim, rotary, sequence, start, lengths, segments, count, yq, yk, apart=None, eps=1e-6):
    apart, half = apart or dim, rotary // 2
    yq, yk = yq.astype(np.float64).copy(), yk.astype(np.float64).copy()
    for i in range(segments):
        n = count if lengths is None else int(lengths[i])
        for r in range(i * count, (i + 1) * count):
            if sequence is not None and sequence[i] < 0:
                yq[r] = yk[r] = 0
                continue
            if r - i * count >= n:
                continue
            p = int(start[i]) + r - i * count
            if not 0 <= p < cos.shape[0]:
                yq[r] = yk[r] = 0
                continue
            for x, w, y, h, step in ((q, wq, yq, heads, apart), (k, wk, yk, kv, dim)):
                for j in range(h):
                    a = x[r, j * step:j * step + dim].astype(np.float64)
                    a = a / np.sqrt((a * a).mean() + eps) * w.astype(np.float64)
                    lo, hi = a[:half].copy(), a[half:rotary].copy()
                    c, s = cos[p].astype(np.float64), sin[p].astype(np.float64)
                    a[:half], a[half:rotary] = lo * c - hi * s, hi * c + lo * s
                    y[r, j * dim:(j + 1) * dim] = a
    return yq, yk


def rule_case(rng, kh, vh, dim, sequences, segments, count, keys="mixed"):
    """Rows as they come from the inputs: normed keys with a common part, decays of short and of long memories."""
    rows = segments * count
    q, k = (t / (1 + np.exp(-t)) for t in rng.standard_normal((2, rows, kh, dim)))
    if keys == "same":  # one key for all tokens: the differences' system is as full as it gets
        k = np.broadcast_to(k[:1], k.shape)
    q = q / np.sqrt((q * q).sum(-1, keepdims=True) + 1e-6) / np.sqrt(dim)
    k = k / np.sqrt((k * k).sum(-1, keepdims=True) + 1e-6)
    rate = 0.005 * 400 ** rng.random(vh)
    decay = np.exp(-rate * np.log1p(np.exp(rng.standard_normal((rows, vh)))))
    beta = 1 / (1 + np.exp(-rng.standard_normal((rows, vh))))
    return {n: np.ascontiguousarray(a, np.float32) for n, a in dict(
        q=q.reshape(rows, -1), k=k.reshape(rows, -1), v=rng.standard_normal((rows, vh * dim)), decay=decay, beta=beta,
        state=0.2 * rng.standard_normal((sequences, dim, vh, dim))).items()}
