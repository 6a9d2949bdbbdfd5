"""Attention over a paged key/value cache held in 8 bits, and the sparse selection that goes with it:
the plain forms of the operators, and the cases on which the CUDA kernels are measured.

The cache. A page holds 64 consecutive tokens (a block) of one sequence for every key/value head. Keys
and values are signed 8-bit codes with one float scale for each page, head and kind; `marks` holds the
lowest and the highest key code of every channel of a block; `open` holds the rows of each sequence's
last block in 32 bits, from which the block's codes are formed again when its scale has to grow.

    codes  int8 [pages][kv heads][2][P * 64]   keys as [P / 64][64 tokens][64 channels], values as
                                               [P channels][64 tokens]; P = dim padded to 64, 128 or 256
    marks  int8 [pages][kv heads][2][P]        lowest, highest key code of the block's tokens
    scales f32  [pages][kv heads][2]           key scale, value scale
    open   f32  [sequences][2][64][kv heads][dim]
    table  i32  [sequences][blocks]            page of each block

The operators. A call works on `segments` runs of `count` tokens; run i belongs to sequence[i] (-1: an
idle slot, whose output is zero) and its first token stands at position start[i].

append:  with amax the largest magnitude of a block's rows so far, scale = amax / 127 and
         code = round(x * (1 / scale)); a block whose amax is below 2^-100 has scale 0 and codes 0.
select:  for each token and key/value head the `top` blocks with the largest bound on the group's
         summed logits, sum_d p_d hi_d + n_d lo_d, where p and n are the positive and negative parts of the
         group's queries added up in fixed point and rounded to 8 bits. The first and the last blocks are
         always among them. Block indices ascend, -1 fills up; ties go to the lower block.
attend:  softmax(q k / sqrt(dim)) v over the tokens at or before the query's own position, of all blocks
         or of the blocks that `picks` lists.
"""
import math
import random

import torch

own = False
BLOCK = 64
TINY = 2.0 ** -100


def _padded(dim):
    return 64 if dim <= 64 else 128 if dim <= 128 else 256


# ---------------------------------------------------------------- cases

def _case(name, op, heads, kv, dim, segments, count, longest, top=0, ragged=False):
    c = dict(op=op, heads=heads, kv=kv, dim=dim, segments=segments, count=count, longest=longest, top=top, ragged=ragged)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one new token of one session, in the hybrid model's attention geometry (24 heads on 2 of 256)
        _case("append one token", "append", 24, 2, 256, 1, 1, 1501),
        # the new tokens of a batch of 64 sessions at positions of their own
        _case("append 64 sessions", "append", 24, 2, 256, 64, 1, 4096, ragged=True),
        # a prompt that continues a session in the middle of a block
        _case("append prompt of 8191", "append", 24, 2, 256, 1, 8191, 8191 + 77),
        # the token step of one session at the model's 2048 cells: latency
        _case("decode at 2048", "attend", 24, 2, 256, 1, 1, 2048),
        # the token step of 64 sessions of all lengths, one slot idle: the cache's bytes
        _case("decode 64 ragged", "attend", 24, 2, 256, 64, 1, 16384, ragged=True),
        # one very long session on another common geometry: few rows over a long axis
        _case("decode at 200001", "attend", 32, 8, 128, 1, 1, 200001),
        # a short odd prompt piece of a small model with a key/value head for each query head
        _case("prompt of 300", "attend", 16, 16, 64, 1, 300, 1801),
        # a prompt chunk late in a long session
        _case("prompt of 2048 at 14336", "attend", 24, 2, 256, 1, 2048, 16384),
        # choosing 32 of about 1000 blocks for the token step of 16 sessions
        _case("select for 16 sessions", "select", 24, 2, 256, 16, 1, 65536, top=32, ragged=True),
        # the same for each token of a prompt chunk
        _case("select for prompt of 2048", "select", 24, 2, 256, 1, 2048, 65536, top=32),
        # attention over the chosen blocks: the token step
        _case("sparse decode of 16", "sparse", 24, 2, 256, 16, 1, 65536, top=32, ragged=True),
        # and a prompt chunk
        _case("sparse prompt of 1024", "sparse", 24, 2, 256, 1, 1024, 65536, top=32),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["append", "attend", "attend", "select", "sparse"])
    dim = rng.choice([16, 40, 64, 72, 80, 96, 128, 128, 160, 192, 256, 256])
    kv = rng.choice([1, 2, 3, 4, 8])
    heads = kv * rng.choice([1, 2, 4, 5, 8, 12, 16])
    prompt = rng.random() < 0.5
    segments = 1 if prompt and rng.random() < 0.6 else _log(rng, 1, 8 if prompt else 96)
    ragged = segments > 1 and rng.random() < 0.8
    if op == "append":
        count = _log(rng, 2, 8192 // segments) if prompt else 1
        return _case("", op, heads, kv, dim, segments, count, count + _log(rng, 1, 4096), ragged=ragged)
    if op == "attend":
        count = _log(rng, 2, 2048 // segments) if prompt else 1
        longest = max(count, _log(rng, 1, 16384 if segments > 4 or prompt else 131072))
        while longest * heads * dim * segments * count > 2048 * 16384 * 24 * 256 or longest * segments * kv * dim > 64 * 16384 * 512:
            longest, count = max(1, longest // 2), max(1, count // 2)
        return _case("", op, heads, kv, dim, segments, count, max(longest, count), ragged=ragged)
    top = _log(rng, 4, 64)
    most = 2048 if op == "select" else 1024
    count = _log(rng, 2, most // segments) if prompt else 1
    longest = max(count, _log(rng, 64, 65536 if segments <= 16 else 16384))
    while op == "sparse" and count * segments * kv * dim * top > 1024 * 2 * 256 * 32:
        count, top = max(1, count // 2), max(4, top // 2)
    while longest * segments * kv * dim > 64 * 16384 * 512:
        longest = max(count, longest // 2)
    return _case("", op, heads, kv, dim, segments, count, longest, top=top, ragged=ragged)


def _lengths(case):
    """Tokens each run's sequence holds once its `count` tokens are in; -1 for an idle slot."""
    s, n, c = case["segments"], case["longest"], case["count"]
    if not case["ragged"]:
        return [n] * s
    got = [c + int((n - c) * ((0.37 + 0.6180339887 * i) % 1.0)) for i in range(s)]
    got[s // 2] = n
    if s >= 8:
        got[s // 3] = -1
    return got


def _blocks(case):
    return (case["longest"] + BLOCK - 1) // BLOCK


# ---------------------------------------------------------------- the cache, plainly

def _pack_keys(codes, padded):
    """[..., 64 tokens, dim] -> [..., padded * 64]"""
    lead = codes.shape[:-2]
    full = torch.zeros(*lead, BLOCK, padded, dtype=torch.int8, device=codes.device)
    full[..., : codes.shape[-1]] = codes
    return full.reshape(*lead, BLOCK, padded // 64, 64).transpose(-3, -2).reshape(*lead, padded * 64)


def _pack_values(codes, padded):
    lead = codes.shape[:-2]
    full = torch.zeros(*lead, padded, BLOCK, dtype=torch.int8, device=codes.device)
    full[..., : codes.shape[-1], :] = codes.transpose(-1, -2)
    return full.reshape(*lead, padded * 64)


def _keys(codes, dim):
    """[..., padded * 64] -> [..., 64 tokens, dim]"""
    lead, padded = codes.shape[:-1], codes.shape[-1] // 64
    return codes.reshape(*lead, padded // 64, BLOCK, 64).transpose(-3, -2).reshape(*lead, BLOCK, padded)[..., :dim]


def _vals(codes, dim):
    lead, padded = codes.shape[:-1], codes.shape[-1] // 64
    return codes.reshape(*lead, padded, BLOCK)[..., :dim, :].transpose(-1, -2)


def _scale_of(amax):
    return torch.where(amax < TINY, torch.zeros_like(amax), amax / torch.full_like(amax, 127.0))


def _codes_of(x, scale):
    """x [..., 64, dim], scale [...]: round(x / scale), as a product with the scale's reciprocal"""
    inv = torch.where(scale > 0, torch.ones_like(scale) / scale, torch.zeros_like(scale))
    return torch.round(x * inv[..., None, None]).clamp(-127, 127).to(torch.int8)


def _append(st, k, v):
    """k, v [segments, count, kv, dim]; st's codes, marks, scales and open rows change in place."""
    c = st["case"]
    kv, dim, S, n = c["kv"], c["dim"], c["segments"], c["count"]
    dev, padded = k.device, _padded(dim)
    live = st["sequence"] >= 0
    seq, start = st["sequence"].clamp(min=0).long(), st["start"].long()
    first, end = start // BLOCK, start + n
    nb = (n + BLOCK - 2) // BLOCK + 1
    block = first[:, None] + torch.arange(nb, device=dev)                          # [S, nb]
    at = block[:, :, None] * BLOCK + torch.arange(BLOCK, device=dev)               # [S, nb, 64] positions
    used = live[:, None] & (block * BLOCK < end[:, None])
    new = (at >= start[:, None, None]) & (at < end[:, None, None]) & used[:, :, None]
    old = (at < start[:, None, None]) & used[:, :, None]
    src = (at - start[:, None, None]).clamp(0, n - 1)
    x = torch.stack([k, v], 1)                                                     # [S, 2, n, kv, dim]
    i = torch.arange(S, device=dev)[:, None, None]
    rows = x.permute(0, 2, 1, 3, 4)[i, src]                                        # [S, nb, 64, 2, kv, dim]
    before = st["open"][seq].permute(0, 2, 1, 3, 4)[:, None]                       # [S, 1, 64, 2, kv, dim]
    zero = torch.zeros((), device=dev)
    rows = torch.where(new[..., None, None, None], rows, torch.where(old[..., None, None, None], before, zero))
    rows = torch.where(torch.isfinite(rows), rows, zero)
    rows = rows.permute(0, 1, 4, 3, 2, 5)                                          # [S, nb, kv, 2, 64, dim]
    page = st["table"][seq[:, None], block.clamp(max=st["table"].shape[1] - 1)].long()
    scale = _scale_of(rows.abs().amax((-1, -2)))                                   # [S, nb, kv, 2]
    codes = _codes_of(rows, scale)
    there = (new | old)[:, :, None, :, None]
    kc = codes[:, :, :, 0].float()
    lo = torch.where(there, kc, torch.full_like(kc, 127.0)).amin(-2).to(torch.int8)
    hi = torch.where(there, kc, torch.full_like(kc, -127.0)).amax(-2).to(torch.int8)
    w = used.nonzero(as_tuple=True)
    st["codes"][page[w]] = torch.stack([_pack_keys(codes[:, :, :, 0], padded), _pack_values(codes[:, :, :, 1], padded)], 3)[w]
    st["scales"][page[w]] = scale[w]
    marks = torch.zeros(S, nb, kv, 2, padded, dtype=torch.int8, device=dev)
    marks[..., 0, :dim], marks[..., 1, :dim] = lo, hi
    st["marks"][page[w]] = marks[w]
    # the last block's rows stay in 32 bits; a block that is full has none to keep
    last = (end - 1) // BLOCK
    j = (last - first)
    tail = x.permute(0, 2, 1, 3, 4)[i, src][torch.arange(S, device=dev), j]        # [S, 64, 2, kv, dim]
    keep = new[torch.arange(S, device=dev), j] & (end % BLOCK != 0)[:, None]       # [S, 64]
    s2, r2 = keep.nonzero(as_tuple=True)
    st["open"].permute(0, 2, 1, 3, 4)[seq[s2], r2] = torch.where(torch.isfinite(tail), tail, zero)[s2, r2]
    return st["codes"], st["marks"], st["scales"], st["open"]


def _visible(st):
    """Keys each token sees: [segments, count]"""
    c = st["case"]
    v = st["start"].long()[:, None] + torch.arange(c["count"], device=st["start"].device) + 1
    return torch.where(st["sequence"][:, None] >= 0, v, torch.zeros_like(v)).clamp(min=0)


def _softmax_v(logits, seen, v):
    logits = logits.masked_fill(~seen, -math.inf)
    m = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(torch.isfinite(m), m, torch.zeros_like(m)))
    s = p.sum(-1, keepdim=True)
    return torch.where(s > 0, torch.matmul(p, v) / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros((), device=v.device))


def _attend(st):
    c = st["case"]
    S, n, H, kv, dim = c["segments"], c["count"], c["heads"], c["kv"], c["dim"]
    G, nb = H // kv, _blocks(c)
    page = st["table"][st["sequence"].clamp(min=0).long(), :nb].long()             # [S, nb]
    codes, scale = st["codes"][page], st["scales"][page]                           # [S, nb, kv, 2, ..]
    k = (_keys(codes[..., 0, :], dim).float() * scale[..., 0, None, None]).transpose(1, 2).reshape(S, kv, nb * BLOCK, dim)
    v = (_vals(codes[..., 1, :], dim).float() * scale[..., 1, None, None]).transpose(1, 2).reshape(S, kv, nb * BLOCK, dim)
    q = st["q"].reshape(S, n, kv, G, dim).permute(0, 2, 1, 3, 4).reshape(S, kv, n * G, dim)
    logits = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(dim))
    seen = torch.arange(nb * BLOCK, device=q.device) < _visible(st)[:, :, None]    # [S, n, L]
    seen = seen[:, None, :, None].expand(S, kv, n, G, nb * BLOCK).reshape(S, kv, n * G, nb * BLOCK)
    y = _softmax_v(logits, seen, v)
    return y.reshape(S, kv, n, G, dim).permute(0, 2, 1, 3, 4).reshape(S * n, H * dim)


def _sparse(st):
    c = st["case"]
    S, n, H, kv, dim, top = c["segments"], c["count"], c["heads"], c["kv"], c["dim"], c["top"]
    G, N = H // kv, S * n
    picks = st["picks"].long().reshape(S, n, kv, top)
    page = st["table"][st["sequence"].clamp(min=0).long()[:, None, None, None], picks.clamp(min=0)].long().reshape(N, kv, top)
    head = torch.arange(kv, device=page.device)[:, None]
    codes, scale = st["codes"][page, head], st["scales"][page, head]               # [N, kv, top, 2, ..]
    k = (_keys(codes[..., 0, :], dim).float() * scale[..., 0, None, None]).reshape(N, kv, top * BLOCK, dim)
    v = (_vals(codes[..., 1, :], dim).float() * scale[..., 1, None, None]).reshape(N, kv, top * BLOCK, dim)
    logits = torch.matmul(st["q"].reshape(N, kv, G, dim), k.transpose(-1, -2)) * (1.0 / math.sqrt(dim))
    at = picks.reshape(N, kv, top, 1) * BLOCK + torch.arange(BLOCK, device=page.device)
    seen = (picks.reshape(N, kv, top, 1) >= 0) & (at < _visible(st).reshape(N, 1, 1, 1))
    y = _softmax_v(logits, seen.reshape(N, kv, 1, top * BLOCK), v)
    return y.reshape(N, H * dim)


def _select(st):
    c = st["case"]
    S, n, H, kv, dim, top = c["segments"], c["count"], c["heads"], c["kv"], c["dim"], c["top"]
    G, nb, padded = H // kv, _blocks(c), _padded(dim)
    zero = torch.zeros((), device=st["q"].device)
    q = st["q"].reshape(S, n, kv, G, dim)
    q = torch.where(torch.isfinite(q), q, zero)
    amax = q.abs().amax((-1, -2))                                                  # [S, n, kv]
    unit = torch.where(amax < TINY, zero, torch.full_like(amax, 32767.0) / amax)
    r = torch.round(q * unit[..., None, None])
    pos, neg = r.clamp(min=0).sum(-2), r.clamp(max=0).sum(-2)                      # whole numbers, exact in 32 bits
    big = torch.maximum(pos.amax(-1), (-neg).amax(-1))
    unit = torch.where(big > 0, torch.full_like(big, 127.0) / big, zero)[..., None]
    p, m = torch.round(pos * unit), torch.round(neg * unit)                        # [S, n, kv, dim]
    page = st["table"][st["sequence"].clamp(min=0).long(), :nb].long()             # [S, nb]
    marks = st["marks"][page][..., :dim].float()                                   # [S, nb, kv, 2, dim]
    bound = torch.einsum("snkd,sbkd->snkb", p, marks[..., 1, :]) + torch.einsum("snkd,sbkd->snkb", m, marks[..., 0, :])
    score = bound * st["scales"][page][..., 0].transpose(1, 2)[:, None]            # whole number times key scale
    have = (_visible(st) + BLOCK - 1) // BLOCK                                     # [S, n] blocks in sight
    b = torch.arange(nb, device=q.device)
    inside = b < have[..., None]
    forced = inside & ((b < c.get("first", 1)) | (b >= have[..., None] - c.get("last", 2)))
    score = score.masked_fill(forced[:, :, None], math.inf).masked_fill(~inside[:, :, None], -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :top]
    if order.shape[-1] < top:
        order = torch.nn.functional.pad(order, (0, top - order.shape[-1]), value=nb)
    order = torch.where(order < have[:, :, None, None], order, torch.full_like(order, 1 << 30)).sort(-1).values
    return torch.where(order < (1 << 30), order, torch.full_like(order, -1)).to(torch.int32).reshape(S * n, kv, top)


# ---------------------------------------------------------------- the framework's calls

def _handle(st):
    """The cache object that a program holds for as long as it has the cache."""
    from stratacuda_b200.kv8 import DeviceCache

    c = st["case"]
    st["cache"] = DeviceCache(kv_heads=c["kv"], dim=c["dim"], pages=st["codes"].shape[0], sequences=st["table"].shape[0],
                              blocks=st["table"].shape[1], codes=st["codes"], marks=st["marks"], scales=st["scales"], open=st["open"],
                              table=st["table"], workspace=st["workspace"])
    return st["cache"]


def _run_own(st):
    c, cache = st["case"], st.get("cache") or _handle(st)
    stream = torch.cuda.current_stream().cuda_stream
    runs = dict(sequence=st["sequence"], start=st["start"], segments=c["segments"], count=c["count"], stream=stream)
    N = c["segments"] * c["count"]
    if c["op"] == "append":
        cache.append(st["k"], st["v"], **runs)
        return st["codes"], st["marks"], st["scales"], st["open"]
    if c["op"] == "select":
        picks = torch.empty(N, c["kv"], c["top"], dtype=torch.int32, device="cuda")
        cache.select(st["q"], c["heads"], picks, top=c["top"], first=1, last=2, **runs)
        return picks
    y = torch.empty(N, c["heads"] * c["dim"], device="cuda")
    if c["op"] == "sparse":
        cache.attend(st["q"], c["heads"], y, picks=st["picks"], top=c["top"], **runs)
    else:
        cache.attend(st["q"], c["heads"], y, **runs)
    return y


# ---------------------------------------------------------------- what the measurement asks for

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    S, n, H, kv, dim = case["segments"], case["count"], case["heads"], case["kv"], case["dim"]
    padded, nb = _padded(dim), _blocks(case)
    lens = _lengths(case)
    st = dict(case=dict(case))
    pages = S * nb + 3
    st["table"] = torch.randperm(pages, generator=g, device="cuda")[: S * nb].to(torch.int32).reshape(S, nb).contiguous()
    st["sequence"] = torch.tensor([i if L >= 0 else -1 for i, L in enumerate(lens)], dtype=torch.int32, device="cuda")
    st["start"] = torch.tensor([L - n if L >= 0 else 0 for L in lens], dtype=torch.int32, device="cuda")
    st["workspace"] = torch.zeros(32 << 20, dtype=torch.uint8, device="cuda")
    # keys have a few large channels, as rotated keys do; values are plain
    loud = 1 + 3 * (torch.rand(kv, 1, dim, generator=g, device="cuda") < 0.06).float()
    if case["op"] == "append":
        st["codes"] = torch.zeros(pages, kv, 2, padded * 64, dtype=torch.int8, device="cuda")
        st["marks"] = torch.zeros(pages, kv, 2, padded, dtype=torch.int8, device="cuda")
        st["scales"] = torch.ones(pages, kv, 2, device="cuda")
        st["open"] = torch.zeros(S, 2, BLOCK, kv, dim, device="cuda")
        # what the open blocks hold so far goes in through the operator's plain form
        st["start"], goal = st["start"] // BLOCK * BLOCK, st["start"]
        held = dict(st, case=dict(case, count=BLOCK - 1))
        k, v = (torch.randn(S, BLOCK - 1, kv, dim, generator=g, device="cuda") for _ in range(2))
        rows = (goal % BLOCK).clamp(min=1)
        gone = torch.arange(BLOCK - 1, device="cuda")[None, :] >= rows[:, None]
        k, v = (torch.where(gone[:, :, None, None], torch.zeros((), device="cuda"), t) for t in (k * loud[:, 0], v))
        _append(held, k, v)
        st["start"] = goal
        # rows past the open ones have not been written: marks come from the rows there are
        _remark(st, goal % BLOCK, goal // BLOCK)
        st["k"] = (torch.randn(S, n, kv, dim, generator=g, device="cuda") * loud[:, 0]).reshape(S * n, kv * dim)
        st["v"] = torch.randn(S, n, kv, dim, generator=g, device="cuda").reshape(S * n, kv * dim)
        return st
    st["open"] = torch.zeros(S, 2, BLOCK, kv, dim, device="cuda")
    st["codes"] = torch.empty(pages, kv, 2, padded * 64, dtype=torch.int8, device="cuda")
    st["marks"] = torch.zeros(pages, kv, 2, padded, dtype=torch.int8, device="cuda")
    st["scales"] = torch.empty(pages, kv, 2, device="cuda")
    step = max(1, (1 << 27) // (kv * BLOCK * dim))
    at = 0
    while at < pages:
        m = min(step, pages - at)
        size = torch.exp(0.3 * torch.randn(m, kv, 1, 1, generator=g, device="cuda"))
        # neighbouring tokens' keys are alike: each block has a direction of its own
        x = (torch.randn(m, kv, BLOCK, dim, generator=g, device="cuda") + torch.randn(m, kv, 1, dim, generator=g, device="cuda")) * size * loud
        s = _scale_of(x.abs().amax((-1, -2)))
        code = _codes_of(x, s)
        st["codes"][at:at + m, :, 0], st["scales"][at:at + m, :, 0] = _pack_keys(code, padded), s
        f = code.float()
        st["marks"][at:at + m, :, 0, :dim], st["marks"][at:at + m, :, 1, :dim] = f.amin(-2).to(torch.int8), f.amax(-2).to(torch.int8)
        x = torch.randn(m, kv, BLOCK, dim, generator=g, device="cuda") * size
        s = _scale_of(x.abs().amax((-1, -2)))
        st["codes"][at:at + m, :, 1], st["scales"][at:at + m, :, 1] = _pack_values(_codes_of(x, s), padded), s
        at += m
    st["q"] = torch.randn(S * n, H * dim, generator=g, device="cuda")
    if case["op"] == "sparse":
        st["picks"] = _select(st)
    return st


def _remark(st, rows, block):
    """Marks of each sequence's open block over its first `rows` tokens."""
    S, dim = st["table"].shape[0], st["case"]["dim"]
    page = st["table"][torch.arange(S, device="cuda"), block.long().clamp(max=st["table"].shape[1] - 1)].long()
    k = _keys(st["codes"][page][:, :, 0], dim).float()
    there = (torch.arange(BLOCK, device="cuda")[None] < rows[:, None])[:, None, :, None]
    st["marks"][page, :, 0, :dim] = torch.where(there, k, torch.full_like(k, 127.0)).amin(-2).to(torch.int8)
    st["marks"][page, :, 1, :dim] = torch.where(there, k, torch.full_like(k, -127.0)).amax(-2).to(torch.int8)


def run(state):
    if own:
        return _run_own(state)
    c = state["case"]
    if c["op"] == "append":
        S, n = c["segments"], c["count"]
        return _append(state, state["k"].reshape(S, n, c["kv"], c["dim"]), state["v"].reshape(S, n, c["kv"], c["dim"]))
    return {"attend": _attend, "select": _select, "sparse": _sparse}[c["op"]](state)


def work(case):
    S, n, H, kv, dim, top = (case[k] for k in ("segments", "count", "heads", "kv", "dim", "top"))
    live = [L for L in _lengths(case) if L >= 0]
    tokens = len(live) * n
    if case["op"] == "append":
        # the new rows, their codes and each touched block's scales and marks; two products, a rounding and the comparisons
        touched = sum((L - 1) // BLOCK - (L - n) // BLOCK + 1 for L in live)
        return dict(bytes=tokens * kv * dim * 2 * 5 + touched * kv * (2 * dim + 8), flops=tokens * kv * dim * 2 * 4)
    rows = tokens * H * dim * 4
    if case["op"] == "select":
        blocks = sum((L + BLOCK - 1) // BLOCK for L in live)
        pairs = sum(sum((p + BLOCK) // BLOCK for p in range(L - n, L)) for L in live)
        return dict(bytes=rows + blocks * kv * (2 * dim + 4) + tokens * kv * top * 4, flops=4 * pairs * kv * dim)
    if case["op"] == "attend":
        pairs = sum(n * L - n * (n - 1) // 2 for L in live)
        seen = sum(live)
    else:
        pairs = sum(min(p + 1, top * BLOCK - (BLOCK - 1 - p % BLOCK)) for L in live for p in range(L - n, L))
        seen = min(pairs, sum(live))
    return dict(bytes=2 * rows + seen * kv * dim * 2 + (seen // BLOCK) * kv * 8, flops=4 * pairs * H * dim)


def exact(case, seed):
    """From the definition, in 64 bits; block choices are whole numbers and have no such value."""
    if case["op"] == "select":
        return None
    st = prepare(case, seed)
    S, n, H, kv, dim = case["segments"], case["count"], case["heads"], case["kv"], case["dim"]
    if case["op"] == "append":
        scales, opened = st["scales"].double(), st["open"].double()
        k, v = (st[x].double().reshape(S, n, kv, dim) for x in "kv")
        for i, s in enumerate(st["sequence"].tolist()):
            if s < 0:
                continue
            start = int(st["start"][i])
            row = start % BLOCK
            joined = torch.cat([opened[s][:, :row], torch.stack([k[i], v[i]])], 1)  # [2, row + n, kv, dim]
            for b in range((row + n + BLOCK - 1) // BLOCK):
                part = joined[:, b * BLOCK:(b + 1) * BLOCK]
                scales[int(st["table"][s, start // BLOCK + b])] = (part.abs().amax((1, 3)) / 127).transpose(0, 1)
            left = (row + n) % BLOCK
            if left:
                opened[s][:, :left] = joined[:, -left:] if left <= joined.shape[1] else joined
        return None, None, scales, opened
    y = torch.zeros(S * n, H * dim, dtype=torch.float64, device="cuda")
    seqs, starts = st["sequence"].tolist(), st["start"].tolist()
    G, padded = H // kv, _padded(dim)
    for i in range(S):
        if seqs[i] < 0:
            continue
        L = starts[i] + n
        nb = (L + BLOCK - 1) // BLOCK
        page = st["table"][seqs[i], :nb].long()
        at = torch.arange(nb * BLOCK, device="cuda")
        pos = starts[i] + torch.arange(n, device="cuda")
        for h in range(kv):
            k = st["codes"][page, h, 0].double().reshape(nb, padded // 64, BLOCK, 64).permute(0, 2, 1, 3).reshape(nb, BLOCK, padded)
            v = st["codes"][page, h, 1].double().reshape(nb, padded, BLOCK).permute(0, 2, 1)
            k = (k * st["scales"][page, h, 0].double()[:, None, None]).reshape(nb * BLOCK, padded)[:, :dim]
            v = (v * st["scales"][page, h, 1].double()[:, None, None]).reshape(nb * BLOCK, padded)[:, :dim]
            allowed = at[None] <= pos[:, None]
            if case["op"] == "sparse":
                mine = st["picks"].reshape(S, n, kv, -1)[i, :, h].long()
                chosen = torch.zeros(n, nb + 1, dtype=torch.bool, device="cuda")
                chosen.scatter_(1, torch.where(mine >= 0, mine, torch.full_like(mine, nb)), True)
                allowed = allowed & chosen[:, :nb].repeat_interleave(BLOCK, 1)
            for g in range(G):
                col = (h * G + g) * dim
                q = st["q"][i * n:(i + 1) * n, col:col + dim].double()
                a = (q @ k.T) / math.sqrt(dim)
                a = torch.softmax(a.masked_fill(~allowed, -math.inf), -1)
                y[i * n:(i + 1) * n, col:col + dim] = a @ v
    return y
