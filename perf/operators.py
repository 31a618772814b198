"""Cases of the 8-bit paged K/V cache and of the operators around it: the
cache written (with what it then holds read back), read back at length,
attended over, and the normed and rotated queries and keys that go into it.

The cache's format, which the plain forms below define as well: a block is 16
positions of one K/V head; its keys (and, apart, its values) share one scale
2^e, e the smallest integer in [-48, 64] for which no element of the block
exceeds 127 * 2^e; an element x is held as the integer nearest x / 2^e (ties
to even, at most 127 in magnitude). Rows written into a block that already
holds earlier positions raise e when they need to, never lower it; the
integers of the earlier positions are then divided by the ratio of the two
scales and rounded again.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 16
E_MIN, E_MAX = -48, 64
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
DEV = "cuda"


# --------------------------------------------------------------------- cases
def listed():
    return [
        # one utterance of the engine's decode loop, a frame into its second minute
        dict(name="attend_one", op="attend", n=1, lo=1000, hi=1000, rows=1, heads=8, kv_heads=8, dim=64, window=0,
             type="f32"),
        # a full serving step: 512 utterances around a thousand positions
        dict(name="attend_streams", op="attend", n=512, lo=500, hi=1500, rows=1, heads=8, kv_heads=8, dim=64,
             window=0, type="f32"),
        # a few utterances near the position limit
        dict(name="attend_long", op="attend", n=8, lo=7900, hi=8100, rows=1, heads=8, kv_heads=8, dim=64, window=0,
             type="f32"),
        # grouped heads of a larger decoder, contexts of every length, bf16 activations
        dict(name="attend_grouped", op="attend", n=48, lo=0, hi=4096, rows=1, heads=32, kv_heads=8, dim=128,
             window=0, type="bf16"),
        # a chunk of prefill over what the stream holds already
        dict(name="attend_prompt", op="attend", n=4, lo=300, hi=2048, rows=256, heads=8, kv_heads=8, dim=64,
             window=0, type="f32"),
        # the latent decoder: 16 rows a frame over a window of 250 keys, 64 requests
        dict(name="attend_window", op="attend", n=64, lo=16, hi=700, rows=16, heads=8, kv_heads=8, dim=64,
             window=250, type="f32"),
        # the rows of one step go into the cache of 512 streams
        dict(name="write_step", op="write", n=512, lo=1, hi=1500, rows=1, kv_heads=8, dim=64, type="f32"),
        # chunks of prompts, from the middle of a block on
        dict(name="write_prompt", op="write", n=16, lo=1, hi=1023, rows=511, kv_heads=8, dim=128, type="bf16"),
        # one long stream handed to another worker
        dict(name="read_stream", op="read", n=1, lo=8000, hi=8000, kv_heads=8, dim=64, type="f32"),
        # a batch of contexts read back for a layer that computes in bf16
        dict(name="read_many", op="read", n=64, lo=0, hi=2047, kv_heads=8, dim=128, type="bf16"),
        # queries and keys of one decode step
        dict(name="turn_step", op="turn", tokens=64, far=8191, heads=8, kv_heads=8, dim=64, rotary=64, pairs="next",
             type="f32"),
        # queries and keys of a prompt, grouped heads, halves paired, three quarters of each head turned
        dict(name="turn_prompt", op="turn", tokens=8192, far=131071, heads=32, kv_heads=8, dim=128, rotary=96,
             pairs="halves", type="bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "write", "read", "turn"])
    kind = rng.choice(["f32", "bf16"])
    dim = rng.choice([32, 64, 64, 128, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 5, 8, 8, 12])
    if op == "turn":
        heads = kv_heads * rng.choice([1, 2, 3, 4, 7])
        tokens = _log(rng, 1, max(2, 8192 * 40 * 128 // ((heads + kv_heads) * dim) // 2))
        rotary = rng.choice([dim, dim, dim // 2, dim // 4 * 3])
        return dict(op=op, tokens=min(tokens, 20000), far=_log(rng, 10, 500000), heads=heads, kv_heads=kv_heads,
                    dim=dim, rotary=rotary, pairs=rng.choice(["next", "halves"]), type=kind)
    hi = _log(rng, 1, 8191)
    most = max(1, 512 * 1000 * 512 // (hi * kv_heads * dim))
    lo = rng.choice([0, 1, hi // 2, hi])
    if op == "read":
        n = _log(rng, 1, min(256, max(1, most // 4)))
        return dict(op=op, n=n, lo=min(lo, hi), hi=hi, kv_heads=kv_heads, dim=dim, type=kind)
    if op == "write":
        n = _log(rng, 1, min(512, max(1, most // 4)))
        rows = rng.choice([1, 1, _log(rng, 1, 600)])
        return dict(op=op, n=n, lo=min(lo, hi), hi=hi, rows=min(rows, hi), kv_heads=kv_heads, dim=dim, type=kind)
    group = rng.choice([1, 1, 2, 3, 4, 7, 8])
    n = _log(rng, 1, min(512, most))
    rows = rng.choice([1, 1, 1, _log(rng, 2, 300)])
    # no more scores than the listed cases' largest
    while n > 1 and n * hi * rows * kv_heads * group > 4 * 2048 * 256 * 32:
        n = (n + 1) // 2
    rows = max(1, min(rows, 4 * 2048 * 256 * 32 // (n * hi * kv_heads * group)))
    return dict(op=op, n=n, lo=min(lo, hi), hi=hi, rows=rows, heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
                window=rng.choice([0, 0, 0, _log(rng, 1, 1000)]), type=kind)


def _shape(case, seed):
    """The batch on the host: lengths and rows of each sequence. Their values are the case's own, their order the
    seed's, so that every seed has the same work."""
    n, lo, hi = case["n"], case["lo"], case["hi"]
    fixed = np.random.RandomState(n * 7919 + hi * 31 + lo)
    lengths = np.sort(fixed.randint(lo, hi + 1, n))
    lengths[-1] = hi
    if case["op"] == "read":
        rows = lengths.copy()
    else:
        rows = np.ones(n, np.int64) if case["rows"] == 1 else fixed.randint(1, case["rows"] + 1, n)
        if case["rows"] > 1:
            rows[-1] = case["rows"]
        rows = np.minimum(rows, np.maximum(lengths, 1 if case["op"] == "attend" else 0))
    order = np.random.RandomState(seed).permutation(n)
    return lengths[order].astype(np.int64), rows[order].astype(np.int64)


def _visible(case, lengths, rows):
    """(positions some row of the batch sees, pairs of a row and a position it sees)"""
    window = case["window"] or (1 << 30)
    first = np.maximum(0, lengths - rows + 1 - window)
    seen = int(np.maximum(0, lengths - first).sum())
    pairs = 0
    for length, count in zip(lengths, rows):
        at = np.arange(length - count, length)
        pairs += int(np.maximum(0, np.minimum(at + 1, window)).sum())
    return seen, pairs


def work(case):
    size = {"f32": 4, "bf16": 2}[case["type"]]
    if case["op"] == "turn":
        values = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * values * size + 4 * case["tokens"], "flops": 8 * values}
    lengths, rows = _shape(case, 0)
    width = case["kv_heads"] * case["dim"]
    held = 2 * width + 2 * case["kv_heads"] / BLOCK  # integers and scales of a position
    if case["op"] == "attend":
        seen, pairs = _visible(case, lengths, rows)
        wide = case["heads"] * case["dim"]
        return {"bytes": seen * held + 2 * int(rows.sum()) * wide * size, "flops": 4 * pairs * wide}
    if case["op"] == "read":
        total = int(lengths.sum())
        return {"bytes": total * (held + 2 * width * size), "flops": 2 * total * width}
    written = int(rows.sum())
    touched = int(_touched(lengths, rows)[1].sum())
    return {"bytes": written * (held + 2 * width * size) + touched * (held + 2 * width * size),
            "flops": 4 * (written + touched) * width}


def _touched(lengths, rows):
    """Of each sequence the first position of the first block that the write touches, and the positions from there."""
    first = (lengths - rows) // BLOCK * BLOCK
    return first, np.where(rows > 0, lengths - first, 0)


# -------------------------------------------------------------------- inputs
def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _history(case, seed, total):
    """Key and value rows [total][kv_heads][dim] as a layer makes them: keys with a few loud channels, both with a
    loudness of their own for each position and head."""
    gen = torch.Generator(device=DEV).manual_seed(seed * 2 + 1)
    kvh, dim, kind = case["kv_heads"], case["dim"], TYPES[case["type"]]
    loud = 1 + 4 * (torch.rand(1, kvh, dim, generator=gen, device=DEV) > 0.95)
    out = []
    for scale in (loud, 1.0):
        x = _normal(gen, total, kvh, dim)
        x *= torch.exp(0.5 * _normal(gen, total, kvh, 1))
        x *= scale
        out.append(x.to(kind))
    return out


def _inputs(case, seed):
    """Everything the operators are given, on the device, and the host's view of the batch."""
    kind = TYPES[case["type"]]
    gen = torch.Generator(device=DEV).manual_seed(seed * 2 + 2)
    if case["op"] == "turn":
        t, h, kvh, dim = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        s = {"packed": (2 * _normal(gen, t, h + 2 * kvh, dim)).to(kind),
             "q_weight": 1 + 0.2 * _normal(gen, dim), "k_weight": 1 + 0.2 * _normal(gen, dim)}
        at = np.random.RandomState(seed).randint(0, case["far"] + 1, t)
        return s | {"positions": torch.tensor(at, dtype=torch.int32, device=DEV)}
    lengths, rows = _shape(case, seed)
    pages = -(-lengths // BLOCK)
    stride = max(1, int(pages.max()))
    pool = int(pages.sum()) + 3
    order = np.random.RandomState(seed + 1).permutation(pool)
    table = np.zeros((len(lengths), stride), np.int32)
    table[np.arange(stride)[None] < pages[:, None]] = order[:int(pages.sum())]
    i32 = lambda a: torch.tensor(np.ascontiguousarray(a), dtype=torch.int32, device=DEV)  # noqa: E731
    begin = lambda a: i32(np.concatenate([[0], np.cumsum(a)]))  # noqa: E731
    s = {"lengths": i32(lengths), "table": i32(table), "row_begin": begin(rows), "rows": int(rows.sum()),
         "pool": pool, "hi": int(lengths.max()), "most": max(1, int(rows.max())), "host": (lengths, rows)}
    k, v = _history(case, seed, int(lengths.sum()))
    if case["op"] == "attend":
        q = _normal(gen, s["rows"], case["heads"], case["dim"]) * torch.exp(0.3 * _normal(gen, s["rows"], case["heads"], 1))
        return s | {"k": k, "v": v, "hist": begin(lengths), "q": q.to(kind)}
    if case["op"] == "read":
        return s | {"k": k, "v": v, "hist": begin(lengths)}
    # a write: the first lengths - rows positions are there before the call, the rest come with it
    new = np.concatenate([np.arange(a, b) for a, b in zip(np.cumsum(lengths) - rows, np.cumsum(lengths))] or [[]])
    old = np.setdiff1d(np.arange(int(lengths.sum())), new)
    pick = lambda x, at: x[torch.tensor(at, dtype=torch.int64, device=DEV)]  # noqa: E731
    first, count = _touched(lengths, rows)
    return s | {"k": pick(k, old), "v": pick(v, old), "hist": begin(lengths - rows), "before": i32(lengths - rows),
                "k_new": pick(k, new), "v_new": pick(v, new), "back_begin": begin(count), "back": int(count.sum()),
                "back_most": max(1, int(count.max()))}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] == "turn":
        t, dim = case["tokens"], case["dim"]
        s["q_out"] = torch.empty(t, case["heads"], dim, dtype=s["packed"].dtype, device=DEV)
        s["k_out"] = torch.empty(t, case["kv_heads"], dim, dtype=s["packed"].dtype, device=DEV)
        if own:
            s["call"] = _own_turn(s)
        return s
    lengths = s["before"] if case["op"] == "write" else s["lengths"]
    if own:
        _own_prepare(s, lengths)
    else:
        shape = (s["pool"], case["kv_heads"], BLOCK, case["dim"])
        s["cache"] = {"k": torch.zeros(shape, dtype=torch.int8, device=DEV),
                      "v": torch.zeros(shape, dtype=torch.int8, device=DEV),
                      "ke": torch.full(shape[:2], E_MIN, dtype=torch.int32, device=DEV),
                      "ve": torch.full(shape[:2], E_MIN, dtype=torch.int32, device=DEV)}
        held = s["host"][0] - (s["host"][1] if case["op"] == "write" else 0)
        blocks = int((-(-held // BLOCK)).sum())
        _write(s["cache"], s["table"], lengths, s["hist"], s["k"], s["v"], blocks)
    if case["op"] == "write":
        s["blocks"] = int((-(-_touched(*s["host"])[1] // BLOCK)).sum())
    for name in ("k", "v", "hist", "host"):
        s.pop(name)
    return s


# --------------------------------------------------------------- plain forms
def _pow2(e):
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _exponent(amax):
    """The smallest e with amax <= 127 * 2^e: amax = m * 2^k, m in [0.5, 1)."""
    m, k = torch.frexp(amax)
    return torch.where(amax > 0, k - 7 + (m > 127 / 128).to(k.dtype), E_MIN).clamp(E_MIN, E_MAX)


def _write(cache, table, lengths, begin, k, v, blocks):
    """Rows [begin[i], begin[i+1]) of k and v become the last positions of sequence i, in `blocks` blocks."""
    if blocks == 0 or k.shape[0] == 0:
        return
    count = (begin[1:] - begin[:-1]).long()
    length = lengths.long()
    start = length - count
    first = start // BLOCK
    held = torch.where(count > 0, (length + BLOCK - 1) // BLOCK - first, 0)
    ends = torch.cumsum(held, 0)
    at = torch.arange(blocks, device=DEV)
    seq = torch.searchsorted(ends, at, right=True)
    block = at - (ends - held)[seq] + first[seq]
    page = table[seq, block].long()
    pos = block[:, None] * BLOCK + torch.arange(BLOCK, device=DEV)
    new = (pos >= start[seq][:, None]) & (pos < length[seq][:, None])
    keep = pos < start[seq][:, None]
    row = (begin[:-1].long()[seq][:, None] + pos - start[seq][:, None]).clamp(0, k.shape[0] - 1)
    for x, codes, exps in ((k, cache["k"], cache["ke"]), (v, cache["v"], cache["ve"])):
        x = torch.where(new[..., None, None], x[row].float(), 0.0).transpose(1, 2)  # [blocks][heads][16][dim]
        e = _exponent(x.abs().amax((2, 3)))
        was = torch.where(keep.any(1)[:, None], exps[page], E_MIN)
        e = torch.maximum(e, was)
        old = torch.round(codes[page].float() * _pow2(was - e)[..., None, None])
        fresh = torch.round(x * _pow2(-e)[..., None, None]).clamp(-127, 127)
        codes[page] = torch.where(keep[:, None, :, None], old, fresh).to(torch.int8)
        exps[page] = e


def _held(cache, which, page):
    """The values of whole blocks: [...][heads][16][dim]"""
    return cache[which][page].float() * _pow2(cache[which + "e"][page])[..., None, None]


def _read(cache, table, lengths, begin, total, kind):
    """The last begin[i+1] - begin[i] positions of every sequence, in 32 bits, then in `kind`."""
    at = torch.arange(total, device=DEV)
    seq = torch.searchsorted(begin[1:].long(), at, right=True).clamp(max=lengths.shape[0] - 1)
    pos = lengths.long()[seq] - begin.long()[seq + 1] + at
    page, slot = table[seq, pos // BLOCK].long(), pos % BLOCK
    return [(cache[w][page, :, slot].float() * _pow2(cache[w + "e"][page])[..., None]).to(kind) for w in ("k", "v")]


def _attend(s, case):
    """Scores, softmax and the weighted sum of values over padded sequences, in 32 bits."""
    n, most, heads, kvh, dim = case["n"], s["most"], case["heads"], case["kv_heads"], case["dim"]
    group = heads // kvh
    table, length = s["table"].long(), s["lengths"].long()
    k = _held(s["cache"], "k", table).transpose(1, 2).reshape(n, kvh, -1, dim)
    v = _held(s["cache"], "v", table).transpose(1, 2).reshape(n, kvh, -1, dim)
    begin = s["row_begin"].long()
    count = begin[1:] - begin[:-1]
    r = torch.arange(most, device=DEV)
    row = (begin[:-1, None] + r).clamp(max=s["rows"] - 1)
    q = s["q"][row].float().reshape(n, most, kvh, group, dim).permute(0, 2, 1, 3, 4).reshape(n, kvh, most * group, dim)
    scores = q @ k.transpose(2, 3) / math.sqrt(dim)
    at = (length - count)[:, None] + r                                  # the position of each row
    key = torch.arange(k.shape[2], device=DEV)
    seen = (key <= at[..., None]) & (key < length[:, None, None])
    if case["window"]:
        seen &= key > at[..., None] - case["window"]
    seen = seen[:, None, :, None].expand(n, 1, most, group, -1).reshape(n, 1, most * group, -1)
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(3, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(3, keepdim=True)
    out = (p @ v) / torch.where(total == 0, 1.0, total)
    out = out.reshape(n, kvh, most, group, dim).permute(0, 2, 1, 3, 4).reshape(n * most, heads, dim)
    at = torch.arange(s["rows"], device=DEV)
    seq = torch.searchsorted(begin[1:], at, right=True)
    return out[seq * most + at - begin[seq]].to(s["q"].dtype)


def _turn(x, weight, positions, rotary, pairs):
    """RMS norm of every head, then the rotation of its first `rotary` values; the angles in 64 bits."""
    y = x.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * weight
    freq = 10000.0 ** (-torch.arange(0, rotary, 2, device=DEV, dtype=torch.float64) / rotary)
    angle = positions.double()[:, None] * freq
    c, n = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    if pairs == "next":
        a, b = y[..., 0:rotary:2].clone(), y[..., 1:rotary:2].clone()
        y[..., 0:rotary:2], y[..., 1:rotary:2] = a * c - b * n, a * n + b * c
    else:
        half = rotary // 2
        a, b = y[..., :half].clone(), y[..., half:rotary].clone()
        y[..., :half], y[..., half:rotary] = a * c - b * n, a * n + b * c
    return y.to(x.dtype)


# ------------------------------------------------------ the framework's calls
def _runtime():
    import sys
    if "speech-mac_b200" not in sys.path:
        sys.path.insert(0, "speech-mac_b200")
    from phonon_b200 import runtime
    return runtime


def _own_turn(s):
    rt, case = _runtime(), s["case"]
    t, h, kvh, dim = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    size = s["packed"].element_size()
    return rt.QkNormRope(
        q_ptr=s["packed"].data_ptr(), k_ptr=s["packed"].data_ptr() + h * dim * size, q_out_ptr=s["q_out"].data_ptr(),
        k_out_ptr=s["k_out"].data_ptr(), rows=t, heads=h, kv_heads=kvh, head_dim=dim, type=_own_type(rt, case),
        q_stride=(h + 2 * kvh) * dim, k_stride=(h + 2 * kvh) * dim, positions_ptr=s["positions"].data_ptr(),
        q_weight_ptr=s["q_weight"].data_ptr(), k_weight_ptr=s["k_weight"].data_ptr(), epsilon=1e-6, theta=10000.0,
        rotary_dim=case["rotary"], halves=case["pairs"] == "halves")


def _own_type(rt, case):
    return rt.ROWS_BF16 if case["type"] == "bf16" else rt.ROWS_F32


def _own_prepare(s, lengths):
    rt, case = _runtime(), s["case"]
    kind = _own_type(rt, case)
    s["cache"] = cache = rt.Kv8Cache(kv_heads=case["kv_heads"], head_dim=case["dim"], pool_pages=s["pool"])
    n, stride = s["table"].shape

    def batch(lengths, begin, rows, most):
        return rt.kv8_batch(sequences=n, rows=rows, lengths_ptr=lengths.data_ptr(), pages_ptr=s["table"].data_ptr(),
                            page_stride=stride, row_begin_ptr=begin.data_ptr(), max_rows=most, max_length=max(1, s["hi"]))

    held = s["k"].shape[0]
    stream = torch.cuda.current_stream().cuda_stream
    if held:
        cache.append(batch(lengths, s["hist"], held, max(1, s["hi"])),
                     rt.kv8_rows(s["k"].data_ptr(), s["v"].data_ptr(), kind), stream_ptr=stream)
        torch.cuda.current_stream().synchronize()  # the rows are let go
    back = lambda rows: [torch.empty(rows, case["kv_heads"], case["dim"], dtype=TYPES[case["type"]], device=DEV)  # noqa: E731
                         for _ in range(2)]
    s["batch"] = batch(s["lengths"], s["row_begin"], s["rows"], s["most"])
    if case["op"] == "attend":
        s["workspace"] = rt.Kv8Workspace(cache)
        s["out"] = torch.empty_like(s["q"])
        s["query"] = rt.kv8_query(s["q"].data_ptr(), s["out"].data_ptr(), kind, heads=case["heads"],
                                  window=case["window"])
    elif case["op"] == "read":
        s["out"] = back(s["rows"])
        s["to"] = rt.kv8_rows(s["out"][0].data_ptr(), s["out"][1].data_ptr(), kind)
    else:
        s["new"] = rt.kv8_rows(s["k_new"].data_ptr(), s["v_new"].data_ptr(), kind)
        s["out"] = back(s["back"])
        s["back_batch"] = batch(s["lengths"], s["back_begin"], s["back"], s["back_most"])
        s["to"] = rt.kv8_rows(s["out"][0].data_ptr(), s["out"][1].data_ptr(), kind)


def _own_run(s):
    op, stream = s["case"]["op"], torch.cuda.current_stream().cuda_stream
    if op == "turn":
        s["call"](stream_ptr=stream)
        return s["q_out"], s["k_out"]
    if op == "attend":
        s["cache"].attention(s["batch"], s["query"], s["workspace"], stream_ptr=stream)
    elif op == "read":
        s["cache"].read(s["batch"], s["to"], stream_ptr=stream)
    else:
        if s["rows"]:
            s["cache"].append(s["batch"], s["new"], stream_ptr=stream)
        if s["back"]:
            s["cache"].read(s["back_batch"], s["to"], stream_ptr=stream)
    return s["out"]


def run(s):
    if own:
        return _own_run(s)
    case = s["case"]
    kind = TYPES[case["type"]]
    if case["op"] == "turn":
        h = case["heads"]
        return (_turn(s["packed"][:, :h], s["q_weight"], s["positions"], case["rotary"], case["pairs"]),
                _turn(s["packed"][:, h:h + case["kv_heads"]], s["k_weight"], s["positions"], case["rotary"], case["pairs"]))
    if case["op"] == "attend":
        return _attend(s, case)
    if case["op"] == "read":
        return _read(s["cache"], s["table"], s["lengths"], s["row_begin"], s["rows"], kind)
    _write(s["cache"], s["table"], s["lengths"], s["row_begin"], s["k_new"], s["v_new"], s["blocks"])
    return _read(s["cache"], s["table"], s["lengths"], s["back_begin"], s["back"], kind)


# ------------------------------------------------------- the same, in 64 bits
def _exact_held(x, before):
    """What a sequence's rows x [length][heads][dim] come back as, `before` of them written first and the rest in a
    second call; all in 64 bits."""
    length = x.shape[0]
    full = -(-length // BLOCK) * BLOCK
    y = torch.zeros(full, *x.shape[1:], dtype=torch.float64, device=DEV)
    y[:length] = x.double()
    y = y.reshape(-1, BLOCK, *x.shape[1:])
    units = torch.tensor([2.0 ** e for e in range(E_MIN, E_MAX + 1)], dtype=torch.float64, device=DEV)

    def step(z):
        return units[torch.searchsorted(127 * units[:-1], z.abs().amax((1, 3)).contiguous())][:, None, :, None]

    def near(z, unit):
        return torch.round(z / unit).clamp(-127, 127)

    cut = torch.arange(full, device=DEV).reshape(-1, BLOCK)[..., None, None] < before
    old = torch.where(cut, y, 0.0)
    unit_old, unit_all = step(old), torch.maximum(step(old), step(torch.where(cut, 0.0, y)))
    mixed = cut.any(1, keepdim=True) & ~(torch.arange(full, device=DEV).reshape(-1, BLOCK)[:, -1:, None, None] < before)
    unit = torch.where(mixed, unit_all, step(y))
    kept = torch.round(near(old, unit_old) * (unit_old / unit))
    held = torch.where(cut & mixed, kept, near(y, unit)) * unit
    return held.reshape(full, *x.shape[1:])[:length]


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "turn":
        h, kvh, rot = case["heads"], case["kv_heads"], case["rotary"]
        at = s["positions"].double()
        out = []
        for x, w in ((s["packed"][:, :h], s["q_weight"]), (s["packed"][:, h:h + kvh], s["k_weight"])):
            x = x.double()
            x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / case["dim"] + 1e-6) * w.double()
            turn = torch.exp(-math.log(10000.0) * torch.arange(rot // 2, device=DEV, dtype=torch.float64) * 2 / rot)
            z = torch.polar(torch.ones(1, dtype=torch.float64, device=DEV), at[:, None, None] * turn)
            head = x[..., :rot]
            if case["pairs"] == "next":
                w2 = torch.view_as_real(torch.view_as_complex(head.reshape(*head.shape[:-1], -1, 2).contiguous()) * z)
                head = w2.reshape(head.shape)
            else:
                w2 = torch.complex(head[..., :rot // 2].contiguous(), head[..., rot // 2:].contiguous()) * z
                head = torch.cat([w2.real, w2.imag], -1)
            out.append(torch.cat([head, x[..., rot:]], -1))
        return tuple(out)
    lengths, rows = s["host"]
    hist = s["hist"].tolist()
    if case["op"] in ("read", "write"):
        outs = [[], []]
        new = s["row_begin"].tolist()
        for i, (length, count) in enumerate(zip(lengths.tolist(), rows.tolist())):
            for o, name in zip(outs, ("k", "v")):
                x = s[name][hist[i]:hist[i + 1]]
                if case["op"] == "read":
                    o.append(_exact_held(x, length) if length else x.double())
                elif count:
                    x = torch.cat([x, s[name + "_new"][new[i]:new[i + 1]]])
                    first = (length - count) // BLOCK * BLOCK
                    o.append(_exact_held(x[first:], length - count - first))
        none = torch.zeros(0, case["kv_heads"], case["dim"], dtype=torch.float64, device=DEV)
        return [torch.cat(o) if o else none for o in outs]
    out = torch.zeros(s["rows"], case["heads"], case["dim"], dtype=torch.float64, device=DEV)
    group = case["heads"] // case["kv_heads"]
    begin = s["row_begin"].tolist()
    for i, (length, count) in enumerate(zip(lengths.tolist(), rows.tolist())):
        if length == 0:
            continue
        k, v = (_exact_held(s[name][hist[i]:hist[i + 1]], length).repeat_interleave(group, 1) for name in ("k", "v"))
        q = s["q"][begin[i]:begin[i + 1]].double()
        score = torch.einsum("rhd,khd->hrk", q, k) * case["dim"] ** -0.5
        at = torch.arange(length - count, length, device=DEV)[:, None]
        key = torch.arange(length, device=DEV)[None]
        hidden = key > at
        if case["window"]:
            hidden |= key <= at - case["window"]
        p = torch.softmax(score.masked_fill(hidden[None], -math.inf), -1)
        out[begin[i]:begin[i + 1]] = torch.einsum("hrk,khd->rhd", p, v)
    return out
