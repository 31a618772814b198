"""Cases of the operators of a prompt's pass through a layer: rows quantised to
8 bits with a scale each, the product of such rows with weights in 8 bits, and
causal attention over packed prompts.

Their definitions, which the plain forms below follow as well:

  quantize  s = max(max|x| / 127, 2^-126) of a row, rounded to 32 bits; an
            element x becomes the integer nearest x / s (ties to even, at most
            127 in magnitude)
  product   y[t][n] = x_scale[t] * w_scale[n] * sum_k x[t][k] w[n][k] + bias[n]
  attend    the row at position p of a prompt sees positions (p - window, p] of
            it ([0, p] where window is 0); softmax(q k / sqrt(dim)) v, query
            head h on K/V head h / (heads / kv_heads)
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
DEV = "cuda"


# --------------------------------------------------------------------- cases
def listed():
    return [
        # the rows of a decode step of 64 utterances, before a projection
        dict(name="quantize_step", op="quantize", rows=64, cols=512, type="f32"),
        # a batch of prompts, before a projection of a larger decoder
        dict(name="quantize_prompt", op="quantize", rows=8192, cols=4096, type="bf16"),
        # the engine's query, key and value projection for one utterance
        dict(name="product_one", op="product", rows=1, channels=1536, depth=512, bias=False, type="f32"),
        # a decode step of a larger decoder: 16 rows, bound by the weights
        dict(name="product_step", op="product", rows=16, channels=4096, depth=4096, bias=False, type="bf16"),
        # the engine's down projection for a serving step of 512 utterances
        dict(name="product_streams", op="product", rows=512, channels=512, depth=2048, bias=True, type="f32"),
        # odd sizes: prompts that end anywhere, a head of no round size
        dict(name="product_ragged", op="product", rows=1001, channels=5003, depth=2064, bias=True, type="bf16"),
        # a batch of prompts through the first half of a feed-forward block
        dict(name="product_prompt", op="product", rows=8192, channels=16384, depth=4096, bias=False, type="bf16"),
        # the engine's prefix of one utterance
        dict(name="attend_prefix", op="attend", n=1, lo=128, hi=128, heads=8, kv_heads=8, dim=64, window=0, type="f32"),
        # prompts of 64 utterances of every length, packed
        dict(name="attend_packed", op="attend", n=64, lo=1, hi=512, heads=8, kv_heads=8, dim=64, window=0, type="bf16"),
        # a few long prefixes of the engine, in its own 32 bits
        dict(name="attend_engine", op="attend", n=4, lo=1024, hi=2048, heads=8, kv_heads=8, dim=64, window=0,
             type="f32"),
        # whole requests of the latent decoder: a window of 250 positions
        dict(name="attend_window", op="attend", n=16, lo=100, hi=3000, heads=8, kv_heads=8, dim=64, window=250,
             type="bf16"),
        # two prompts of a larger decoder near the position limit, grouped heads
        dict(name="attend_long", op="attend", n=2, lo=7000, hi=8191, heads=32, kv_heads=8, dim=128, window=0,
             type="bf16"),
    ]


LARGEST = {"quantize": 8192 * 4096, "product": 8192 * 16384 * 4096, "attend": 2 * 7600 * 7600 // 2 * 32 * 128}


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "product", "product", "attend", "attend", "attend"])
    kind = rng.choice(["f32", "bf16"])
    if op == "quantize":
        cols = 16 * _log(rng, 1, 1024)
        return dict(op=op, rows=_log(rng, 1, min(20000, LARGEST[op] // cols)), cols=cols, type=kind)
    if op == "product":
        depth = 16 * _log(rng, 1, 512)
        channels = _log(rng, 1, 16384)
        rows = _log(rng, 1, max(1, min(8192, LARGEST[op] // (depth * channels))))
        return dict(op=op, rows=rows, channels=channels, depth=depth, bias=rng.random() < 0.5, type=kind)
    dim = rng.choice([32, 64, 64, 128, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 5, 8, 8, 12])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 7, 8])
    window = rng.choice([0, 0, 0, _log(rng, 1, 1000)])
    hi = _log(rng, 1, 8191)
    # in 32 bits the products cost several times as much
    most = LARGEST[op] // (heads * dim) // (6 if kind == "f32" else 1)
    hi = min(hi, int(math.sqrt(2 * most)))
    n = _log(rng, 1, max(1, min(256, 2 * most // (hi * hi), 60_000_000 // (hi * heads * dim))))
    return dict(op=op, n=n, lo=min(hi, rng.choice([0, 1, hi // 2, hi])), hi=hi, heads=heads, kv_heads=kv_heads, dim=dim,
                window=window, type=kind)


def _lengths(case, seed):
    """Lengths of the prompts: the values are the case's own, their order the seed's, so that every seed has the same
    work."""
    fixed = np.random.RandomState(case["n"] * 7919 + case["hi"] * 31 + case["lo"])
    lengths = np.sort(fixed.randint(case["lo"], case["hi"] + 1, case["n"]))
    lengths[-1] = case["hi"]
    return lengths[np.random.RandomState(seed).permutation(case["n"])].tolist()


def work(case):
    size = {"f32": 4, "bf16": 2}[case["type"]]
    if case["op"] == "quantize":
        values = case["rows"] * case["cols"]
        return {"bytes": values * (size + 1) + 4 * case["rows"], "flops": 4 * values}
    if case["op"] == "product":
        t, n, k = case["rows"], case["channels"], case["depth"]
        return {"bytes": t * k + n * k + t * n * size + 4 * (t + n * (2 if case["bias"] else 1)), "flops": 2 * t * n * k}
    lengths = _lengths(case, 0)
    window = case["window"] or (1 << 30)
    pairs = sum(int(np.minimum(np.arange(length) + 1, window).sum()) for length in lengths)
    values = sum(lengths) * 2 * (case["heads"] + case["kv_heads"]) * case["dim"]
    return {"bytes": values * size, "flops": 4 * pairs * case["heads"] * case["dim"]}


# -------------------------------------------------------------------- inputs
def _inputs(case, seed):
    kind = TYPES[case["type"]]
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    if case["op"] == "quantize":
        # activations: a loudness of each row, a few loud channels
        x = normal(case["rows"], case["cols"])
        x *= torch.exp(0.5 * normal(case["rows"], 1))
        x *= 1 + 7 * (torch.rand(1, case["cols"], generator=gen, device=DEV) > 0.98)
        return {"x": x.to(kind)}
    if case["op"] == "product":
        def eighths(rows, cols):  # rows as a quantiser leaves them
            out = torch.empty(rows, cols, dtype=torch.int8, device=DEV)
            for at in range(0, rows, 4096):
                y = normal(min(4096, rows - at), cols)
                out[at:at + 4096] = torch.round(y * (127 / y.abs().amax(1, keepdim=True)))
            return out
        t, n, k = case["rows"], case["channels"], case["depth"]
        s = {"x": eighths(t, k), "x_scales": 0.02 * torch.exp(0.5 * normal(t)), "w": eighths(n, k),
             "w_scales": 0.03 / math.sqrt(k) * torch.exp(0.2 * normal(n))}
        return s | ({"bias": 0.1 * normal(n)} if case["bias"] else {})
    lengths = _lengths(case, seed)
    rows, h, kvh, dim = sum(lengths), case["heads"], case["kv_heads"], case["dim"]
    # queries, keys and values side by side, as a projection leaves them
    packed = normal(max(1, rows), h + 2 * kvh, dim)
    packed[:, :h + kvh] *= 1 + 1.5 * (torch.rand(1, 1, dim, generator=gen, device=DEV) > 0.95)
    packed[:, h + kvh:] *= torch.exp(0.5 * normal(max(1, rows), kvh, 1))
    begin = torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device=DEV)
    return {"packed": packed.to(kind), "begin": begin, "lengths": lengths, "rows": rows}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        _own_prepare(s)
    return s


# --------------------------------------------------------------- plain forms
def _quantize(x):
    # (a quotient of tensors: by a number it would be a product with the rounded inverse)
    scales = (x.float().abs().amax(1) / torch.full((1,), 127.0, device=DEV)).clamp(min=2.0 ** -126)
    # (values next to a border: the quotient in 64 bits)
    codes = torch.round(x.double() / scales.double()[:, None]).clamp(-127, 127)
    return codes.to(torch.int8), scales


def _product(s, kind):
    y = s["x"].float() @ s["w"].float().t()
    y *= s["x_scales"][:, None]
    y *= s["w_scales"]
    if "bias" in s:
        y += s["bias"]
    return y.to(kind)


def _unseen(length, rows, window):
    """Which of the positions [0, length) the rows do not see."""
    key = torch.arange(length, device=DEV)
    hidden = key > rows[:, None]
    if window:
        hidden |= key <= rows[:, None] - window
    return hidden


def _attend(s, case):
    h, kvh, dim = case["heads"], case["kv_heads"], case["dim"]
    group = h // kvh
    out = torch.empty(s["rows"], h, dim, dtype=s["packed"].dtype, device=DEV)
    at = 0
    for length in s["lengths"]:
        x = s["packed"][at:at + length].float()
        q, k, v = x[:, :h].transpose(0, 1), x[:, h:h + kvh].transpose(0, 1), x[:, h + kvh:].transpose(0, 1)
        hidden = _unseen(length, torch.arange(length, device=DEV), case["window"])
        step = max(1, (1 << 29) // max(1, group * length * length))  # K/V heads at a time
        for c in range(0, kvh if length else 0, step):
            e = min(kvh, c + step)
            qs = q[c * group:e * group].reshape(e - c, group * length, dim)
            scores = (qs @ k[c:e].transpose(1, 2) / math.sqrt(dim)).reshape(e - c, group, length, length)
            scores.masked_fill_(hidden, -math.inf)
            p = torch.exp(scores - scores.amax(3, keepdim=True))
            y = (p.reshape(e - c, group * length, length) @ v[c:e]).reshape(e - c, group, length, dim)
            y = y / p.sum(3, keepdim=True)
            out[at:at + length, c * group:e * group] = y.reshape((e - c) * group, length, dim).transpose(0, 1).to(out.dtype)
        at += length
    return out


# ------------------------------------------------------ the framework's calls
def _runtime():
    import sys
    if "speech-mac_b200" not in sys.path:
        sys.path.insert(0, "speech-mac_b200")
    from phonon_b200 import runtime
    return runtime


def _own_prepare(s):
    rt, case = _runtime(), s["case"]
    kind = rt.ROWS_BF16 if case["type"] == "bf16" else rt.ROWS_F32
    if case["op"] == "quantize":
        s["out"] = (torch.empty(case["rows"], case["cols"], dtype=torch.int8, device=DEV),
                    torch.empty(case["rows"], device=DEV))
        s["call"] = rt.QuantizeRows(x_ptr=s["x"].data_ptr(), q_ptr=s["out"][0].data_ptr(), scales_ptr=s["out"][1].data_ptr(),
                                    rows=case["rows"], cols=case["cols"], type=kind)
    elif case["op"] == "product":
        s["out"] = torch.empty(case["rows"], case["channels"], dtype=TYPES[case["type"]], device=DEV)
        s["call"] = rt.I8Product(x_ptr=s["x"].data_ptr(), x_scales_ptr=s["x_scales"].data_ptr(), w_ptr=s["w"].data_ptr(),
                                 w_scales_ptr=s["w_scales"].data_ptr(), y_ptr=s["out"].data_ptr(), rows=case["rows"],
                                 channels=case["channels"], depth=case["depth"], type=kind,
                                 bias_ptr=s["bias"].data_ptr() if "bias" in s else None)
    else:
        h, kvh, dim = case["heads"], case["kv_heads"], case["dim"]
        s["out"] = torch.empty(s["rows"], h, dim, dtype=TYPES[case["type"]], device=DEV)
        at, size, stride = s["packed"].data_ptr(), s["packed"].element_size(), (h + 2 * kvh) * dim
        s["call"] = rt.PromptAttention(
            q_ptr=at, k_ptr=at + h * dim * size, v_ptr=at + (h + kvh) * dim * size, out_ptr=s["out"].data_ptr(),
            row_begin_ptr=s["begin"].data_ptr(), prompts=case["n"], rows=s["rows"], max_rows=max(1, max(s["lengths"])),
            heads=h, kv_heads=kvh, head_dim=dim, type=kind, window=case["window"], q_stride=stride, k_stride=stride,
            v_stride=stride)


def run(s):
    case = s["case"]
    if own:
        s["call"](stream_ptr=torch.cuda.current_stream().cuda_stream)
        return s["out"]
    if case["op"] == "quantize":
        return _quantize(s["x"])
    if case["op"] == "product":
        return _product(s, TYPES[case["type"]])
    return _attend(s, case)


# ------------------------------------------------------- the same, in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "quantize":
        # the scale is a number of 32 bits, and the integers are relative to that
        x = s["x"].double()
        top = torch.maximum(x.max(1).values, -x.min(1).values)
        scales = torch.maximum((top / torch.full((1,), 127.0, dtype=torch.float64, device=DEV)).float(), torch.tensor(2.0 ** -126, device=DEV)).double()
        low = torch.floor(x / scales[:, None])
        rest = x / scales[:, None] - low
        up = (rest > 0.5) | ((rest == 0.5) & (torch.remainder(low, 2) == 1))
        return (low + up).clamp(-127, 127), scales
    if case["op"] == "product":
        out = torch.empty(case["rows"], case["channels"], dtype=torch.float64, device=DEV)
        w = s["w"].double()
        for at in range(0, case["rows"], 2048):
            out[at:at + 2048] = torch.einsum("tk,nk->tn", s["x"][at:at + 2048].double(), w)
        out *= s["x_scales"].double()[:, None] * s["w_scales"].double()[None]
        return out + s["bias"].double() if "bias" in s else out
    h, kvh, dim, window = case["heads"], case["kv_heads"], case["dim"], case["window"]
    out = torch.zeros(s["rows"], h, dim, dtype=torch.float64, device=DEV)
    begin = s["begin"].tolist()
    for b, e in zip(begin, begin[1:]):
        for r in range(b, e, 1024):  # the rows [r, last), which see no position before `low`
            last = min(e, r + 1024)
            low = max(b, r - window + 1) if window else b
            k, v = (s["packed"][low:last, h + c * kvh:h + (c + 1) * kvh].double() for c in (0, 1))
            hidden = _unseen(last - low, torch.arange(r - low, last - low, device=DEV), window)
            for head in range(h):
                c = head * kvh // h
                score = s["packed"][r:last, head].double() @ k[:, c].t() * dim ** -0.5
                out[r:last, head] = torch.softmax(score.masked_fill(hidden, -math.inf), 1) @ v[:, c]
    return out
