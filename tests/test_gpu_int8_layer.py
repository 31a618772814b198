"""The attention half of a layer with 8-bit weights, as a server runs it: prompts packed together go through the
projection in 8 bits, the norm and rotation of their heads, causal attention and the output projection, and into the
8-bit cache; then each sequence goes on by single tokens over the cache. Each stage is held to its definition in 64 bits
over the rows that it got."""
import numpy as np
import pytest

import kv8_model
from phonon_b200 import runtime as rt
from test_gpu_i8 import check_product, product_case, product_want, quantized
from test_gpu_kv8 import Cache, f64
from test_gpu_prompt import call as prompt_call
from test_gpu_prompt import formula as prompt_formula
from test_gpu_qk_norm_rope import bound as rope_bound
from test_gpu_qk_norm_rope import formula as rope_formula

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

HEADS, KVH, DIM, WIDTH = 6, 2, 64, 256
EPS, THETA = 1e-6, 10000.0


class Stage:
    """Rows through one pass of the layer: calls made once, over buffers of their own."""

    def __init__(self, rows, dtype, weights, positions, attend):
        kind = rt.ROWS_BF16 if dtype == torch.bfloat16 else rt.ROWS_F32
        empty = lambda *shape, t=dtype: torch.empty(*shape, dtype=t, device="cuda")  # noqa: E731
        qkv = (HEADS + 2 * KVH) * DIM
        self.rows, self.bf16, self.weights, self.positions = rows, dtype == torch.bfloat16, weights, positions
        self.x, self.codes, self.scales = empty(rows, WIDTH), empty(rows, WIDTH, t=torch.int8), empty(rows, t=torch.float32)
        self.packed, self.seen = empty(rows, HEADS + 2 * KVH, DIM), empty(rows, HEADS, DIM)
        self.q, self.k, self.v = self.packed[:, :HEADS], self.packed[:, HEADS:HEADS + KVH], self.packed[:, HEADS + KVH:]
        self.out_codes, self.out_scales = empty(rows, HEADS * DIM, t=torch.int8), empty(rows, t=torch.float32)
        self.y = empty(rows, WIDTH)
        self.raw = empty(rows, HEADS + 2 * KVH, DIM)
        w, ws, bias, wo, wos, norm = weights
        self.first = [rt.QuantizeRows(self.x.data_ptr(), self.codes.data_ptr(), self.scales.data_ptr(), rows, WIDTH, kind),
                      rt.I8Product(self.codes.data_ptr(), self.scales.data_ptr(), w.data_ptr(), ws.data_ptr(), self.packed.data_ptr(),
                                   rows, qkv, WIDTH, kind, bias_ptr=bias.data_ptr())]
        stride = self.packed.stride(0)
        self.rope = rt.QkNormRope(self.q.data_ptr(), self.k.data_ptr(), self.q.data_ptr(), self.k.data_ptr(), rows, HEADS, KVH, DIM,
                                  positions.data_ptr(), kind, stride, stride, stride, stride, norm.data_ptr(), norm.data_ptr(), EPS, THETA)
        self.attend = attend(self)
        self.last = [rt.QuantizeRows(self.seen.data_ptr(), self.out_codes.data_ptr(), self.out_scales.data_ptr(), rows, HEADS * DIM, kind),
                     rt.I8Product(self.out_codes.data_ptr(), self.out_scales.data_ptr(), wo.data_ptr(), wos.data_ptr(), self.y.data_ptr(),
                                  rows, WIDTH, HEADS * DIM, kind)]

    def run(self, stream):
        for c in self.first:
            c(stream_ptr=stream)
        self.raw.copy_(self.packed)
        self.rope(stream_ptr=stream)
        for c in self.attend:
            c(stream)
        for c in self.last:
            c(stream_ptr=stream)

    def check(self):
        """All but the attention."""
        w, ws, bias, wo, wos, norm = self.weights
        for x, codes, scales in ((self.x, self.codes, self.scales), (self.seen.reshape(self.rows, -1), self.out_codes, self.out_scales)):
            want, s = quantized(f64(x))
            assert np.array_equal(f64(codes), want) and np.array_equal(f64(scales), s)
        check_product(self.raw.reshape(self.rows, -1), *product_want(self.codes, w, self.scales, ws, bias), self.bf16)
        check_product(self.y, *product_want(self.out_codes, wo, self.out_scales, wos, None), self.bf16)
        at, scale = f64(self.positions), f64(norm)
        for raw, got in ((self.raw[:, :HEADS], self.q), (self.raw[:, HEADS:HEADS + KVH], self.k)):
            want = rope_formula(f64(raw), scale, at, DIM, False, EPS, THETA)
            assert (np.abs(f64(got) - want) <= rope_bound(f64(raw), scale, DIM, EPS, want, self.bf16)).all()
        assert torch.equal(self.raw[:, HEADS + KVH:], self.v)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lengths", [[1, 37, 130, 64], [300, 2, 15]])
def test_prompts_then_single_tokens(cuda_ok, lengths, dtype):
    rng = np.random.default_rng(sum(lengths))
    bf16, n, steps = dtype == torch.bfloat16, len(lengths), 3
    _, w, _, ws = product_case(rng, 1, (HEADS + 2 * KVH) * DIM, WIDTH)
    _, wo, _, wos = product_case(rng, 1, WIDTH, HEADS * DIM)
    floats = lambda x: torch.tensor(x, dtype=torch.float32, device="cuda")  # noqa: E731
    weights = (w, ws, floats(rng.standard_normal((HEADS + 2 * KVH) * DIM)), wo, wos, floats(1 + 0.2 * rng.standard_normal(DIM)))
    cache = Cache(KVH, DIM, [m + steps for m in lengths])
    workspace = rt.Kv8Workspace(cache.kv)
    kind = rt.ROWS_BF16 if bf16 else rt.ROWS_F32
    begin = [0] + [int(b) for b in np.cumsum(lengths)]
    full = cache.batch(lengths, lengths)

    def rows_of(s):
        return rt.kv8_rows(s.k.data_ptr(), s.v.data_ptr(), kind, stride=s.packed.stride(0))

    def prompts(s):
        c = prompt_call(s.q, s.k, s.v, s.seen, begin, bf16=bf16)
        return [lambda stream: c(stream_ptr=stream), lambda stream: cache.kv.append(full, rows_of(s), stream_ptr=stream)]

    now = torch.tensor(lengths, dtype=torch.int32, device="cuda")  # lengths with the step's token
    one = rt.kv8_batch(n, now.data_ptr(), cache.table.data_ptr(), cache.stride, max_length=cache.stride * 16)

    def tokens(s):
        query = rt.kv8_query(s.q.data_ptr(), s.seen.data_ptr(), kind, heads=HEADS, q_stride=s.packed.stride(0))
        return [lambda stream: cache.kv.append(one, rows_of(s), stream_ptr=stream),
                lambda stream: cache.kv.attention(one, query, workspace, stream_ptr=stream)]

    at = torch.tensor(np.concatenate([np.arange(m) for m in lengths]), dtype=torch.int32, device="cuda")
    prompt, token = Stage(begin[-1], dtype, weights, at, prompts), Stage(n, dtype, weights, torch.empty_like(now), tokens)
    inputs = [torch.tensor(rng.standard_normal((begin[-1], WIDTH)), dtype=torch.float32).to(dtype).cuda()]
    inputs += [torch.tensor(rng.standard_normal((n, WIDTH)), dtype=torch.float32).to(dtype).cuda() for _ in range(steps)]

    def pass_over(run_prompt, run_token, check):
        now.copy_(torch.tensor(lengths, dtype=torch.int32))
        prompt.x.copy_(inputs[0])
        run_prompt()
        torch.cuda.synchronize()
        found = [prompt.seen.clone(), prompt.y.clone()]
        if check:
            prompt.check()
            want, lim = prompt_formula(prompt.q, prompt.k, prompt.v, begin, tol=bf16)
            assert ((prompt.seen.double() - want).abs() <= lim).all()
            held = [[kv8_model.Held(KVH, DIM) for _ in lengths] for _ in range(2)]
            for h, x in zip(held, (prompt.k, prompt.v)):
                for i, one_of in enumerate(h):
                    one_of.append(f64(x[begin[i]:begin[i + 1]]))
        for step in range(steps):
            token.positions.copy_(now)
            now.add_(1)
            token.x.copy_(inputs[1 + step])
            run_token()
            torch.cuda.synchronize()
            found += [token.seen.clone(), token.y.clone()]
            if not check:
                continue
            token.check()
            for h, x in zip(held, (token.k, token.v)):
                for i, one_of in enumerate(h):
                    one_of.append(f64(x[i:i + 1]))
            for i, m in enumerate(lengths):
                keys, values = held[0][i].values(), held[1][i].values()
                want, size = kv8_model.attention(f64(token.q[i:i + 1]), keys, values)
                lim = kv8_model.attention_bound(size, np.abs(values).max(), want, DIM, m + step + 1, bf16)
                assert (np.abs(f64(token.seen[i:i + 1]) - want) <= lim).all()
        return found

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def on_stream(s):
        with torch.cuda.stream(stream):
            s.run(stream.cuda_stream)

    eager = pass_over(lambda: on_stream(prompt), lambda: on_stream(token), True)
    graphs = []
    for s in (prompt, token):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            s.run(torch.cuda.current_stream().cuda_stream)
    for _ in range(2):
        for a, b in zip(eager, pass_over(graphs[0].replay, graphs[1].replay, False)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("window", [0, 50])
def test_a_prompt_and_the_cache_of_it_agree(cuda_ok, window, bf16):
    """Keys and values that 8 bits hold exactly: attention over the rows and over the cache of them are of the same numbers."""
    rng = np.random.default_rng(5)
    lengths, dtype = [70, 1, 200], torch.bfloat16 if bf16 else torch.float32
    begin = [0, 70, 71, 271]
    codes = torch.tensor(rng.integers(-127, 128, (271, 2 * KVH, DIM)), dtype=torch.float32, device="cuda")
    k, v = (codes / 64).to(dtype)[:, :KVH], (codes / 32).to(dtype)[:, KVH:]
    q = torch.tensor(rng.standard_normal((271, HEADS, DIM)), dtype=torch.float32).to(dtype).cuda()
    out = torch.empty_like(q)
    prompt_call(q, k, v, out, begin, bf16=bf16, window=window)()
    cache = Cache(KVH, DIM, lengths)
    cache.append(lengths, [k[a:b] for a, b in zip(begin, begin[1:])], [v[a:b] for a, b in zip(begin, begin[1:])])
    again, workspace = torch.empty_like(q), rt.Kv8Workspace(cache.kv)
    kind = rt.ROWS_BF16 if bf16 else rt.ROWS_F32
    cache.kv.attention(cache.batch(lengths, lengths), rt.kv8_query(q.data_ptr(), again.data_ptr(), kind, heads=HEADS, window=window),
                       workspace)
    torch.cuda.synchronize()
    got = cache.read(lengths)
    for i, (a, b) in enumerate(zip(begin, begin[1:])):
        assert np.array_equal(got[0][i], k[a:b].float().cpu().numpy()) and np.array_equal(got[1][i], v[a:b].float().cpu().numpy())
    want, lim = prompt_formula(q, k, v, begin, window, tol=bf16)
    assert ((out.double() - want).abs() <= lim).all()
    for a, b in zip(begin, begin[1:]):
        exact, size = kv8_model.attention(f64(q[a:b]), f64(k[a:b]), f64(v[a:b]), window)
        off = kv8_model.attention_bound(size, np.abs(f64(v[a:b])).max(), exact, DIM, b - a, bf16)
        assert (np.abs(f64(again[a:b]) - f64(out[a:b])) <= off + f64(lim[a:b])).all()


def test_offsets_past_32_bits(cuda_ok):
    """Operands whose rows lie more than 2^31 elements apart from the first to the last: the quantising pass and all of the
    product's kernels (few rows, whole tiles, a shared depth)."""
    rng = np.random.default_rng(6)
    depth, channels = 256, 160
    wide = 1 << 24
    big = torch.zeros(140, wide, dtype=torch.int8, device="cuda")      # 2.3 GB
    y_big = torch.zeros(140, wide, dtype=torch.bfloat16, device="cuda")  # 4.7 GB
    for rows in (130, 140):
        x, w, xs, ws = product_case(rng, rows, channels, depth)
        big[:rows, 4096:4096 + depth] = x
        x_far, y_far = big[:rows, 4096:4096 + depth], y_big[:rows, 160:160 + channels]
        rt.I8Product(x_far.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), y_far.data_ptr(), rows, channels, depth, rt.ROWS_BF16,
                     x_stride=wide, y_stride=wide)()
        torch.cuda.synchronize()
        check_product(y_far, *product_want(x, w, xs, ws, None), True)
    x, w, xs, ws = product_case(rng, 5, 140, depth)
    big[:140, :depth] = w
    for rows in (5, 40):
        x, _, xs, _ = product_case(rng, rows, 140, depth)
        y = torch.empty(rows, 140, device="cuda")
        rt.I8Product(x.data_ptr(), xs.data_ptr(), big.data_ptr(), ws.data_ptr(), y.data_ptr(), rows, 140, depth, w_stride=wide)()
        torch.cuda.synchronize()
        check_product(y, *product_want(x, w, xs, ws, None), False)
    x = torch.tensor(rng.standard_normal((140, 272)), dtype=torch.float32).to(torch.bfloat16).cuda()
    y_big[:, 1024:1296] = x
    scales = torch.empty(140, device="cuda")
    rt.QuantizeRows(y_big[:, 1024:].data_ptr(), big[:, 512:].data_ptr(), scales.data_ptr(), 140, 272, rt.ROWS_BF16, wide, wide)()
    torch.cuda.synchronize()
    want, s = quantized(f64(x))
    assert np.array_equal(f64(big[:, 512:784]), want) and np.array_equal(f64(scales), s)


def test_a_device_that_is_not_there(cuda_ok):
    a = torch.zeros(8192, device="cuda")
    p, device = a.data_ptr(), torch.cuda.device_count() + 7
    for c in (rt.QuantizeRows(p, p + 4096, p + 8192, 2, 32, device=device),
              rt.I8Product(p, p + 4096, p + 8192, p + 4096, p + 12288, 2, 16, 32, device=device),
              rt.PromptAttention(p, p + 4096, p + 8192, p + 12288, p, 1, 4, 4, 2, 1, 32, device=device)):
        with pytest.raises(rt.CudaError) as e:
            c()
        assert e.value.status == rt.DEVICE_ERROR
    torch.cuda.synchronize()
    assert (a == 0).all()
