"""The decode context on 8-bit K/V pages (PHONON_CUDA_KV_Q8).

Every layer of a step is held to the oracle given the same K/V values: the
device's pages are read back (exactly) right after the step, the row that the
step appended included, and the layer's output must agree within the
per-layer tolerance, as for the other K/V types (tests/parity.py). The
appended rows themselves must be the oracle's rounded to the page's scale."""
import numpy as np
import pytest

from phonon_b200 import runtime as rt
from phonon_b200 import synth

import kv8_model as model
import parity

pytestmark = pytest.mark.gpu
FINAL_TOL = 1e-3


def context(weights, n, pages, **kw):
    return rt.Context(weights, max_streams=n + 2, max_batch=n, pool_pages=pages, kv_type=rt.KV_Q8, **kw)


# 3: per-stage GEMVs; 5 and 40: tensor-core projections; 100: two lanes
@pytest.mark.parametrize("n", [1, 3, 5, 40, 100])
def test_layers_of_batched_steps(cuda_ok, oracle, weights12, n):
    steps = 3
    lens = [(17 * i) % 90 + (0 if i % 3 else 15) for i in range(n)]
    ctx = context(weights12, n, sum(x // 16 + 2 for x in lens) + 4)
    trace = parity.Trace(ctx, n)
    om = oracle.model(weights12)
    g = synth.Generator(88 + n)
    streams = []
    for i, length in enumerate(lens):
        s = ctx.stream_alloc(length + steps)
        if length:
            ctx.fill_synthetic(s, length, 300 + i)
        streams.append(s)
    stats = parity.Stats()
    checked = sorted({0, n // 2, n - 1})
    for t in range(steps):
        x = g.normal(n * 512).reshape(n, 512)
        pos = [length + t for length in lens]
        y, status = ctx.step(streams, pos, x, raise_on_status=False)
        assert not status.any()
        tr = trace.read(n)
        np.testing.assert_array_equal(tr[-1], y)
        for i in checked:
            parity.check_stream_oracle(ctx, om, streams[i], [pos[i]], [x[i]], [tr], i, stats, False, f"stream {i}")
    trace.close()
    ctx.close()
    print(stats)
    assert stats.rel < parity.PER_LAYER_TOL, stats


def test_appended_rows_are_the_fp32_rows_rounded(cuda_ok, weights12):
    """Layer 0's keys and values depend on the inputs alone: the fp32 context's rows, put through the 64-bit definition
    in the same pieces (a prefill, then single steps), are what the 8-bit context holds, bit for bit."""
    length, steps = 293, 25  # several prefill passes would need max_batch rows; here one pass and a partial page
    g = synth.Generator(4)
    rows = g.normal((length + steps) * 512).reshape(-1, 512)
    got = {}
    for kind in (rt.KV_F32, rt.KV_Q8):
        ctx = rt.Context(weights12[:2], max_streams=2, max_batch=4, pool_pages=40, kv_type=kind)
        ctx.set_batch_paths(1 << 20, rt.FUSED_MAX_BATCH, 1 << 20)
        ctx.set_cluster_step(0)
        s = ctx.stream_alloc(length + steps)
        ctx.append(s, rows[:length])
        for t in range(steps):
            ctx.step([s], [length + t], rows[length + t][None])
        got[kind] = ctx.kv_read(s, 0, length + steps, 0, 1)
        ctx.close()
    chunks = [256, length - 256] + [1] * steps  # a prefill pass is 256 rows
    for exact, held in zip(got[rt.KV_F32], got[rt.KV_Q8]):
        h, at = model.Held(8, 64), 0
        for n in chunks:
            h.append(exact[0, at:at + n].reshape(n, 8, 64))
            at += n
        np.testing.assert_array_equal(held[0].reshape(-1, 8, 64), h.values().astype(np.float32))


def test_prefill_output_given_its_pages(cuda_ok, oracle, weights12):
    length = 300
    ctx = context(weights12, 1, 24)
    s = ctx.stream_alloc(length)
    rows = synth.Generator(6).normal(length * 512).reshape(length, 512)
    last = ctx.append(s, rows)
    k, v = ctx.kv_read(s, 0, length)
    om = oracle.model(weights12)
    cache = om.new_stream(length)
    om.load_kv(cache, k, v)
    x = rows[-1]
    for layer in range(12):
        ok, x, _, _ = om.layer_step_forced(cache, layer, length - 1, x)
        assert ok
    om.free_stream(cache)
    ctx.close()
    assert rt.rel_err(last, x) < FINAL_TOL


def test_replayed_steps_equal_direct_ones(cuda_ok, weights12):
    """Repeated step shapes run as a graph; launches timed one by one do not. Same bits either way, across page and
    length-class boundaries."""
    n, steps = 6, 40
    lens = [0, 5, 14, 100, 250, 120]
    outs = []
    for direct in (False, True):
        ctx = context(weights12, n, 80)
        streams = [ctx.stream_alloc(400) for _ in range(n)]
        for i, (s, length) in enumerate(zip(streams, lens)):
            if length:
                ctx.fill_synthetic(s, length, i)
        ctx.profile(direct)
        g = synth.Generator(12)
        outs.append([ctx.step(streams, [x + t for x in lens], g.normal(n * 512).reshape(n, 512)) for t in range(steps)])
        if direct:
            prof = ctx.profile_read()
            assert prof["attention"]["launches"] == 12 * steps
        ctx.close()
    for a, b in zip(*outs):
        np.testing.assert_array_equal(a, b)


def test_pages_written_read_and_reused(cuda_ok, weights12):
    rng = np.random.default_rng(2)
    ctx = context(weights12[:3], 2, 4)
    s = ctx.stream_alloc(64)
    loud = 1e6 * rng.standard_normal((3, 64, 512)).astype(np.float32)
    ctx.kv_write(s, 0, loud, -loud)
    k, v = ctx.kv_read(s, 0, 64)
    for got, sign in ((k, 1), (v, -1)):
        for layer in range(3):
            h = model.Held(8, 64)
            h.append(sign * loud[layer].reshape(64, 8, 64))
            np.testing.assert_array_equal(got[layer].reshape(64, 8, 64), h.values().astype(np.float32))
    ctx.stream_free(s)
    # the same pages again, first written from the middle on: the old scales are gone
    s = ctx.stream_alloc(64)
    quiet = rng.standard_normal((2, 3, 512)).astype(np.float32)
    ctx.kv_write(s, 21, quiet, quiet, layer_begin=1)
    k, _ = ctx.kv_read(s, 21, 3, 1, 2)

    def units(rows):  # [layers][rows][512]: each head's scale, its maximum being in these rows
        e = [[model.exponent(np.abs(x).max()) for x in layer.reshape(-1, 8, 64).swapaxes(0, 1)] for layer in rows]
        return np.repeat(2.0 ** np.array(e), 64, 1)[:, None]

    assert (np.abs(k - quiet) <= units(quiet) / 2).all()
    more = 100 * rng.standard_normal((2, 1, 512)).astype(np.float32)
    ctx.kv_write(s, 24, more, more, layer_begin=1)  # raises the scale of rows 21..23
    k, _ = ctx.kv_read(s, 21, 4, 1, 2)
    wide = units(more)
    assert (np.abs(k[:, 3:] - more) <= wide / 2).all() and (np.abs(k[:, :3] - quiet) < wide).all()
    zeros, _ = ctx.kv_read(s, 48, 4)
    assert (zeros == 0).all()
    ctx.close()


def test_synthetic_fill_is_the_fp32_fill_rounded(cuda_ok, weights12):
    length = 50
    got = []
    for kind in (rt.KV_F32, rt.KV_Q8):
        ctx = rt.Context(weights12[:2], max_streams=2, max_batch=2, pool_pages=8, kv_type=kind)
        s = ctx.stream_alloc(64)
        ctx.fill_synthetic(s, length, 9)
        got.append(ctx.kv_read(s, 0, length))
        ctx.close()
    for exact, held in zip(*got):
        np.testing.assert_array_equal(held, (np.rint(exact.astype(np.float64) * 32) / 32).astype(np.float32))


def test_limits_failures_and_the_position_limit(cuda_ok, weights12):
    ctx = context(weights12, 3, 1030)
    assert ctx.set_cluster_step(rt.MAX_POSITIONS) == 0  # steps run per stage
    s = [ctx.stream_alloc(8192), ctx.stream_alloc(40), ctx.stream_alloc(40)]
    ctx.fill_synthetic(s[0], 8191, 5)
    x = synth.Generator(1).normal(3 * 512).reshape(3, 512)
    x[1, 7] = np.nan
    y, status = ctx.step(s, [8191, 0, 0], x, raise_on_status=False)
    assert status.tolist() == [rt.OK, rt.NON_FINITE, rt.OK] and np.isfinite(y[[0, 2]]).all()
    assert [ctx.length(q) for q in s] == [8192, 0, 1]
    calls = []
    with pytest.raises(rt.CudaError) as e:
        ctx.step([s[2]], [1], x[2:], cancel=lambda _: calls.append(1) or len(calls) > 4)
    assert e.value.status == rt.CANCELLED and ctx.length(s[2]) == 0
    ctx.close()
    with pytest.raises(rt.CudaError):
        rt.Context(weights12[:1], max_streams=1, max_batch=1, pool_pages=1, kv_type=3)


def test_frame_loop(cuda_ok, weights12):
    """The frame loop advances on 8-bit pages; its step is the context's step on the embedded latent."""
    import torch

    import heads
    n = 4
    outs = []
    for kind in (rt.KV_F32, rt.KV_Q8):
        ctx = rt.Context(weights12, max_streams=n, max_batch=n, pool_pages=32, kv_type=kind)
        h = rt.Head(ctx, heads.random_head(7), heads.random_frame(7))
        rng = np.random.default_rng(70)
        streams = [ctx.stream_alloc(64) for _ in range(n)]
        for i, s in enumerate(streams):
            ctx.fill_synthetic(s, 20 + i, i)
        state = torch.tensor(rng.standard_normal((n, 512)), dtype=torch.float32, device="cuda")
        cond = torch.tensor(0.5 * rng.standard_normal((n, 512)), dtype=torch.float32, device="cuda")
        raw = rng.standard_normal((n, 32)).astype(np.float32)
        logit, latent, status = h.frame_step(streams, [20 + i for i in range(n)], state.data_ptr(), cond.data_ptr(), raw, 0.8)
        assert not status.any() and [ctx.length(s) for s in streams] == [21 + i for i in range(n)]
        outs.append((logit, latent, state.cpu().numpy()))
        h.close()
        ctx.close()
    # what does not pass through the cache is the same; the new state is near
    np.testing.assert_array_equal(outs[0][0], outs[1][0])
    np.testing.assert_array_equal(outs[0][1], outs[1][1])
    assert np.isfinite(outs[1][2]).all()


def test_prefill_of_a_long_context(cuda_ok, oracle, weights12):
    """7400 positions, 256 rows a pass: the last passes are work enough for the 128-row attention in every layer."""
    length = 7400
    weights = weights12[:2]
    ctx = context(weights, 1, 256 * (length // 16 + 1))  # a pass lists its rows' pages, as many as the pool has
    s = ctx.stream_alloc(length)
    rows = synth.Generator(7).normal(length * 512).reshape(length, 512)
    last = ctx.append(s, rows)
    k, v = ctx.kv_read(s, 0, length)
    om = oracle.model(weights)
    cache = om.new_stream(length)
    om.load_kv(cache, k, v)
    x = rows[-1]
    for layer in range(2):
        ok, x, _, _ = om.layer_step_forced(cache, layer, length - 1, x)
        assert ok
    om.free_stream(cache)
    ctx.close()
    assert rt.rel_err(last, x) < FINAL_TOL


@pytest.mark.parametrize("n", [6, 40])
def test_prefills_and_steps_of_the_same_rows_take_turns(cuda_ok, weights12, n):
    """Prompts of n rows and steps of n streams have the same row count, buffers and length class: neither may replay the
    other's graph. Bit for bit what direct launches give."""
    outs = []
    for direct in (False, True):
        ctx = context(weights12[:3], n, 8 * (n + 2))
        ctx.profile(direct)
        g = synth.Generator(31)
        streams = [ctx.stream_alloc(64) for _ in range(n)]
        got = [ctx.append(s, g.normal(n * 512).reshape(n, 512)) for s in streams]
        got += [ctx.step(streams, [n + t] * n, g.normal(n * 512).reshape(n, 512)) for t in range(4)]
        more = [ctx.stream_alloc(64) for _ in range(2)]
        got += [ctx.append(s, g.normal(n * 512).reshape(n, 512)) for s in more]
        got += [ctx.step(streams, [n + 4 + t] * n, g.normal(n * 512).reshape(n, 512)) for t in range(3)]
        got += [x for s in streams + more for x in ctx.kv_read(s, 0, n + 7 if s in streams else n)]
        outs.append(got)
        ctx.close()
    for a, b in zip(*outs):
        np.testing.assert_array_equal(a, b)


def test_a_long_prefill_needs_no_more_pages_than_its_own(cuda_ok, oracle, weights12):
    """7000 positions in a pool of exactly their pages, in passes of 256 rows, then a step that takes none."""
    length = 7000
    weights = weights12[:2]
    ctx = context(weights, 1, length // 16 + 1)
    s = ctx.stream_alloc(length + 1)
    rows = synth.Generator(17).normal((length + 1) * 512).reshape(length + 1, 512)
    om = oracle.model(weights)
    for at in (length - 1, length):
        out = ctx.append(s, rows[:length]) if at < length else ctx.step([s], [at], rows[at][None])[0]
        cache = om.new_stream(at + 1)
        om.load_kv(cache, *ctx.kv_read(s, 0, at + 1))
        x = rows[at]
        for layer in range(2):
            ok, x, _, _ = om.layer_step_forced(cache, layer, at, x)
            assert ok
        om.free_stream(cache)
        assert rt.rel_err(out, x) < FINAL_TOL
    ctx.close()
