"""The operators around an evicting cache together, as a serving loop uses them, and how they are
called: under graph capture, on several streams and threads, with tensors past 4 GiB."""
import math
import threading

import numpy as np
import pytest

import cache_ops_ref as ref
import llm_hip
from helpers import from_dev_bf16, to_dev
from llm_hip import workloads
from test_gpu_cache_ops import assert_out, assert_rounded, assert_weights, bf16, f, heavy, split, view_bf16

pytestmark = pytest.mark.gpu

BT = 16


class Layer:
    """One layer's rows: norms, frequencies, and the fused projection of `n` tokens."""

    def __init__(self, Hq, Hkv, D, R, seed):
        self.Hq, self.Hkv, self.D, self.seed = Hq, Hkv, D, seed
        self.wq, self.wk = bf16(seed, D), bf16(seed + 1, D)
        self.freq = (1e4 ** (-np.arange(0, R, 2) / R)).astype(np.float32)
        self.dev = [view_bf16(self.wq), view_bf16(self.wk), to_dev(self.freq)]

    def rows(self, n, salt):
        return bf16(self.seed + 100 + salt, n, (self.Hq + 2 * self.Hkv) * self.D)

    def desc(self, ctx, t, pos):
        q, k, v = split(t, self.Hq, self.Hkv, self.D)
        return ctx.qk_rope_desc(q, k, v, pos, self.dev[2], q_weight=self.dev[0], k_weight=self.dev[1])

    def expect(self, rows, pos):
        """(queries, keys, values) of the rows in 64 bits, unrounded."""
        Hq, Hkv, D = self.Hq, self.Hkv, self.D
        x = f(rows).astype(np.float64)
        q = ref.norm_rope(x[:, :Hq * D].reshape(-1, Hq, D), pos, self.freq, f(self.wq))
        k = ref.norm_rope(x[:, Hq * D:(Hq + Hkv) * D].reshape(-1, Hkv, D), pos, self.freq, f(self.wk))
        return q, k, x[:, (Hq + Hkv) * D:].reshape(-1, Hkv, D)


@pytest.mark.parametrize("fmt", ref.FMTS)
@pytest.mark.parametrize("Hq,Hkv,D,R", [(16, 8, 128, 128), (16, 2, 256, 64), (4, 2, 64, 32)])
def test_serving_loop(ctx, fmt, Hq, Hkv, D, R):
    """Prompts enter the cache, their last rows observe them, decode steps accumulate, the caches are cut
    to a budget and decoding goes on at positions that are no longer slots.  Every step is checked
    on what the GPU holds: the pool's rows, the queries it made and the weights before it."""
    import torch

    layer = Layer(Hq, Hkv, D, R, 7)
    F, scale = ref.FMTS[fmt], 1.0 / math.sqrt(D)
    prompts, budget, sinks, recent, steps = [70, 33, 150], 48, 2, 16, 3
    B, stride, observe = len(prompts), 256, 5
    nb = [-(-(p + 8) // BT) for p in prompts]
    per = -(-(budget + 8) // BT)
    n_blocks = sum(nb) + B * per + 3
    perm = np.random.default_rng(3).permutation(n_blocks)
    pool = ctx.pool(F, BT, Hkv, D, n_blocks)
    tables = np.full((B, max(nb)), -1, np.int32)
    at = 0
    for b, k in enumerate(nb):
        tables[b, :k] = perm[at:at + k]
        at += k
    dst = np.array(perm[at:at + B * per], np.int32).reshape(B, per)

    def enter(tables, slots_of, pos, rows, q_out):
        slots = np.array([int(tables[b, s // BT]) * BT + s % BT for b, s in slots_of], np.int64)
        keep = [view_bf16(rows), to_dev(np.array(pos, np.int32)), to_dev(slots)]
        ctx.qk_norm_rope_append(pool, layer.desc(ctx, keep[0], keep[1]), keep[2], q_out)
        torch.cuda.synchronize()
        want, k, v = layer.expect(rows, pos)
        assert_rounded(from_dev_bf16(q_out.view(torch.int16)), want, np.abs(want).max(-1, keepdims=True), "queries")
        if fmt in ("bf16", "f16"):
            arr = ref.pool_arrays(pool)
            got = arr["k"][slots // BT, :, slots % BT]
            got = f(got) if fmt == "bf16" else got.view(np.float16).astype(np.float32)
            # the fp16 pool's second rounding: 2^-11 of the value
            assert (np.abs(got - k) <= np.abs(k) * (2.0**-8 + 2.0**-11) + np.abs(k).max() * 2.0**-18).all()
        return from_dev_bf16(q_out.view(torch.int16))

    def check_attention(tables, lens, q, rows, out, before, after, decay):
        at = 0
        for b, n in enumerate(lens):
            k, v, live = ref.cached(pool, F, BT, Hkv, D, n_blocks, tables[b], n)
            o, acc = ref.attend(f(q[at:at + rows[b]]).astype(np.float64), k, v, live, scale)
            assert_out(out[at:at + rows[b]], o, f"sequence {b}")
            assert_weights(after[b, :, :n], before[b, :, :n] * np.float64(np.float32(decay)) + acc, f"sequence {b}")
            assert np.array_equal(after[b, :, n:], before[b, :, n:])
            at += rows[b]

    weights = torch.zeros((B, Hkv, stride), device="cuda")
    # prompts, observed by their last rows
    rows = layer.rows(sum(prompts), 0)
    q_out = torch.empty((sum(prompts), Hq, D), dtype=torch.bfloat16, device="cuda")
    pos = np.concatenate([np.arange(p) for p in prompts])
    q = enter(tables, [(b, s) for b, p in enumerate(prompts) for s in range(p)], pos, rows, q_out)
    ends = np.cumsum(prompts)
    last = np.concatenate([np.arange(e - observe, e) for e in ends])
    qo = q_out[torch.from_numpy(last).cuda()].contiguous()
    out = torch.empty_like(qo)
    starts = to_dev((np.arange(B + 1) * observe).astype(np.int32))
    d_lens, d_tables = to_dev(np.array(prompts, np.int32)), to_dev(tables)
    ctx.paged_prefill_weights(pool, ctx.prefill_desc(starts, d_lens, d_tables, Hq, observe), max(prompts), qo, out, scale,
                              None, weights)
    torch.cuda.synchronize()
    check_attention(tables, prompts, q[last], [observe] * B, from_dev_bf16(out.view(torch.int16)),
                    np.zeros((B, Hkv, stride)), weights.cpu().numpy(), 1.0)

    def decode(tables, lens, positions, salt, weights):
        """One token for each sequence, at slot lens[b] and its own position."""
        rows = layer.rows(B, salt)
        q_out = torch.empty((B, Hq, D), dtype=torch.bfloat16, device="cuda")
        q = enter(tables, [(b, n) for b, n in enumerate(lens)], positions, rows, q_out)
        lens = [n + 1 for n in lens]
        before = weights.clone()
        out = torch.empty_like(q_out)
        keep = [to_dev(np.array(lens, np.int32)), to_dev(tables)]
        d = ctx.decode_desc(keep[0], keep[1], Hq, max(lens))
        ctx.paged_decode_weights(pool, d, q_out, out, scale, weights, weights, 0.9)
        torch.cuda.synchronize()
        check_attention(tables, lens, q, [1] * B, from_dev_bf16(out.view(torch.int16)), before.cpu().numpy(),
                        weights.cpu().numpy(), 0.9)
        return lens

    lens, positions = list(prompts), list(prompts)
    for s in range(steps):
        lens = decode(tables, lens, positions, 1 + s, weights)
        positions = [p + 1 for p in positions]
    # cut
    keep = torch.full((B, Hkv, budget), -1, dtype=torch.int32, device="cuda")
    kept = torch.zeros(B, dtype=torch.int32, device="cuda")
    d_lens, d_tables, d_dst = to_dev(np.array(lens, np.int32)), to_dev(tables), to_dev(dst)
    ctx.kv_select(ctx.select_desc(d_lens, Hkv, max(lens), budget, sinks, recent, stride, budget), weights, keep, kept)
    fresh = torch.zeros_like(weights)
    before = ref.pool_arrays(pool)
    ctx.kv_compact(pool, ctx.compact_desc(d_lens, kept, keep, d_tables, d_dst, budget, weights, fresh))
    torch.cuda.synchronize()
    host_w, host_keep = weights.cpu().numpy(), keep.cpu().numpy()
    n_kept = [min(n, budget) for n in lens]
    assert kept.tolist() == n_kept
    for b, n in enumerate(lens):
        for h in range(Hkv):
            want = ref.select(host_w[b, h], n, budget, sinks, recent)
            assert np.array_equal(host_keep[b, h, :n_kept[b]], want)
            assert np.array_equal(fresh[b, h, :n_kept[b]].cpu().numpy(), host_w[b, h, want])
    want = ref.compact(before, F, BT, host_keep, n_kept, tables, dst)
    got = ref.pool_arrays(pool)
    for key in want:
        assert np.array_equal(got[key], want[key]), key
    # on from there: new tokens behind the kept ones, at the positions that follow
    lens = n_kept
    for s in range(steps):
        lens = decode(dst, lens, positions, 10 + s, fresh)
        positions = [p + 1 for p in positions]
    assert ctx.device_errors() == 0, ctx.last_error()


class Step:
    """A decode step, selection and compaction over one pool, with everything it needs."""

    def __init__(self, ctx, lens, Hq, Hkv, D, budget, seed, fmt=llm_hip.KV_BF16, long=0):
        import torch

        self.ctx, self.D, self.budget = ctx, D, budget
        lens = np.array(lens, np.int32)
        B = lens.size
        batch = workloads.paged_batch(lens, BT, 0.1, seed)
        per = -(-budget // BT)
        n = batch.n_blocks + B * per
        self.pool = ctx.pool(fmt, BT, Hkv, D, n)
        ctx.write_blocks(self.pool, to_dev(np.arange(n, dtype=np.int32)), to_dev(bf16(seed, n, BT, Hkv, D)),
                         to_dev(bf16(seed + 1, n, BT, Hkv, D)))
        self.lens, self.tables = to_dev(lens), to_dev(batch.tables)
        self.dst = to_dev((batch.n_blocks + np.arange(B * per, dtype=np.int32)).reshape(B, per))
        self.first_dst = batch.n_blocks
        stride = int(lens.max())
        self.layer = Layer(Hq, Hkv, D, D, seed + 2)
        self.rows = view_bf16(self.layer.rows(B, 0))
        self.pos = self.lens - 1
        last = lens.astype(np.int64) - 1
        self.slots = to_dev(batch.tables[np.arange(B), last // BT].astype(np.int64) * BT + last % BT)
        self.rope = self.layer.desc(ctx, self.rows, self.pos)
        self.q = torch.zeros((B, Hq, D), dtype=torch.bfloat16, device="cuda")
        self.out = torch.zeros_like(self.q)
        self.w_in = to_dev(heavy(seed, B, Hkv, stride).astype(np.float32))
        self.w = torch.zeros_like(self.w_in)
        self.w_kept = torch.zeros((B, Hkv, budget), device="cuda")
        self.keep = torch.zeros((B, Hkv, budget), dtype=torch.int32, device="cuda")
        self.kept = torch.zeros(B, dtype=torch.int32, device="cuda")
        self.decode = ctx.decode_desc(self.lens, self.tables, Hq, int(lens.max()))
        self.select = ctx.select_desc(self.lens, Hkv, int(lens.max()), budget, 1, budget // 4, stride, budget)
        self.compact = ctx.compact_desc(self.lens, self.kept, self.keep, self.tables, self.dst, budget, self.w, self.w_kept)
        self.long = long  # positions of a further selection in tiles
        if long:
            self.lw = to_dev(heavy(seed + 3, 1, 2, long).astype(np.float32))
            self.llens = to_dev(np.array([long], np.int32))
            self.lkeep = torch.zeros((1, 2, 64), dtype=torch.int32, device="cuda")
            self.lkept = torch.zeros(1, dtype=torch.int32, device="cuda")
            self.lselect = ctx.select_desc(self.llens, 2, long, 64, 0, 8, long, 64)

    def run(self, stream=None):
        c = self.ctx
        c.qk_norm_rope_append(self.pool, self.rope, self.slots, self.q, stream)
        c.paged_decode_weights(self.pool, self.decode, self.q, self.out, 1.0 / math.sqrt(self.D), self.w_in, self.w, 0.9,
                               stream)
        c.kv_select(self.select, self.w, self.keep, self.kept, stream)
        c.kv_compact(self.pool, self.compact, stream)
        if self.long:
            c.kv_select(self.lselect, self.lw, self.lkeep, self.lkept, stream)

    def outputs(self):
        t = [self.q, self.out, self.w, self.keep, self.kept, self.w_kept]
        return t + ([self.lkeep, self.lkept] if self.long else [])

    def snapshot(self):
        import torch

        torch.cuda.synchronize()
        return [x.clone() for x in self.outputs()] + [self.pool.raw()]

    def clear(self):
        for x in self.outputs():
            x.zero_()

    def assert_same(self, want, what):
        import torch

        got = self.snapshot()
        for x, y in zip(got[:-1], want[:-1]):
            assert torch.equal(x.view(torch.int16) if x.dtype == torch.bfloat16 else x,
                               y.view(torch.int16) if y.dtype == torch.bfloat16 else y), what
        for key in want[-1]:
            assert np.array_equal(got[-1][key], want[-1][key]), (what, key)


@pytest.mark.parametrize("fmt", [llm_hip.KV_BF16, llm_hip.KV_INT8])
def test_captured_and_replayed(ctx, fmt):
    """A captured step replays to the eager step's bits, between eager calls, and after a larger call on
    the stream has taken a larger scratch; capture without the scratch is refused."""
    import torch

    step = Step(ctx, [300, 17, 900], 16, 8, 128, 64, 11, fmt, long=40000)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        # nothing reserved: refused under capture, and the capture goes on
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step.q.zero_()
            with pytest.raises(llm_hip.LlhError) as e:
                ctx.paged_decode_weights(step.pool, step.decode, step.q, step.out, 0.1, step.w_in, step.w)
            assert e.value.status == llm_hip.ERR_CAPACITY
    need = max(ctx.weights_workspace_bytes(3, 1, 16, 128, 900), ctx.select_workspace_bytes(1, 2, 40000),
               ctx.qk_rope_workspace_bytes(3, 8, 128))
    ctx.reserve_ops_workspace(need, s)
    held = ctx.metrics()["workspace_bytes"]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        step.run(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step.run()
    want = step.snapshot()
    assert ctx.metrics()["workspace_bytes"] == held
    other = Step(ctx, [5000, 3000], 32, 4, 128, 100, 12, long=300000)
    for i in range(4):
        with torch.cuda.stream(s):
            step.clear()
            graph.replay()
        step.assert_same(want, f"replay {i}")
        with torch.cuda.stream(s):
            step.run()
        step.assert_same(want, f"eager {i}")
        if i >= 1:
            with torch.cuda.stream(s):
                other.run()
                other.run()
            torch.cuda.synchronize()
    assert ctx.metrics()["workspace_bytes"] > held
    assert ctx.device_errors() == 0, ctx.last_error()
    ctx.release_stream(s)


def test_streams_and_threads(ctx):
    """Two threads on streams of their own, many steps at once: each stream's scratch is its own."""
    import torch

    steps = [Step(ctx, [300, 17, 900], 16, 8, 128, 64, 21, long=40000), Step(ctx, [1200, 44], 16, 2, 256, 96, 22)]
    want = []
    for st in steps:
        st.run()
        want.append(st.snapshot())
        st.clear()
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    errors = []

    def worker(st, s):
        try:
            for _ in range(50):
                st.run(s)
        except Exception as e:  # pragma: no cover
            errors.append(repr(e))

    threads = [threading.Thread(target=worker, args=a) for a in zip(steps, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=100)
    assert not errors, errors
    for st, w in zip(steps, want):
        st.assert_same(w, "threads")
    assert ctx.device_errors() == 0, ctx.last_error()
    for s in streams:
        ctx.release_stream(s)


def test_one_stream_from_two_threads(ctx):
    """Calls of two threads on one stream take turns at its scratch."""
    import torch

    steps = [Step(ctx, [300, 900], 16, 8, 128, 64, 31), Step(ctx, [700], 16, 2, 256, 96, 32)]
    want = []
    for st in steps:
        st.run()
        want.append(st.snapshot())
        st.clear()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    errors = []

    def worker(st):
        try:
            for _ in range(50):
                st.run(s)
        except Exception as e:  # pragma: no cover
            errors.append(repr(e))

    threads = [threading.Thread(target=worker, args=(st,)) for st in steps]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=100)
    assert not errors, errors
    for st, w in zip(steps, want):
        st.assert_same(w, "one stream")
    ctx.release_stream(s)


def test_per_thread_stream_is_refused(ctx):
    """hipStreamPerThread is another stream in every thread: calls that keep scratch refuse it."""
    import torch

    step = Step(ctx, [300], 16, 8, 128, 64, 41, llm_hip.KV_INT8, long=40000)
    for call in (lambda: ctx.paged_decode_weights(step.pool, step.decode, step.q, step.out, 0.1, None, step.w, stream=2),
                 lambda: ctx.kv_select(step.lselect, step.lw, step.lkeep, step.lkept, stream=2),
                 lambda: ctx.qk_norm_rope_append(step.pool, step.rope, step.slots, step.q, stream=2)):
        with pytest.raises(llm_hip.LlhError) as e:
            call()
        assert e.value.status == llm_hip.ERR_UNSUPPORTED
    torch.cuda.synchronize()


def test_tensors_past_four_gib(ctx):
    """Blocks whose rows lie past 4 GiB in the pool, and accumulators whose rows lie 2.4 GB apart."""
    import torch

    Hq, Hkv, D, n = 16, 8, 128, 140000  # 4.6 GB of K and of V
    pool = ctx.pool(llm_hip.KV_BF16, BT, Hkv, D, n)
    lens = np.array([200, 130], np.int32)
    src = np.array([[n - 1 - 2 * i - b for i in range(13)] for b in range(2)], np.int32)
    dst = np.array([[n - 100 - 2 * i - b for i in range(4)] for b in range(2)], np.int32)
    layer = Layer(Hq, Hkv, D, D, 51)
    rows, pos = layer.rows(330, 0), np.concatenate([np.arange(200), np.arange(130)])
    slots = np.array([int(src[b, s // BT]) * BT + s % BT for b, m in enumerate(lens) for s in range(m)], np.int64)
    assert slots.max() * Hkv * D * 2 > 1 << 32
    keep_alive = [view_bf16(rows), to_dev(pos.astype(np.int32)), to_dev(slots)]
    q_out = torch.empty((330, Hq, D), dtype=torch.bfloat16, device="cuda")
    ctx.qk_norm_rope_append(pool, layer.desc(ctx, keep_alive[0], keep_alive[1]), keep_alive[2], q_out)
    k_out = torch.empty((330, Hkv, D), device="cuda")
    v_out = torch.empty_like(k_out)
    ctx.export_rows_f32(pool, keep_alive[2], k_out, v_out)
    _, k, v = layer.expect(rows, pos)
    assert (np.abs(k_out.cpu().numpy() - k) <= np.abs(k) * 2.0**-8 + np.abs(k).max() * 2.0**-18).all()
    assert np.array_equal(v_out.cpu().numpy(), v.astype(np.float32))
    stride = 600_000_000
    last = torch.tensor([199, 329], device="cuda")
    q = q_out[last].contiguous()
    out = torch.empty_like(q)
    weights = torch.empty((2, Hkv, 256), device="cuda")
    d_lens, d_src, d_dst = to_dev(lens), to_dev(src), to_dev(dst)
    ctx.paged_decode_weights(pool, ctx.decode_desc(d_lens, d_src, Hq, 200), q, out, 1.0 / math.sqrt(D), None, weights)
    torch.cuda.synchronize()
    hk, hv = k_out.cpu().numpy().astype(np.float64), v_out.cpu().numpy().astype(np.float64)
    for b, (a, m) in enumerate([(0, 200), (200, 130)]):
        o, acc = ref.attend(q[b:b + 1].float().cpu().numpy().astype(np.float64), hk[a:a + m], hv[a:a + m],
                            np.ones(m, bool), 1.0 / math.sqrt(D))
        assert_out(from_dev_bf16(out[b:b + 1].contiguous().view(torch.int16)), o, f"sequence {b}")
        assert_weights(weights[b, :, :m].cpu().numpy(), acc, f"sequence {b}")
    # rows of an accumulator 2.4 GB apart: selection from the last ones, and their move
    far = torch.empty((1, 4, stride), device="cuda")
    far[0, :, :200] = weights[0, :4, :200]
    near = weights[:1, :4].contiguous()
    keeps = []
    for x, st in ((far, stride), (near, 256)):
        keep = torch.zeros((1, 4, 64), dtype=torch.int32, device="cuda")
        kept = torch.zeros(1, dtype=torch.int32, device="cuda")
        ctx.kv_select(ctx.select_desc(d_lens[:1].contiguous(), 4, 200, 64, 2, 16, st, 64), x, keep, kept)
        keeps.append(keep)
    torch.cuda.synchronize()
    assert torch.equal(*keeps)
    del far
    keep = torch.zeros((2, Hkv, 64), dtype=torch.int32, device="cuda")
    kept = torch.zeros(2, dtype=torch.int32, device="cuda")
    moved = torch.zeros((2, Hkv, 64), device="cuda")
    ctx.kv_select(ctx.select_desc(d_lens, Hkv, 200, 64, 2, 16, 256, 64), weights, keep, kept)
    ctx.kv_compact(pool, ctx.compact_desc(d_lens, kept, keep, d_src, d_dst, 64, weights, moved))
    at = np.array([int(dst[b, s // BT]) * BT + s % BT for b in range(2) for s in range(64)], np.int64)
    k2, v2 = torch.empty((128, Hkv, D), device="cuda"), torch.empty((128, Hkv, D), device="cuda")
    ctx.export_rows_f32(pool, to_dev(at), k2, v2)
    torch.cuda.synchronize()
    assert ctx.device_errors() == 0
    hkeep = keep.cpu().numpy()
    for b in range(2):
        for h in range(Hkv):
            p = hkeep[b, h] + (0, 200)[b]
            assert np.array_equal(k2[64 * b:64 * b + 64, h].cpu().numpy(), hk[p, h].astype(np.float32))
            assert np.array_equal(v2[64 * b:64 * b + 64, h].cpu().numpy(), hv[p, h].astype(np.float32))
    pool.close()
