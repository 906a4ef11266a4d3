"""The operators around an evicting cache on the GPU, against their formulas in 64 bits
(cache_ops_ref): norms and rotation of queries and keys, attention that accumulates its weights,
the selection of the tokens to keep, and their move."""
import math

import numpy as np
import pytest

import cache_ops_ref as ref
import llm_hip
import oracle
from cache_ops_ref import FMTS
from helpers import from_dev_bf16, to_dev
from llm_hip import workloads
from test_gpu_decode import build_case

pytestmark = pytest.mark.gpu

BT = 16
ALL_FMTS = dict(FMTS, int8_row=llm_hip.KV_INT8_ROW)


def bf16(seed, *shape):
    return oracle.normal_bf16(seed, int(np.prod(shape))).reshape(shape)


def f(x):
    return oracle.bf16_to_f32(np.ascontiguousarray(x).ravel()).reshape(x.shape)


def view_bf16(a):
    import torch

    return to_dev(a).view(torch.bfloat16)


# ---------------------------------------------------------------------------
# norms and rotation
# ---------------------------------------------------------------------------
def rope_case(n, Hq, Hkv, D, R, seed, far=1 << 20, pad=0):
    """A fused projection's rows (with `pad` elements behind each token), weights, positions."""
    qkv = bf16(seed, n, (Hq + 2 * Hkv) * D + pad)
    wq, wk = bf16(seed + 1, D), bf16(seed + 2, D)
    pos = np.random.default_rng(seed).integers(0, far, size=n).astype(np.int32)
    freq = (1e6 ** (-np.arange(0, R, 2) / max(R, 1))).astype(np.float32)
    return qkv, wq, wk, pos, freq


def split(t, Hq, Hkv, D):
    n = t.shape[0]
    q, k, v = t[:, :Hq * D], t[:, Hq * D:(Hq + Hkv) * D], t[:, (Hq + Hkv) * D:(Hq + 2 * Hkv) * D]
    return q.unflatten(1, (Hq, D)), k.unflatten(1, (Hkv, D)), v.unflatten(1, (Hkv, D))


def assert_rounded(got, want, scale, what):
    """bf16's half step (2^-8 of the value), and for the f32 arithmetic before it 2^-18 of the row's
    largest element: the sum of D squares, the root and three products lose under (D / 64 + 8) 2^-24,
    the sine and cosine of an angle held to 2^-25 turns under 2^-20."""
    bad = ~(np.abs(f(got) - want) <= np.abs(want) * 2.0**-8 + scale * 2.0**-18)
    assert not bad.any(), f"{what}: {bad.sum()} of {want.size}, worst {np.abs(f(got) - want)[bad].max():.3e}"


ROPES = [
    # n, Hq, Hkv, D, R, adjacent, offset, pad
    (1, 16, 8, 128, 128, False, 0.0, 0),
    (5, 16, 8, 128, 64, False, 1.0, 0),
    (3, 32, 4, 128, 128, True, 0.0, 8),
    (17, 16, 2, 256, 64, False, 1.0, 0),
    (4, 8, 4, 256, 256, True, 0.0, 0),
    (2, 8, 4, 256, 128, False, 0.0, 16),
    (3, 3, 1, 128, 16, False, 0.0, 0),
    (3, 3, 1, 128, 112, False, 0.0, 0),
    (3, 5, 1, 128, 2, False, 0.0, 0),
    (3, 5, 1, 128, 6, True, 0.0, 0),
    (2, 2, 2, 256, 0, False, 0.0, 0),
    (7, 4, 2, 64, 64, False, 0.0, 0),
    (3, 3, 3, 80, 80, False, 0.0, 1),
    (2, 5, 1, 96, 24, True, 1.0, 3),
    (2, 1, 1, 512, 512, False, 0.0, 0),
    (2, 1, 1, 7, 6, False, 0.0, 0),
    (2, 2, 1, 1, 0, False, 0.0, 0),
]


@pytest.mark.parametrize("n,Hq,Hkv,D,R,adjacent,offset,pad", ROPES)
def test_norm_rope(ctx, n, Hq, Hkv, D, R, adjacent, offset, pad):
    import torch

    qkv, wq, wk, pos, freq = rope_case(n, Hq, Hkv, D, R, 10 + D + R, pad=pad)
    t = view_bf16(qkv)
    q, k, _ = split(t, Hq, Hkv, D)
    dev = [view_bf16(wq), view_bf16(wk), to_dev(pos), to_dev(freq)]
    for weights in (True, False):
        d = ctx.qk_rope_desc(q, k, None, dev[2], dev[3] if R else None, q_weight=dev[0] if weights else None,
                             k_weight=dev[1] if weights else None, weight_offset=offset, adjacent=adjacent)
        qo = torch.full((n, Hq, D), math.nan, dtype=torch.bfloat16, device="cuda")
        ko = torch.full((n, Hkv, D), math.nan, dtype=torch.bfloat16, device="cuda")
        ctx.qk_norm_rope(d, qo, ko)
        torch.cuda.synchronize()
        assert ctx.device_errors() == 0
        for name, out, x, w in (("q", qo, q, wq), ("k", ko, k, wk)):
            want = ref.norm_rope(x.float().cpu().numpy(), pos, freq, f(w) if weights else None, offset, 1e-6, adjacent)
            top = np.abs(want).max(-1, keepdims=True)
            assert_rounded(from_dev_bf16(out.view(torch.int16)), want, top, f"{name}, weights {weights}")


def test_norm_rope_far_positions_and_extremes(ctx):
    """The largest positions keep their angles; a zero row stays zero; rows near bf16's largest
    value overflow the sum of squares, as the formula in f32 does."""
    import torch

    n, D = 6, 128
    qkv, wq, _, pos, freq = rope_case(n, 2, 1, D, D, 77)
    pos[:] = [0, 1, 2**31 - 1, 2**31 - 2, 10**9 + 7, 131071]
    x = qkv[:, :2 * D].reshape(n, 2, D).copy()
    x[1] = 0
    t, k = view_bf16(x), view_bf16(np.ascontiguousarray(x[:, :1]))
    dev = [view_bf16(wq), to_dev(pos), to_dev(freq)]
    qo, ko = torch.empty_like(t), torch.empty_like(k)
    ctx.qk_norm_rope(ctx.qk_rope_desc(t, k, None, dev[1], dev[2], q_weight=dev[0], k_weight=dev[0]), qo, ko)
    want = ref.norm_rope(f(x), pos, freq, f(wq))
    top = np.abs(want).max(-1, keepdims=True)
    assert_rounded(from_dev_bf16(qo.view(torch.int16)), want, top, "far")
    assert (qo[1] == 0).all()


def test_norm_rope_in_place(ctx):
    import torch

    for D, Hq, Hkv in [(128, 16, 8), (256, 16, 2), (64, 4, 2)]:
        qkv, wq, wk, pos, freq = rope_case(9, Hq, Hkv, D, D, 5)
        q = view_bf16(np.ascontiguousarray(qkv[:, :Hq * D])).view(9, Hq, D)
        k = view_bf16(np.ascontiguousarray(qkv[:, Hq * D:(Hq + Hkv) * D])).view(9, Hkv, D)
        dev = [view_bf16(wq), view_bf16(wk), to_dev(pos), to_dev(freq)]
        d = ctx.qk_rope_desc(q, k, None, dev[2], dev[3], q_weight=dev[0], k_weight=dev[1])
        qo, ko = torch.empty_like(q), torch.empty_like(k)
        ctx.qk_norm_rope(d, qo, ko)
        ctx.qk_norm_rope(d, q, k)
        assert torch.equal(q.view(torch.int16), qo.view(torch.int16))
        assert torch.equal(k.view(torch.int16), ko.view(torch.int16))


@pytest.mark.parametrize("n,Hq,Hkv,D,R,adjacent", [
    # prompts, whose workgroups take several heads of their tokens: odd counts, both pairings
    (1037, 16, 8, 128, 128, False), (1024, 5, 1, 128, 128, True), (1041, 32, 4, 128, 64, False),
    (1029, 3, 1, 128, 2, True), (1037, 16, 2, 256, 64, False), (1025, 9, 2, 256, 256, True), (1031, 4, 2, 64, 64, False),
    # more heads than a workgroup's wavefronts load at once
    (5, 64, 8, 128, 128, False), (2, 96, 96, 128, 64, True), (3, 40, 8, 256, 64, False), (2, 64, 2, 256, 256, True),
])
@pytest.mark.parametrize("off", [0, 1])
def test_norm_rope_many_rows(ctx, n, Hq, Hkv, D, R, adjacent, off):
    """Against the formula, written elsewhere and over the input; off: outputs off their 16 bytes."""
    import torch

    qkv, wq, wk, pos, freq = rope_case(n, Hq, Hkv, D, R, 31 + D + n)
    t = view_bf16(qkv)
    q, k, _ = split(t, Hq, Hkv, D)
    dev = [view_bf16(wq), view_bf16(wk), to_dev(pos), to_dev(freq)]
    d = ctx.qk_rope_desc(q, k, None, dev[2], dev[3], q_weight=dev[0], k_weight=dev[1], adjacent=adjacent)
    outs = [torch.full((n * H * D + 2,), math.nan, dtype=torch.bfloat16, device="cuda") for H in (Hq, Hkv)]
    qo, ko = (o[off:off + n * H * D].view(n, H, D) for o, H in zip(outs, (Hq, Hkv)))
    ctx.qk_norm_rope(d, qo, ko)
    torch.cuda.synchronize()
    assert ctx.device_errors() == 0
    for name, out, x, w in (("q", qo, q, wq), ("k", ko, k, wk)):
        want = ref.norm_rope(x.float().cpu().numpy(), pos, freq, f(w), 0.0, 1e-6, adjacent)
        top = np.abs(want).max(-1, keepdims=True)
        assert_rounded(from_dev_bf16(out.contiguous().view(torch.int16)), want, top, name)
    for o, H in zip(outs, (Hq, Hkv)):  # nothing beside the rows
        assert o[:off].isnan().all() and o[off + n * H * D:].isnan().all()
    if off == 0:
        qc, kc = q.contiguous(), k.contiguous()
        ctx.qk_norm_rope(ctx.qk_rope_desc(qc, kc, None, dev[2], dev[3], q_weight=dev[0], k_weight=dev[1],
                                          adjacent=adjacent), qc, kc)
        assert torch.equal(qc.view(torch.int16), qo.view(torch.int16))
        assert torch.equal(kc.view(torch.int16), ko.view(torch.int16))


def fresh_pool(ctx, fmt, bt, hkv, d, n, seed):
    """A pool whose blocks all hold rows."""
    pool = ctx.pool(fmt, bt, hkv, d, n)
    ctx.write_blocks(pool, to_dev(np.arange(n, dtype=np.int32)), to_dev(bf16(seed, n, bt, hkv, d)),
                     to_dev(bf16(seed + 1, n, bt, hkv, d)))
    return pool


@pytest.mark.parametrize("fmt", ALL_FMTS)
@pytest.mark.parametrize("Hq,Hkv,D,bt,pad", [(16, 8, 128, 16, 0), (16, 2, 256, 16, 0), (4, 2, 64, 16, 0),
                                             (4, 1, 128, 8, 0), (16, 8, 128, 16, 4), (3, 1, 256, 16, 1)])
def test_norm_rope_append_is_the_two_calls(ctx, fmt, Hq, Hkv, D, bt, pad):
    """Whole blocks, a run that starts inside a block, scattered slots, and a block filled backwards:
    the same bytes in the pool, everywhere, and the same queries."""
    import torch

    whole = np.arange(3 * bt, 5 * bt)
    inside = np.arange(6 * bt + 3, 8 * bt + 5)
    scattered = np.array([9 * bt + 1, 2 * bt, 11 * bt - 1, 0])
    slots = np.concatenate([whole, inside, scattered, np.arange(13 * bt - 1, 12 * bt - 1, -1)]).astype(np.int64)
    n = slots.size
    qkv, wq, wk, pos, freq = rope_case(n, Hq, Hkv, D, D, 3, pad=pad)
    t = view_bf16(qkv)
    q, k, v = split(t, Hq, Hkv, D)
    dev = [view_bf16(wq), view_bf16(wk), to_dev(pos), to_dev(freq), to_dev(slots)]
    d = ctx.qk_rope_desc(q, k, v, dev[2], dev[3], q_weight=dev[0], k_weight=dev[1])
    one, two = (fresh_pool(ctx, ALL_FMTS[fmt], bt, Hkv, D, 14, 90) for _ in range(2))
    q1, q2 = (torch.full((n, Hq, D), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    k2 = torch.empty((n, Hkv, D), dtype=torch.bfloat16, device="cuda")
    ctx.qk_norm_rope_append(one, d, dev[4], q1)
    ctx.qk_norm_rope(d, q2, k2)
    ctx.append(two, dev[4], k2, v.contiguous())
    torch.cuda.synchronize()
    assert ctx.device_errors() == 0
    assert torch.equal(q1.view(torch.int16), q2.view(torch.int16))
    a, b = one.raw(), two.raw()
    for key in a:
        assert np.array_equal(a[key], b[key]), key


@pytest.mark.parametrize("fmt", ["bf16", "f16", "int8", "fp8"])
@pytest.mark.parametrize("n,Hq,Hkv,D", [(1037, 16, 8, 128), (1030, 16, 2, 256), (1026, 5, 1, 128), (35, 64, 8, 128),
                                        (33, 40, 8, 256)])
def test_norm_rope_append_many_rows(ctx, fmt, n, Hq, Hkv, D):
    """Prompts of several sequences, which start and end inside blocks, and many heads."""
    import torch

    rng = np.random.default_rng(n)
    blocks = rng.permutation(-(-n // BT) + 8)
    slots, at = [], 0
    for length in (n // 3, 1, n - n // 3 - 1):  # each from some offset of its own blocks
        first = int(rng.integers(0, BT))
        rows = np.arange(first, first + length)
        slots.append(blocks[at + rows // BT] * BT + rows % BT)
        at += rows[-1] // BT + 1
    slots = np.concatenate(slots).astype(np.int64)
    assert slots.size == n and np.unique(slots).size == n and at <= blocks.size
    qkv, wq, wk, pos, freq = rope_case(n, Hq, Hkv, D, D, 4)
    q, k, v = split(view_bf16(qkv), Hq, Hkv, D)
    dev = [view_bf16(wq), view_bf16(wk), to_dev(pos), to_dev(freq), to_dev(slots)]
    d = ctx.qk_rope_desc(q, k, v, dev[2], dev[3], q_weight=dev[0], k_weight=dev[1])
    one, two = (fresh_pool(ctx, FMTS[fmt], BT, Hkv, D, blocks.size, 92) for _ in range(2))
    q1, q2 = (torch.full((n, Hq, D), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    k2 = torch.empty((n, Hkv, D), dtype=torch.bfloat16, device="cuda")
    ctx.qk_norm_rope_append(one, d, dev[4], q1)
    ctx.qk_norm_rope(d, q2, k2)
    ctx.append(two, dev[4], k2, v.contiguous())
    torch.cuda.synchronize()
    assert ctx.device_errors() == 0
    assert torch.equal(q1.view(torch.int16), q2.view(torch.int16))
    a, b = one.raw(), two.raw()
    for key in a:
        assert np.array_equal(a[key], b[key]), key


@pytest.mark.parametrize("D", [128, 256])
def test_norm_rope_append_unaligned_values_and_output(ctx, D):
    """Values and queries that lie anywhere, keys in 16-byte pieces: the same bits."""
    import torch

    Hq, Hkv, n = 4, 2, 37
    qkv, wq, wk, pos, freq = rope_case(n, Hq, Hkv, D, 64, 8)
    t = view_bf16(qkv)
    q, k, v = split(t, Hq, Hkv, D)
    odd = torch.zeros(v.numel() + 1, dtype=torch.bfloat16, device="cuda")
    odd[1:] = v.reshape(-1)
    dev = [view_bf16(wq), view_bf16(wk), to_dev(pos), to_dev(freq), to_dev(np.arange(5, 5 + n, dtype=np.int64))]
    pools = [fresh_pool(ctx, llm_hip.KV_F16, 16, Hkv, D, 3, 90) for _ in range(2)]
    outs = []
    for pool, values, off in ((pools[0], v, 0), (pools[1], odd[1:].view(n, Hkv, D), 1)):
        buf = torch.zeros(n * Hq * D + 1, dtype=torch.bfloat16, device="cuda")
        d = ctx.qk_rope_desc(q, k, values, dev[2], dev[3], q_weight=dev[0], k_weight=dev[1])
        ctx.qk_norm_rope_append(pool, d, dev[4], buf[off:])
        outs.append(buf[off:off + n * Hq * D].clone())
    torch.cuda.synchronize()
    assert ctx.device_errors() == 0
    assert torch.equal(outs[0].view(torch.int16), outs[1].view(torch.int16))
    a, b = (p.raw() for p in pools)
    for key in a:
        assert np.array_equal(a[key], b[key]), key


@pytest.mark.parametrize("fmt", ["bf16", "f16", "int8"])
def test_norm_rope_append_bad_slots(ctx, fmt):
    """Slots outside the pool are flagged and write nothing; the others are written."""
    import torch

    Hq, Hkv, D, n = 4, 2, 128, 20
    slots = np.arange(16, 16 + n).astype(np.int64)
    slots[[2, 9]] = [-1, 4 * 16]
    slots[17] = 1 << 40
    qkv, wq, wk, pos, freq = rope_case(n, Hq, Hkv, D, D, 3)
    q, k, v = split(view_bf16(qkv), Hq, Hkv, D)
    dev = [to_dev(pos), to_dev(freq)]
    d = ctx.qk_rope_desc(q, k, v, *dev)
    pool, other = (fresh_pool(ctx, FMTS[fmt], 16, Hkv, D, 4, 91) for _ in range(2))
    qo = torch.empty((n, Hq, D), dtype=torch.bfloat16, device="cuda")
    ctx.qk_norm_rope_append(pool, d, to_dev(slots), qo)
    assert ctx.device_errors() == llm_hip.ERR_FLAG_BAD_BLOCK
    ko = torch.empty((n, Hkv, D), dtype=torch.bfloat16, device="cuda")
    ctx.qk_norm_rope(d, qo, ko)
    ok = torch.from_numpy(np.flatnonzero((slots >= 0) & (slots < 64))).cuda()
    ctx.append(other, to_dev(slots)[ok], ko[ok].contiguous(), v[ok].contiguous())
    assert ctx.device_errors() == 0
    a, b = pool.raw(), other.raw()
    for key in a:
        assert np.array_equal(a[key], b[key]), key


def test_rope_python_refusals(ctx):
    import torch

    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device="cuda")
    k = torch.zeros((2, 2, 64), dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    freq = torch.ones(32, device="cuda")
    for bad in [dict(q=q.transpose(1, 2)), dict(q=q[..., ::2]), dict(q=q[:1]), dict(k=k[..., :32].contiguous()),
                dict(v=q), dict(q=q.float()), dict(positions=pos.long()), dict(positions=pos[:1]),
                dict(inv_freq=freq.double()), dict(q_weight=freq)]:
        args = dict(q=q, k=k, v=None, positions=pos, inv_freq=freq)
        args.update(bad)
        with pytest.raises(llm_hip.LlhError):
            ctx.qk_rope_desc(**args)


# ---------------------------------------------------------------------------
# attention with accumulated weights
# ---------------------------------------------------------------------------
# f32 scores of up to ~10 units from N(0, 1) rows: D / 8 + 4 roundings of 2^-24 of the sum of the
# products' magnitudes (0.64 sqrt(D)) leave 9e-6 at head_dim 128 and 2.2e-5 at 256 in a score, so
# as much relative error in its weight; the row's sum averages it
W_REL, W_ABS = 3e-5, 1e-9


def assert_weights(got, want, what):
    bad = ~(np.abs(got - want) <= np.abs(want) * W_REL + W_ABS)
    assert not bad.any(), f"{what}: {bad.sum()} of {want.size}, worst {np.abs(got - want)[bad].max():.3e}"


def assert_out(got, want, what):
    """bf16's half step of the result, and 1e-4 for weights in two 16-bit terms times values up to 5."""
    bad = ~(np.abs(f(got) - want) <= np.abs(want) * 2.0**-8 + 1e-4)
    assert not bad.any(), f"{what}: {bad.sum()} of {want.size}, worst {np.abs(f(got) - want)[bad].max():.3e}"


EDGES = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 129, 256, 257, 700]


def weights_ref(ctx, pool, fmt, bt, Hkv, D, batch, tables, q, rows, window, gate=None):
    """(out, weights) of every sequence; rows: query rows per sequence."""
    outs, accs, at = [], [], 0
    Hq = q.shape[1]
    for b, n in enumerate(batch.seq_lens.tolist()):
        r = rows[b]
        k, v, live = ref.cached(pool, fmt, bt, Hkv, D, batch.n_blocks, tables[b], n)
        if n == 0:
            o, acc = np.zeros((r, Hq, D)), np.zeros((Hkv, 0))
        else:
            o, acc = ref.attend(f(q[at:at + r]).astype(np.float64), k, v, live, 1.0 / math.sqrt(D), window)
        outs.append(o)
        accs.append(acc)
        at += r
    out = np.concatenate(outs)
    if gate is not None:
        out = out / (1.0 + np.exp(-f(gate).astype(np.float64)))
    return out, accs


def run_weights(ctx, pool, batch, tables, q, rows, window, w_in, w_out, decay=1.0, gate=None, stream=None,
                max_len=None):
    import torch

    Hq, D = q.shape[1], q.shape[2]
    out = torch.full(q.shape, 0x7FC0, dtype=torch.int16, device="cuda")
    max_len = int(batch.seq_lens.max()) if max_len is None else max_len
    keep = [to_dev(batch.seq_lens), to_dev(tables), to_dev(q), None if gate is None else to_dev(gate)]
    if rows is None:
        d = ctx.decode_desc(keep[0], keep[1], Hq, max_len, window, gate=keep[3])
        ctx.paged_decode_weights(pool, d, keep[2], out, 1.0 / math.sqrt(D), w_in, w_out, decay, stream)
    else:
        starts = to_dev(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32))
        d = ctx.prefill_desc(starts, keep[0], keep[1], Hq, max(rows), window, gate=keep[3])
        ctx.paged_prefill_weights(pool, d, max_len, keep[2], out, 1.0 / math.sqrt(D), w_in, w_out, decay, stream)
    torch.cuda.synchronize()
    return from_dev_bf16(out)


def check_weights(ctx, fmt, lens, Hq, Hkv, D, window=0, rows=None, bt=BT, gate=False, seed=5, pad=5):
    import torch

    lens = np.array(lens, np.int32)
    batch = workloads.paged_batch(lens, bt, 0.1, seed)
    pool, _ = build_case(ctx, batch, Hq, Hkv, ALL_FMTS[fmt], seed, head_dim=D)
    T = len(lens) if rows is None else sum(rows)
    q = bf16(seed + 9, T, Hq, D)
    g = bf16(seed + 10, T, Hq, D) if gate else None
    want, acc = weights_ref(ctx, pool, ALL_FMTS[fmt], bt, Hkv, D, batch, batch.tables, q,
                            [1] * len(lens) if rows is None else rows, window, g)
    stride = max(1, int(lens.max())) + pad
    # from nothing
    w = torch.full((len(lens), Hkv, stride), -7.0, device="cuda")
    out = run_weights(ctx, pool, batch, batch.tables, q, rows, window, None, w, gate=g)
    assert ctx.device_errors() == 0, ctx.last_error()
    assert_out(out, want, f"{fmt} D{D}")
    first = w.cpu().numpy()
    for b, n in enumerate(lens.tolist()):
        assert_weights(first[b, :, :n], acc[b], f"{fmt} D{D} sequence {b} ({n})")
        assert (first[b, :, n:] == -7.0).all()  # rows behind the sequence
        for x in acc[b].reshape(-1)[first[b, :, :n].reshape(-1) == 0.0]:
            assert x < 1e-30
    # accumulated, fading, from another tensor and in place: the same bits
    before = torch.rand((len(lens), Hkv, stride), device="cuda") + 0.5
    other = torch.full_like(before, -7.0)
    out2 = run_weights(ctx, pool, batch, batch.tables, q, rows, window, before, other, 0.75, gate=g)
    assert np.array_equal(out, out2)
    inplace = before.clone()
    run_weights(ctx, pool, batch, batch.tables, q, rows, window, inplace, inplace, 0.75, gate=g)
    old, new = before.cpu().numpy().astype(np.float64), other.cpu().numpy()
    for b, n in enumerate(lens.tolist()):
        assert np.array_equal(inplace[b, :, :n].cpu().numpy(), new[b, :, :n])
        assert torch.equal(inplace[b, :, n:], before[b, :, n:])
        # the product and the sum round once each
        assert_weights(new[b, :, :n], 0.75 * old[b, :, :n] + acc[b], f"{fmt} D{D} accumulated {b}")
    assert ctx.device_errors() == 0


@pytest.mark.parametrize("window", [0, 1, 100])
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("Hq,Hkv,D", [(16, 8, 128), (32, 4, 128), (16, 2, 256), (20, 1, 256), (34, 2, 128)])
def test_decode_weights(ctx, Hq, Hkv, D, fmt, window):
    check_weights(ctx, fmt, EDGES, Hq, Hkv, D, window)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("Hq,Hkv,D", [(16, 8, 128), (16, 2, 256)])
def test_decode_weights_splits(ctx, fmt, Hq, Hkv, D):
    """One long sequence in many splits beside short ones, gated."""
    check_weights(ctx, fmt, [9000, 3, 1500], Hq, Hkv, D, gate=True)
    check_weights(ctx, fmt, [4097], Hq, Hkv, D, window=2049)


@pytest.mark.parametrize("window", [0, 129])
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("Hq,Hkv,D", [(16, 8, 128), (32, 8, 128), (8, 8, 256), (24, 8, 128)])
def test_decode_weights_of_many_sequences(ctx, Hq, Hkv, D, fmt, window):
    """Few rows of many kv heads, whose weights a wavefront adds up alone, over ends at every side of
    its 256 positions."""
    lens = [255, 256, 257, 0, 1, 321, 511, 512, 513, 767, 769, 1023, 1024, 1025, 1100, 3, 64, 700, 900, 400]
    check_weights(ctx, fmt, lens, Hq, Hkv, D, window, gate=True)


@pytest.mark.parametrize("Hq,Hkv,D", [(16, 8, 128), (16, 2, 256), (4, 2, 64)])
@pytest.mark.parametrize("chunk", [False, True])
def test_weights_over_a_ring_of_blocks(ctx, Hq, Hkv, D, chunk):
    """A window served by a ring of blocks: positions far past the table row, read modulo its length."""
    import torch

    window, ring, n = 100, 9, 1003
    rows = 4 if chunk else 1
    pool = fresh_pool(ctx, llm_hip.KV_BF16, BT, Hkv, D, 12, 71)
    table = np.random.default_rng(5).permutation(12)[:ring].astype(np.int32)[None]
    batch = workloads.PagedBatch(np.array([n], np.int32), table, 12, BT, np.zeros(1, np.int32))
    q = bf16(73, rows, Hq, D)
    k, v, live = ref.cached(pool, llm_hip.KV_BF16, BT, Hkv, D, 12, np.resize(table[0], -(-n // BT)), n)
    want, acc = ref.attend(f(q).astype(np.float64), k, v, live, 1.0 / math.sqrt(D), window)
    w = torch.full((1, Hkv, n + 1), 0.5, device="cuda")
    out = run_weights(ctx, pool, batch, table, q, [rows] if chunk else None, window, w, w)
    assert ctx.device_errors() == 0
    assert_out(out, want, "ring")
    assert_weights(w[0, :, :n].cpu().numpy(), 0.5 + acc, "ring")


@pytest.mark.parametrize("fmt,Hq,Hkv,D,bt", [("int8_row", 4, 2, 128, 16), ("bf16", 4, 2, 64, 16), ("f16", 4, 4, 96, 8),
                                             ("int8", 6, 2, 80, 16), ("fp8", 4, 1, 64, 32), ("bf16", 2, 1, 512, 16),
                                             ("bf16", 3, 1, 7, 5)])
def test_weights_other_shapes(ctx, fmt, Hq, Hkv, D, bt):
    check_weights(ctx, fmt, [0, 1, 17, 70, 300], Hq, Hkv, D, bt=bt)
    check_weights(ctx, fmt, [33, 300], Hq, Hkv, D, window=20, bt=bt)
    check_weights(ctx, fmt, [5, 40, 9, 300], Hq, Hkv, D, rows=[5, 3, 0, 7], bt=bt, gate=True)


@pytest.mark.parametrize("window", [0, 33])
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("Hq,Hkv,D", [(16, 8, 128), (16, 2, 256), (6, 2, 128), (8, 1, 256)])
def test_chunk_weights(ctx, Hq, Hkv, D, fmt, window):
    """Ragged chunks (an empty one included) in one tile of 16 packed rows and in several."""
    rows = [8, 0, 1, 13, 5]
    check_weights(ctx, fmt, [8, 40, 530, 256, 512], Hq, Hkv, D, window, rows)
    check_weights(ctx, fmt, [64, 1100, 65], Hq, Hkv, D, window, [64, 64, 33], gate=True)


def test_forced_generic_and_unaligned(ctx, opts):
    """The element-wise kernel on the packed-row kernel's shapes, by option and by alignment."""
    import torch

    opts(llm_hip.OPT_FORCE_GENERIC, 1)
    check_weights(ctx, "bf16", [0, 17, 300], 16, 8, 128)
    opts(llm_hip.OPT_FORCE_GENERIC, 0)
    lens = np.array([30, 200], np.int32)
    batch = workloads.paged_batch(lens, BT, 0.1, 3)
    pool, _ = build_case(ctx, batch, 4, 2, llm_hip.KV_BF16, 3)
    q = bf16(4, 2, 4, 128)
    want, acc = weights_ref(ctx, pool, llm_hip.KV_BF16, BT, 2, 128, batch, batch.tables, q, [1, 1], 0)
    buf = torch.zeros(q.size + 1, dtype=torch.int16, device="cuda")
    buf[1:] = to_dev(q).view(-1)
    out = torch.zeros(q.size + 1, dtype=torch.int16, device="cuda")
    w = torch.zeros((2, 2, 200), device="cuda")
    keep = [to_dev(lens), to_dev(batch.tables)]
    d = ctx.decode_desc(keep[0], keep[1], 4, 200)
    ctx.paged_decode_weights(pool, d, buf[1:], out[1:], 1.0 / math.sqrt(128), None, w)
    assert_out(from_dev_bf16(out[1:].contiguous()).reshape(q.shape), want, "unaligned")
    for b in range(2):
        assert_weights(w[b, :, :lens[b]].cpu().numpy(), acc[b], "unaligned")


@pytest.mark.parametrize("D,Hq,Hkv", [(128, 16, 8), (256, 16, 2), (64, 4, 2)])
@pytest.mark.parametrize("chunk", [False, True])
def test_weights_bad_blocks_and_lengths(ctx, D, Hq, Hkv, chunk):
    """Blocks outside the pool are masked and flagged; a sequence with none left gives zeros and
    adds nothing; a length above the bound is flagged and left alone."""
    import torch

    lens = np.array([60, 200, 48], np.int32)
    batch = workloads.paged_batch(lens, BT, 0.1, 21)
    pool, _ = build_case(ctx, batch, Hq, Hkv, llm_hip.KV_BF16, 22, head_dim=D)
    tables = batch.tables.copy()
    tables[1, 3], tables[1, 12] = batch.n_blocks, -5
    tables[2] = 1 << 30
    rows = [2, 3, 4] if chunk else None
    q = bf16(23, 9 if chunk else 3, Hq, D)
    want, acc = weights_ref(ctx, pool, llm_hip.KV_BF16, BT, Hkv, D, batch, tables, q, rows or [1] * 3, 0)
    w = torch.zeros((3, Hkv, 200), device="cuda")
    out = run_weights(ctx, pool, batch, tables, q, rows, 0, w, w)
    assert ctx.device_errors() == llm_hip.ERR_FLAG_BAD_BLOCK
    assert_out(out, want, "bad blocks")
    for b in range(3):
        assert_weights(w[b, :, :lens[b]].cpu().numpy(), acc[b], f"sequence {b}")
    assert (w[2] == 0).all() and (w[1, :, 48:64] == 0).all()
    # a bound below the second sequence's length: the others are computed
    w2 = torch.full((3, Hkv, 200), -7.0, device="cuda")
    out2 = run_weights(ctx, pool, batch, batch.tables, q, rows, 0, None, w2, max_len=100)
    assert ctx.device_errors() == llm_hip.ERR_FLAG_TOO_MANY_SPLITS
    assert (w2[1] == -7.0).all()
    want, acc = weights_ref(ctx, pool, llm_hip.KV_BF16, BT, Hkv, D, batch, batch.tables, q, rows or [1] * 3, 0)
    assert_weights(w2[0, :, :60].cpu().numpy(), acc[0], "beside")
    first = sum(rows[:1]) if chunk else 1
    assert_out(out2[:first], want[:first], "beside")


@pytest.mark.parametrize("D,Hq,Hkv", [(128, 16, 8), (64, 4, 2)])
def test_weights_non_finite(ctx, D, Hq, Hkv):
    """A non-finite score is flagged; values of masked slots may be anything."""
    import torch

    lens = np.array([60, 40], np.int32)
    batch = workloads.paged_batch(lens, BT, 0.1, 21)
    pool, _ = build_case(ctx, batch, Hq, Hkv, llm_hip.KV_BF16, 22, head_dim=D)
    q = bf16(23, 2, Hq, D)
    want, acc = weights_ref(ctx, pool, llm_hip.KV_BF16, BT, Hkv, D, batch, batch.tables, q, [1, 1], 0)
    # NaN behind the lengths, in keys and values
    for b, n in enumerate(lens.tolist()):
        slots = np.arange(n, -(-n // BT) * BT)
        at = batch.tables[b, slots // BT].astype(np.int64) * BT + slots % BT
        nan = torch.full((slots.size, Hkv, D), math.nan, dtype=torch.bfloat16, device="cuda")
        if slots.size:
            ctx.append(pool, to_dev(at), nan, nan)
    w = torch.zeros((2, Hkv, 64), device="cuda")
    out = run_weights(ctx, pool, batch, batch.tables, q, None, 0, None, w)
    assert ctx.device_errors() == 0
    assert_out(out, want, "NaN behind")
    assert_weights(w[0, :, :60].cpu().numpy(), acc[0], "NaN behind")
    q[1, 1, 3] = 0x7F80
    run_weights(ctx, pool, batch, batch.tables, q, None, 0, None, w)
    assert ctx.device_errors() & llm_hip.ERR_FLAG_NON_FINITE
    assert_weights(w[0, :, :60].cpu().numpy(), acc[0], "the other sequence")


# ---------------------------------------------------------------------------
# selection
# ---------------------------------------------------------------------------
def check_select(ctx, w, lens, budget, sinks, recent, max_len=None, stream=None):
    import torch

    B, H, stride = w.shape
    max_len = stride if max_len is None else max_len
    keep = torch.full((B, H, budget + 3), -9, dtype=torch.int32, device="cuda")
    kept = torch.full((B,), -9, dtype=torch.int32, device="cuda")
    dev = [to_dev(np.array(lens, np.int32)), to_dev(w)]
    d = ctx.select_desc(dev[0], H, max_len, budget, sinks, recent, stride, budget + 3)
    ctx.kv_select(d, dev[1], keep, kept, stream)
    torch.cuda.synchronize()
    assert ctx.device_errors() == 0
    keep, kept = keep.cpu().numpy(), kept.cpu().numpy()
    for b, n in enumerate(lens):
        m = min(n, budget)
        assert kept[b] == m
        for h in range(H):
            want = ref.select(w[b, h], n, budget, sinks, recent)
            assert np.array_equal(keep[b, h, :m], want), (b, h, n, budget, sinks, recent)
            assert (keep[b, h, m:] == -9).all()


def heavy(seed, *shape):
    rng = np.random.default_rng(seed)
    w = np.exp(3 * rng.standard_normal(shape) - 3).astype(np.float32)
    return w * (rng.random(shape) > 0.1)


SELECT_LENS = [0, 1, 2, 63, 64, 65, 100, 1023, 1024, 1025, 2047, 2500]


@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (64, 4, 16), (64, 32, 32), (64, 0, 0),
                                                 (1000, 4, 256), (2499, 7, 9), (2500, 0, 0)])
def test_select(ctx, budget, sinks, recent):
    check_select(ctx, heavy(budget, len(SELECT_LENS), 3, 2500), SELECT_LENS, budget, sinks, recent)


@pytest.mark.parametrize("n,budget", [(5000, 777), (16383, 4096), (16385, 100), (32768, 8000), (32769, 31), (65537, 20000),
                                      (131072, 8192), (200001, 64)])
def test_select_long(ctx, n, budget):
    """Long rows beside short ones, an odd stride (rows that do not start at 16 bytes)."""
    w = heavy(n, 2, 2, n + 3)
    check_select(ctx, w, [n, n // 3], budget, 4, min(16, budget - 4))


def test_select_long_rows_of_many(ctx):
    """More rows than are cut into tiles, of lengths about what one workgroup's registers hold."""
    lens = [20000, 16385, 300, 32768, 31999] + [1500 + 900 * i for i in range(30)]
    check_select(ctx, heavy(3, len(lens), 2, 32768), lens, 1111, 4, 100)


@pytest.mark.parametrize("n", [300, 3000, 40000, 100000])
def test_select_ties_and_odd_values(ctx, n):
    """Equal weights to the lowest position; -0 equals 0; infinities in order; NaN last of all."""
    rng = np.random.default_rng(n)
    w = np.zeros((1, 8, n), np.float32)
    w[0, 1] = np.float32(0.25)
    w[0, 2] = rng.integers(0, 4, n)
    w[0, 3] = np.where(rng.random(n) < 0.5, np.float32(0.0), np.float32(-0.0))
    w[0, 4] = np.where(rng.random(n) < 0.5, np.nan, rng.standard_normal(n))
    w[0, 5] = rng.choice(np.array([np.inf, -np.inf, np.nan, 1.0, -1.0], np.float32), n)
    w[0, 6] = np.nan
    w[0, 7] = np.where(rng.random(n) < 0.3, np.finfo(np.float32).min, 1e-45 * rng.integers(0, 3, n)).astype(np.float32)
    for budget, sinks, recent in [(n // 7, 0, 0), (n // 2, 3, 11), (n - 1, 0, 5), (n // 10, n // 20, n // 10 - n // 20)]:
        check_select(ctx, w, [n], budget, sinks, recent)


def test_select_flags(ctx):
    """A length above the bound, or a negative one, keeps nothing."""
    import torch

    w = to_dev(heavy(1, 3, 2, 64))
    lens = to_dev(np.array([40, 65, -1], np.int32))
    keep = torch.full((3, 2, 16), -9, dtype=torch.int32, device="cuda")
    kept = torch.full((3,), -9, dtype=torch.int32, device="cuda")
    ctx.kv_select(ctx.select_desc(lens, 2, 64, 16, 0, 4, 64, 16), w, keep, kept)
    assert ctx.device_errors() == llm_hip.ERR_FLAG_TOO_MANY_SPLITS
    assert kept.tolist() == [16, 0, 0]
    assert (keep[1:] == -9).all() and (keep[0] >= 0).all()


# ---------------------------------------------------------------------------
# compaction
# ---------------------------------------------------------------------------
def compact_case(lens, kept, Hkv, bt, seed, n_dst_extra=0):
    """Tables of the sequences, positions to keep, and destination tables over further blocks."""
    rng = np.random.default_rng(seed)
    batch = workloads.paged_batch(np.array(lens, np.int32), bt, 0.1, seed)
    need = [-(-k // bt) for k in kept]
    perm = batch.n_blocks + rng.permutation(sum(need) + n_dst_extra)
    dst = np.full((len(lens), max(max(need), 1)), -1, np.int32)
    at = 0
    for b, k in enumerate(need):
        dst[b, :k] = perm[at:at + k]
        at += k
    keep = np.full((len(lens), Hkv, max(kept) + 2), -1, np.int32)
    for b, (n, k) in enumerate(zip(lens, kept)):
        for h in range(Hkv):
            keep[b, h, :k] = np.sort(rng.permutation(n)[:k])
    return batch, keep, dst, batch.n_blocks + sum(need) + n_dst_extra


def run_compact(ctx, pool, lens, kept, keep, src, dst, w=None, w_out=None, max_kept=None):
    dev = [to_dev(np.asarray(x, np.int32)) for x in (lens, kept, keep, src, dst)]
    d = ctx.compact_desc(*dev, max(kept) if max_kept is None else max_kept, w, w_out)
    ctx.kv_compact(pool, d)


COMPACTS = [
    # lens, kept
    ([40], [40]),
    ([1], [1]),
    ([100, 7, 33], [17, 7, 16]),
    ([0, 500, 16, 31], [0, 100, 15, 1]),
    ([2000], [333]),
    ([3000, 3000], [64, 2999]),
]


@pytest.mark.parametrize("lens,kept", COMPACTS)
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("Hkv,D,bt", [(8, 128, 16), (2, 256, 16), (3, 64, 16), (1, 96, 8), (2, 40, 20)])
def test_compact(ctx, Hkv, D, bt, fmt, lens, kept):
    import torch

    batch, keep, dst, n = compact_case(lens, kept, Hkv, bt, 31 + D)
    pool = fresh_pool(ctx, FMTS[fmt], bt, Hkv, D, n, 41)
    before = ref.pool_arrays(pool)
    want = ref.compact(before, FMTS[fmt], bt, keep, kept, batch.tables, dst)
    w = torch.rand((len(lens), Hkv, max(max(lens), 1) + 3), device="cuda")
    w_out = torch.full((len(lens), Hkv, max(kept) + 5), -7.0, device="cuda")
    run_compact(ctx, pool, lens, kept, keep, batch.tables, dst, w, w_out)
    torch.cuda.synchronize()
    assert ctx.device_errors() == 0
    got = ref.pool_arrays(pool)
    for key in want:  # every block of the pool: the others as they were
        assert np.array_equal(got[key], want[key]), key
    src_w, new_w = w.cpu().numpy(), w_out.cpu().numpy()
    for b, k in enumerate(kept):
        for h in range(Hkv):
            assert np.array_equal(new_w[b, h, :k], src_w[b, h, keep[b, h, :k]])
        assert (new_w[b, :, k:] == -7.0).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("Hkv,D,bt", [(4, 128, 16), (2, 256, 16), (2, 64, 8)])
def test_compact_bad_indices(ctx, fmt, Hkv, D, bt):
    """Bad positions and source blocks leave zero tokens, bad destinations are skipped, all flagged."""
    import torch

    lens, kept = [100, 70], [40, 33]
    batch, keep, dst, n = compact_case(lens, kept, Hkv, bt, 61)
    pool = fresh_pool(ctx, FMTS[fmt], bt, Hkv, D, n, 62)
    before = ref.pool_arrays(pool)
    zero = [(0, 1, 3, -1), (0, 0, 20, 100), (1, 0, 0, 2**31 - 1), (1, 1, 32, -2**31)]
    bad = keep.copy()
    for b, h, i, p in zero:
        bad[b, h, i] = p
    src = batch.tables.copy()
    src[0, 1] = n + 5
    bad_dst = dst.copy()
    bad_dst[1, 1] = -3
    w = torch.rand((2, Hkv, 100), device="cuda") + 1.0
    w_out = torch.full((2, Hkv, 40), -7.0, device="cuda")
    run_compact(ctx, pool, lens, kept, bad, src, bad_dst, w, w_out)
    assert ctx.device_errors() == llm_hip.ERR_FLAG_BAD_BLOCK
    got = ref.pool_arrays(pool)
    new_w = w_out.cpu().numpy()
    # the expected blocks: a token of zeros in the place of a bad one, by way of a zeroed block
    arr = {k: np.concatenate([a, np.zeros_like(a[:1])]) for k, a in before.items()}
    table = np.concatenate([src, np.full((2, 1), n, np.int32)], 1)  # one more entry: the zero block
    fixed = bad.copy()
    last = src.shape[1] * bt
    gone = []
    for b in range(2):
        for h in range(Hkv):
            for i in range(kept[b]):
                p = int(bad[b, h, i])
                if p < 0 or p >= lens[b] or src[b, p // bt] >= n:
                    fixed[b, h, i] = last
                    gone.append((b, h, i))
    assert len(gone) >= 4
    ok_dst = np.where(bad_dst < 0, n, bad_dst)  # the skipped one: into the extra block
    want = ref.compact(arr, FMTS[fmt], bt, fixed, kept, table, ok_dst)
    for key in got:
        assert np.array_equal(got[key], want[key][:n]), key
    for b, h, i in gone:
        assert new_w[b, h, i] == 0.0


def test_compact_lengths(ctx):
    """A kept length above the call's bound is flagged and its sequence left alone."""
    import torch

    lens, kept = [100, 70], [40, 20]
    batch, keep, dst, n = compact_case(lens, kept, 2, 16, 61)
    pool = fresh_pool(ctx, llm_hip.KV_BF16, 16, 2, 128, n, 62)
    before = ref.pool_arrays(pool)
    run_compact(ctx, pool, lens, kept, keep, batch.tables, dst, max_kept=39)
    assert ctx.device_errors() == llm_hip.ERR_FLAG_TOO_MANY_SPLITS
    want = ref.compact(before, llm_hip.KV_BF16, 16, keep, [0, 20], batch.tables, dst)
    got = ref.pool_arrays(pool)
    for key in want:
        assert np.array_equal(got[key], want[key]), key
    with pytest.raises(llm_hip.LlhError) as e:
        run_compact(ctx, ctx.pool(llm_hip.KV_INT8_ROW, 16, 2, 128, n), lens, kept, keep, batch.tables, dst)
    assert e.value.status == llm_hip.ERR_UNSUPPORTED
    torch.cuda.synchronize()


def test_compact_fp8_same_blocks_keep_their_codes(ctx):
    """Every token kept: each block's scale, and so its codes, are what they were."""
    lens = [160, 48]
    batch, keep, dst, n = compact_case(lens, lens, 2, 16, 9)
    pool = fresh_pool(ctx, llm_hip.KV_FP8_E4M3, 16, 2, 128, n, 10)
    a = ref.pool_arrays(pool)
    run_compact(ctx, pool, lens, lens, keep, batch.tables, dst)
    b = ref.pool_arrays(pool)
    for s in range(2):
        for j in range(lens[s] // 16):
            assert np.array_equal(a["k"][batch.tables[s, j]], b["k"][dst[s, j]])
            assert np.array_equal(a["v"][batch.tables[s, j]], b["v"][dst[s, j]])
