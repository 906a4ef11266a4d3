"""What the operators around an evicting key-value cache are measured on.

One layer of a serving program: the norms and the rotation of a token's queries and keys on their
way into the paged cache, attention that also accumulates how much weight each cached token has
received, the choice of the tokens to keep, and the move of the kept ones to fewer blocks.  Shapes
are the layers of this repository's workloads and tests: 16 or 32 query heads over 8 or 4 kv heads
at head_dim 128, 16 over 2 and 8 over 4 at head_dim 256.

Blocks hold 16 tokens: keys [block][head][token][dim], values [block][head][dim][token], int8 scales
[block][head][token][K, V], fp8 scales [block][head][K, V].  Block tables are a permutation of the
pool, and sequences end inside their last block.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

BT = 16
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "int8": torch.int8, "fp8": torch.float8_e4m3fn}
ELEM = {"bf16": 2, "f16": 2, "int8": 1, "fp8": 1}
PIECE = 2048  # blocks made at a time
EPS = 1e-6

_context = []


def _llm_hip():
    path = os.path.join(os.getcwd(), "kir-ai_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import llm_hip

    return llm_hip


def _ctx():
    """A serving program keeps one context for the process."""
    if not _context:
        _context.append(_llm_hip().Context(0))
    return _context[0]


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one token of one request enters the cache: the smallest call, where launches count
        dict(name="rope_token", kind="rope", fmt="bf16", D=128, Hq=16, Hkv=8, rot=128, adjacent=False, offset=0.0,
             B=1, new_lo=1, new_hi=1, pos_hi=40960, seed=1),
        # a batch of prompts, whole blocks of them: the largest traffic of this operator
        dict(name="rope_prompts", kind="rope", fmt="bf16", D=128, Hq=32, Hkv=4, rot=128, adjacent=False, offset=0.0,
             B=4, new_lo=1024, new_hi=1024, pos_hi=0, seed=2),
        # ragged chunks behind far positions, partly rotated heads, (1 + w) norms, over fp16 blocks
        dict(name="rope_partial_d256", kind="rope", fmt="f16", D=256, Hq=16, Hkv=2, rot=64, adjacent=False, offset=1.0,
             B=5, new_lo=1, new_hi=129, pos_hi=131072, seed=3),
        # one request, one token
        dict(name="weights_single", kind="decode", fmt="bf16", D=128, Hq=16, Hkv=8, B=1, len_lo=512, len_hi=512,
             window=0, gate=False, decay=1.0, seed=4),
        # a serving batch of ragged contexts
        dict(name="weights_ragged", kind="decode", fmt="bf16", D=128, Hq=16, Hkv=8, B=32, len_lo=256, len_hi=4096,
             window=0, gate=False, decay=1.0, seed=5),
        # long contexts over int8 blocks, fading weights: the largest case
        dict(name="weights_int8_long", kind="decode", fmt="int8", D=128, Hq=32, Hkv=8, B=64, len_lo=8192, len_hi=8192,
             window=0, gate=False, decay=0.99, seed=6),
        # a prompt's short chunk over a cached prefix, the chunk length of the reference's driver
        dict(name="chunk_weights", kind="chunk", fmt="bf16", D=128, Hq=16, Hkv=8, B=1, prefix_lo=4099, prefix_hi=4099,
             new_lo=8, new_hi=8, window=0, gate=False, decay=1.0, seed=7),
        # the last rows of ragged prompts as observers of their contexts, over fp8 blocks, gated
        dict(name="chunk_fp8_d256", kind="chunk", fmt="fp8", D=256, Hq=16, Hkv=2, B=4, prefix_lo=200, prefix_hi=1700,
             new_lo=5, new_hi=32, window=0, gate=True, decay=1.0, seed=8),
        # the choice after a batch of decode steps
        dict(name="select_ragged", kind="select", Hkv=8, B=32, len_lo=1025, len_hi=4096, budget=1024, sinks=4,
             recent=256, seed=9),
        # the choice in one very long context of few heads
        dict(name="select_long", kind="select", Hkv=2, B=1, len_lo=131072, len_hi=131072, budget=8192, sinks=4,
             recent=1024, seed=10),
        # the batch's caches cut to a quarter
        dict(name="compact_batch", kind="compact", fmt="bf16", D=128, Hkv=8, B=32, len_lo=4096, len_hi=4096,
             budget=1024, seed=11),
        # a few ragged caches over fp8 blocks, whose scales follow the kept rows
        dict(name="compact_fp8_d256", kind="compact", fmt="fp8", D=256, Hkv=2, B=5, len_lo=100, len_hi=2000,
             budget=333, seed=12),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "decode", "decode", "chunk", "select", "compact"])
    D, Hq, Hkv = rng.choice([(128, 16, 8), (128, 32, 8), (128, 32, 4), (256, 16, 2), (256, 8, 4)])
    fmt = rng.choice(["bf16", "f16", "int8", "fp8"])
    seed = rng.randrange(1 << 30)
    if kind == "rope":
        B = _log_int(rng, 1, 32)
        hi = max(1, _log_int(rng, 1, 4096) // B)
        return dict(kind=kind, fmt=rng.choice(["bf16", "f16"]), D=D, Hq=Hq, Hkv=Hkv, rot=rng.choice([64, D // 2, D]),
                    adjacent=rng.random() < 0.3, offset=rng.choice([0.0, 1.0]), B=B,
                    new_lo=rng.choice([1, hi // 2 + 1, hi]), new_hi=hi, pos_hi=rng.choice([0, 4096, 131072]), seed=seed)
    if kind == "select":
        Hkv, B = rng.choice([2, 4, 8]), _log_int(rng, 1, 64)
        hi = _log_int(rng, 64, max(64, 1048576 // (B * Hkv)))
        budget = rng.randint(hi // 8 + 1, hi)
        recent = rng.randint(0, budget // 2)
        return dict(kind=kind, Hkv=Hkv, B=B, len_lo=rng.choice([1, hi // 2, hi]), len_hi=hi, budget=budget,
                    sinks=rng.randint(0, min(8, budget - recent)), recent=recent, seed=seed)
    B = _log_int(rng, 1, 32)
    limit = (1 << 27) // (Hkv * D * B)
    if kind == "compact":
        hi = min(limit, _log_int(rng, 32, 16384))
        return dict(kind=kind, fmt=fmt, D=D, Hkv=Hkv, B=B, len_lo=rng.choice([1, hi // 2 + 1, hi]), len_hi=hi,
                    budget=rng.randint(hi // 8 + 1, hi), seed=seed)
    window = rng.choice([0, 0, 0, _log_int(rng, 64, 4096)])
    case = dict(kind=kind, fmt=fmt, D=D, Hq=Hq, Hkv=Hkv, B=B, window=window, gate=D == 256 and rng.random() < 0.5,
                decay=rng.choice([1.0, 1.0, 0.97]), seed=seed)
    if kind == "chunk":
        B = case["B"] = min(B, 8)
        p_hi = _log_int(rng, 16, 8192)
        n_hi = _log_int(rng, 2, 32)
        case.update(prefix_lo=rng.choice([0, p_hi // 2, p_hi]), prefix_hi=p_hi, new_lo=rng.choice([1, n_hi]),
                    new_hi=n_hi)
        return case
    hi = min(limit, _log_int(rng, 16, 32768))
    case.update(len_lo=rng.choice([1, hi // 8 + 1, hi]), len_hi=hi)
    return case


# ---------------------------------------------------------------------------
# geometry (from the case alone)
# ---------------------------------------------------------------------------
def _ints(seed, lo, hi, n):
    """n lengths in [lo, hi], one of them hi."""
    v = np.random.Generator(np.random.PCG64(seed)).integers(lo, hi + 1, size=n).astype(np.int64)
    v[n // 2] = hi
    return v


def _lens(case):
    """Context lengths (new tokens included) and each sequence's query rows."""
    if case["kind"] == "chunk":
        new = _ints(case["seed"], case["new_lo"], case["new_hi"], case["B"])
        return _ints(case["seed"] + 1, case["prefix_lo"], case["prefix_hi"], case["B"]) + new, new
    if case["kind"] == "rope":
        new = _ints(case["seed"], case["new_lo"], case["new_hi"], case["B"])
        return new, new
    lens = _ints(case["seed"], case["len_lo"], case["len_hi"], case["B"])
    return lens, np.ones_like(lens)


def _tables(lens, seed, first_block=0, n_blocks=None):
    """Block-table rows: a permutation of the blocks that the sequences need and a tenth more."""
    nblk = -(-lens // BT)
    need = int(nblk.sum())
    n = need + need // 10 + 1 if n_blocks is None else n_blocks
    perm = np.random.Generator(np.random.PCG64(seed + 2)).permutation(n) + first_block
    tables = np.full((lens.size, int(nblk.max())), -1, np.int32)
    ends = np.cumsum(nblk)
    for b, (end, k) in enumerate(zip(ends, nblk)):
        tables[b, :k] = perm[end - k:end]
    return tables, n


def _kept(case):
    lens, _ = _lens(case)
    return np.minimum(lens, case["budget"])


def _firsts(case):
    """The first position that any row of each sequence attends."""
    lens, new = _lens(case)
    return np.maximum(0, lens - new - case["window"] + 1) if case["window"] else np.zeros_like(lens)


# ---------------------------------------------------------------------------
# inputs (from the seed)
# ---------------------------------------------------------------------------
def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + salt) & 0x7FFFFFFFFFFFFFFF)
    return g


def _randn(seed, salt, *shape):
    return torch.randn(shape, generator=_gen(seed, salt), device="cuda")


def _dev(a, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(a.astype(dtype))).cuda()


def _memory(case, n):
    """Keys, values and scales of n blocks, and the framework's pool over them."""
    D, Hkv, fmt = case["D"], case["Hkv"], case["fmt"]
    dt = DTYPES[fmt]
    if own:
        lib = _llm_hip()
        code = {"bf16": lib.KV_BF16, "f16": lib.KV_F16, "int8": lib.KV_INT8, "fp8": lib.KV_FP8_E4M3}[fmt]
        pool = _ctx().pool(code, BT, Hkv, D, n)
        i = pool.info
        k = torch.as_tensor(_View(pool, i.d_k, i.k_bytes), device="cuda").view(dt).view(n, Hkv, BT, D)
        v = torch.as_tensor(_View(pool, i.d_v, i.k_bytes), device="cuda").view(dt).view(n, Hkv, D, BT)
        s = torch.as_tensor(_View(pool, i.d_k_scales, 2 * i.scale_bytes), device="cuda") if i.scale_bytes else None
        s = s if s is None else s.view(torch.float16).view(n, Hkv, BT, 2) if fmt == "int8" else s.view(
            torch.float32).view(n, Hkv, 2)
        return dict(k=k, v=v, s=s, pool=pool)
    s = None
    if fmt == "int8":
        s = torch.empty((n, Hkv, BT, 2), dtype=torch.float16, device="cuda")
    if fmt == "fp8":
        s = torch.empty((n, Hkv, 2), dtype=torch.float32, device="cuda")
    return dict(k=torch.empty((n, Hkv, BT, D), dtype=dt, device="cuda"),
                v=torch.empty((n, Hkv, D, BT), dtype=dt, device="cuda"), s=s)


def _raw(x):
    """8-bit floating elements as their codes, which can be moved."""
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


class _View:
    """A pool's memory as a tensor, which keeps the pool alive."""

    def __init__(self, pool, ptr, nbytes):
        self.pool = pool
        self.__cuda_array_interface__ = dict(shape=(nbytes,), typestr="|u1", data=(ptr, False), version=2)


def _pieces(case, seed, n):
    """(first block, keys [m][Hkv][16][D], values, scales) as the cache of the case's format holds them."""
    Hkv, D, fmt = case["Hkv"], case["D"], case["fmt"]
    gk, gv = _gen(seed, 1), _gen(seed, 2)
    gain = torch.exp(0.3 * _randn(seed, 3, Hkv, 1, D))  # channels of projected keys differ in scale
    for first in range(0, n, PIECE):
        m = min(PIECE, n - first)
        k = torch.randn((m, Hkv, BT, D), generator=gk, device="cuda") * gain
        v = torch.randn((m, Hkv, BT, D), generator=gv, device="cuda")
        if fmt == "int8":
            s = torch.stack([x.abs().amax(-1) / 127 for x in (k, v)], -1).half()
            k, v = (torch.round(x / s[..., i:i + 1].float()).clamp(-127, 127) for i, x in enumerate((k, v)))
        elif fmt == "fp8":
            s = torch.stack([x.abs().amax((-1, -2)) / 448 for x in (k, v)], -1)
            k, v = ((x / s[..., i, None, None]).clamp(-448, 448) for i, x in enumerate((k, v)))
        else:
            s = None
        yield first, k.to(DTYPES[fmt]), v.to(DTYPES[fmt]), s


def _fill(case, seed, mem, n):
    for first, k, v, s in _pieces(case, seed, n):
        _raw(mem["k"])[first:first + len(k)] = _raw(k)
        _raw(mem["v"])[first:first + len(v)] = _raw(v).transpose(2, 3)
        if s is not None:
            mem["s"][first:first + len(s)] = s


def _accumulated(case, seed, stride):
    """Weights that earlier steps left: a few tokens hold most, many hold next to nothing."""
    w = torch.exp(1.5 * _randn(seed, 21, case["B"], case["Hkv"], stride) - 5.0)
    return w * (torch.rand(w.shape, generator=_gen(seed, 22), device="cuda") > 0.1)


def _positions(case):
    """The new tokens' positions: behind their sequence's earlier ones."""
    new, _ = _lens(case)
    start = np.random.Generator(np.random.PCG64(case["seed"] + 5)).integers(0, case["pos_hi"] + 1, size=new.size)
    return np.concatenate([s + np.arange(n) for s, n in zip(start, new)])


def _rope_inputs(case, seed):
    """A fused projection's rows (queries, keys, values side by side), norm weights and frequencies."""
    D, Hq, Hkv, T = case["D"], case["Hq"], case["Hkv"], int(_lens(case)[0].sum())
    qkv = (2.0 * _randn(seed, 31, T, (Hq + 2 * Hkv) * D)).to(torch.bfloat16)
    wq, wk = (((1.0 - case["offset"]) + 0.2 * _randn(seed, salt, D)).to(torch.bfloat16) for salt in (32, 33))
    freq = 1e6 ** (-torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64) / case["rot"])
    return qkv, wq, wk, freq.float()


def _keep(case, seed, stride):
    """Kept positions of each (sequence, kv head), ascending, the most recent ones among them."""
    lens, _ = _lens(case)
    lens = _dev(lens)[:, None, None]
    at = torch.arange(int(lens.max()), device="cuda", dtype=torch.int32)
    x = torch.rand((case["B"], case["Hkv"], at.numel()), generator=_gen(seed, 41), device="cuda")
    x = torch.where(at >= lens - case["budget"] // 4, 2.0, x)
    x = torch.where(at < lens, x, -1.0)
    idx = x.topk(min(case["budget"], at.numel()), dim=-1).indices.to(torch.int32)
    idx = torch.where(idx < lens, idx, 1 << 30).sort(dim=-1).values
    keep = torch.full((case["B"], case["Hkv"], stride), -1, dtype=torch.int32, device="cuda")
    keep[..., :idx.shape[-1]] = torch.where(idx < (1 << 30), idx, -1)
    return keep


def prepare(case, seed):
    kind = case["kind"]
    st = dict(case=case)
    lens, new = _lens(case)
    st["lens"] = _dev(lens)
    if kind == "select":
        stride = -(-case["len_hi"] // 64) * 64
        st["w"] = _accumulated(case, seed, stride)
        st["keep"] = torch.full((case["B"], case["Hkv"], case["budget"]), -1, dtype=torch.int32, device="cuda")
        st["kept"] = torch.zeros(case["B"], dtype=torch.int32, device="cuda")
        if own:
            d = _ctx().select_desc(st["lens"], case["Hkv"], int(lens.max()), case["budget"], case["sinks"],
                                   case["recent"], stride, case["budget"])
            st["call"] = _ctx().bind("llh_kv_select", d, st["w"], st["keep"], st["kept"], torch.cuda.current_stream())
        return st
    tables, n = _tables(lens, case["seed"])
    st["tables"] = _dev(tables)
    if kind == "compact":
        kept = _kept(case)
        dst, n_dst = _tables(kept, case["seed"] + 7, first_block=n, n_blocks=int((-(-kept // BT)).sum()))
        mem = _memory(case, n + n_dst)
        _fill(case, seed, mem, n)
        for x in (mem["k"], mem["v"], mem["s"]):
            if x is not None:
                x.view(torch.uint8)[n:] = 0
        stride = -(-case["len_hi"] // 64) * 64
        st.update(mem, first_dst=n, kept=_dev(kept), dst=_dev(dst), keep=_keep(case, seed, case["budget"]),
                  w=_accumulated(case, seed, stride),
                  w_out=torch.zeros((case["B"], case["Hkv"], case["budget"]), device="cuda"))
        if own:
            d = _ctx().compact_desc(st["lens"], st["kept"], st["keep"], st["tables"], st["dst"], int(kept.max()),
                                    weights_in=st["w"], weights_out=st["w_out"])
            st["call"] = _ctx().bind("llh_kv_compact", st["pool"], d, torch.cuda.current_stream())
        return st
    mem = _memory(case, n)
    _fill(case, seed, mem, n)
    st.update(mem)
    D, Hq, Hkv = case["D"], case["Hq"], case["Hkv"]
    T = int(new.sum())
    if kind == "rope":
        seq = np.repeat(np.arange(lens.size), lens)
        at = np.concatenate([np.arange(k) for k in lens])
        st["slots"] = _dev(tables[seq, at // BT].astype(np.int64) * BT + at % BT, np.int64)
        st["pos"] = _dev(_positions(case))
        st["qkv"], st["wq"], st["wk"], st["freq"] = _rope_inputs(case, seed)
        st["q_out"] = torch.empty((T, Hq, D), dtype=torch.bfloat16, device="cuda")
        if own:
            q, k, v = _split(case, st["qkv"])
            d = _ctx().qk_rope_desc(q, k, v, st["pos"], st["freq"], q_weight=st["wq"], k_weight=st["wk"], eps=EPS,
                                    weight_offset=case["offset"], adjacent=case["adjacent"])
            st["call"] = _ctx().bind("llh_qk_norm_rope_append", st["pool"], d, st["slots"], st["q_out"],
                                     torch.cuda.current_stream())
        return st
    st["q"] = (_randn(seed, 11, T, Hq, D) * torch.exp(0.3 * _randn(seed, 12, Hq, D))).to(torch.bfloat16)
    st["gate"] = _randn(seed, 13, T, Hq, D).to(torch.bfloat16) if case["gate"] else None
    st["scale"] = 1.0 / math.sqrt(D)
    stride = -(-int(lens.max()) // 64) * 64
    st["w"] = _accumulated(case, seed, stride)
    st["w_out"] = torch.zeros_like(st["w"])
    st["out"] = torch.empty_like(st["q"])
    st["new"] = _dev(new)
    st["starts"] = _dev(np.concatenate([[0], np.cumsum(new)]))
    if own:
        ctx, stream = _ctx(), torch.cuda.current_stream()
        tail = (st["w"], st["w_out"], stride, case["decay"], stream)
        if kind == "decode":
            d = ctx.decode_desc(st["lens"], st["tables"], Hq, int(lens.max()), case["window"],
                                total_tokens_hint=int((lens - _firsts(case)).sum()), gate=st["gate"])
            st["call"] = ctx.bind("llh_paged_decode_weights", st["pool"], d, st["q"], st["out"], st["scale"], *tail)
        else:
            d = ctx.prefill_desc(st["starts"], st["lens"], st["tables"], Hq, int(new.max()), case["window"],
                                 total_q_rows=T, gate=st["gate"])
            st["call"] = ctx.bind("llh_paged_prefill_weights", st["pool"], d, int(lens.max()), st["q"], st["out"],
                                  st["scale"], *tail)
    return st


def _split(case, qkv):
    """The queries, keys and values of a fused projection, [T][heads][D] each."""
    D, Hq, Hkv = case["D"], case["Hq"], case["Hkv"]
    q, k, v = qkv.split([Hq * D, Hkv * D, Hkv * D], dim=-1)
    return q.unflatten(-1, (Hq, D)), k.unflatten(-1, (Hkv, D)), v.unflatten(-1, (Hkv, D))


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _turned(case, st, x, w):
    """Root-mean-square norm of each head and the rotation of its first `rot` dims."""
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (w.float() + case["offset"])
    a = st["pos"].double()[:, None] * st["freq"].double()  # far positions: 32 bits are not enough for an angle
    c, s = torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]
    R = case["rot"]
    if case["adjacent"]:
        u, v = x[..., 0:R:2], x[..., 1:R:2]
        turned = torch.stack([u * c - v * s, v * c + u * s], -1).flatten(-2)
    else:
        u, v = x[..., :R // 2], x[..., R // 2:R]
        turned = torch.cat([u * c - v * s, v * c + u * s], -1)
    return torch.cat([turned, x[..., R:]], -1).to(torch.bfloat16)


def _plain_rope(case, st):
    q, k, v = _split(case, st["qkv"])
    blk, off = st["slots"] // BT, st["slots"] % BT
    st["k"][blk, :, off] = _turned(case, st, k, st["wk"]).to(st["k"].dtype)
    st["v"][blk, :, :, off] = v.to(st["v"].dtype)
    return {"q": _turned(case, st, q, st["wq"]), "k": st["k"], "v": st["v"]}


def _cached(case, st, tables):
    """Keys and values of the tables' blocks, [B][Hkv][tokens][D] in 32 bits."""
    at, dt = tables.long().clamp(min=0), st["k"].dtype
    k, v = _raw(st["k"])[at].view(dt).float(), _raw(st["v"])[at].view(dt).float().transpose(-1, -2)
    if case["fmt"] == "int8":
        s = st["s"][at].float()
        k, v = k * s[..., 0:1], v * s[..., 1:2]
    if case["fmt"] == "fp8":
        s = st["s"][at]
        k, v = k * s[..., 0, None, None], v * s[..., 1, None, None]
    return k.transpose(1, 2).flatten(2, 3), v.transpose(1, 2).flatten(2, 3)


def _plain_attention(case, st):
    """Attention of each sequence's last rows, and its weights added up over rows and a kv head's query heads."""
    B, Hkv, D = case["B"], case["Hkv"], case["D"]
    G = case["Hq"] // Hkv
    R = int(case["new_hi"]) if case["kind"] == "chunk" else 1
    k, v = _cached(case, st, st["tables"])
    N = k.shape[2]
    row = torch.arange(R, device="cuda")
    live = row < st["new"][:, None]                                      # [B][R]
    src = (st["starts"][:-1, None] + row).clamp(max=st["q"].shape[0] - 1).long()
    q = st["q"][src].float()                                             # [B][R][Hq][D]
    q = q.view(B, R, Hkv, G, D).permute(0, 2, 4, 1, 3).reshape(B, Hkv, D, R * G).contiguous()
    s = (torch.matmul(k, q) * st["scale"]).view(B, Hkv, N, R, G)
    key = torch.arange(N, device="cuda")[None, :, None]
    pos = (st["lens"] - st["new"])[:, None, None] + row
    on = (key <= pos) & (key < st["lens"][:, None, None]) & live[:, None, :]
    if case["window"]:
        on = on & (key > pos - case["window"])
    s = torch.where(on[:, None, :, :, None], s, -math.inf)
    top = s.amax(2, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(2, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = torch.matmul(p.view(B, Hkv, N, R * G).transpose(2, 3).contiguous(), v.contiguous())
    o = o.view(B, Hkv, R, G, D).transpose(1, 2).reshape(B, R, Hkv * G, D)[live]
    if case["gate"]:
        o = o / (1 + torch.exp(-st["gate"].float()))
    st["out"].copy_(o)
    N = min(N, st["w"].shape[2])
    w = st["w"][..., :N] * case["decay"] + p.sum((3, 4))[..., :N]
    at = torch.arange(N, device="cuda") < st["lens"][:, None, None]
    st["w_out"][..., :N] = torch.where(at, w, st["w_out"][..., :N])
    return {"out": st["out"], "weights": st["w_out"]}


def _plain_select(case, st):
    n = st["lens"][:, None, None]
    at = torch.arange(st["w"].shape[2], device="cuda")
    x = torch.where((at < case["sinks"]) | (at >= n - case["recent"]), math.inf, st["w"])
    x = torch.where(at < n, x, -math.inf)
    idx = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :case["budget"]]
    idx = torch.where(idx < n, idx, 1 << 40).sort(-1).values
    m = idx.shape[-1]
    st["keep"][..., :m] = torch.where(idx < (1 << 40), idx, st["keep"][..., :m].long()).int()
    st["kept"].copy_(st["lens"].clamp(max=case["budget"]))
    return {"keep": st["keep"], "kept": st["kept"]}


def _plain_compact(case, st):
    B, Hkv, D = case["B"], case["Hkv"], case["D"]
    width = st["dst"].shape[1] * BT
    at = torch.arange(width, device="cuda")
    on = (at < st["kept"][:, None, None]).expand(B, Hkv, width)          # [B][Hkv][width]
    pos = torch.zeros((B, Hkv, width), dtype=torch.int64, device="cuda")
    m = min(width, st["keep"].shape[2])
    pos[..., :m] = st["keep"][..., :m].long().clamp(min=0)
    blk = torch.gather(st["tables"].long()[:, None].expand(B, Hkv, -1), 2, pos // BT).clamp(min=0)
    off, h = pos % BT, torch.arange(Hkv, device="cuda")[None, :, None]
    k, v = _raw(st["k"])[blk, h, off], _raw(st["v"])[blk, h, :, off]     # [B][Hkv][width][D]
    used = st["dst"] >= 0
    to = st["dst"][used].long()

    def blocks(x):
        """[B][Hkv][width][...] as the destination blocks in use, [n][Hkv][16][...]"""
        x = x.unflatten(2, (-1, BT)).transpose(1, 2)
        return x[used]

    if case["fmt"] == "fp8":
        old = st["s"][blk, h]                                            # [B][Hkv][width][2]
        k, v = (x.view(torch.float8_e4m3fn).float() * old[..., i:i + 1] for i, x in enumerate((k, v)))
        k, v = (blocks(torch.where(on[..., None], x, 0.0)) for x in (k, v))
        s = torch.stack([x.abs().amax((-1, -2)) / 448 for x in (k, v)], -1)
        k, v = (torch.where(s[..., i, None, None] > 0, x / s[..., i, None, None], 0.0).clamp(-448, 448)
                .to(torch.float8_e4m3fn).view(torch.uint8) for i, x in enumerate((k, v)))
        st["s"][to] = s
    else:
        k, v = (blocks(torch.where(on[..., None], x, 0)) for x in (k, v))
        if case["fmt"] == "int8":
            st["s"][to] = blocks(torch.where(on[..., None], st["s"][blk, h, off], 0.0))
    _raw(st["k"])[to] = k
    _raw(st["v"])[to] = v.transpose(-1, -2)
    w = torch.gather(st["w"], 2, pos[..., :m])
    st["w_out"][..., :m] = torch.where(on[..., :m], w, st["w_out"][..., :m])
    return _compacted(st)


def _compacted(st):
    n = st["first_dst"]
    out = {"k": st["k"][n:], "v": st["v"][n:], "weights": st["w_out"]}
    if st["s"] is not None:
        out["scales"] = st["s"][n:]
    return out


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        st["call"]()
        if kind == "rope":
            return {"q": st["q_out"], "k": st["k"], "v": st["v"]}
        if kind == "select":
            return {"keep": st["keep"], "kept": st["kept"]}
        if kind == "compact":
            return _compacted(st)
        return {"out": st["out"], "weights": st["w_out"]}
    if kind == "rope":
        return _plain_rope(case, st)
    if kind == "select":
        return _plain_select(case, st)
    if kind == "compact":
        return _plain_compact(case, st)
    return _plain_attention(case, st)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def _scale_bytes(case, tokens, blocks):
    if case["fmt"] == "int8":
        return tokens * case["Hkv"] * 4
    return blocks * case["Hkv"] * 8 if case["fmt"] == "fp8" else 0


def work(case):
    kind, Hkv = case["kind"], case["Hkv"]
    lens, new = _lens(case)
    n = int(lens.sum())
    if kind == "select":
        kept = int(_kept(case).sum())
        return {"bytes": 4 * Hkv * (n + kept) + 8 * lens.size, "flops": 0}
    D, e = case["D"], ELEM[case["fmt"]]
    if kind == "compact":
        kept = _kept(case)
        m, blocks = int(kept.sum()), int((-(-kept // BT)).sum())
        row = m * Hkv * 2 * D * e + _scale_bytes(case, m, blocks)
        return {"bytes": 2 * row + m * Hkv * (4 + 8) + 8 * blocks, "flops": 0}
    Hq = case["Hq"]
    if kind == "rope":
        elems = n * (Hq + Hkv) * D
        return {"bytes": 2 * elems + 2 * n * Hq * D + n * Hkv * D * (2 + 2 * e) + 12 * n, "flops": 8 * elems}
    first = _firsts(case)
    attended = int((lens - first).sum())
    blocks = int((-(-lens // BT) - first // BT).sum())
    T = int(new.sum())
    moved = attended * Hkv * D * e * 2 + _scale_bytes(case, attended, blocks) + 4 * blocks + 8 * n * Hkv
    moved += T * Hq * D * 2 * (3 if case["gate"] else 2)
    pairs = 0
    for length, rows in zip(lens.tolist(), new.tolist()):
        pos = np.arange(length - rows, length, dtype=np.int64)
        lo = np.maximum(0, pos - case["window"] + 1) if case["window"] else np.zeros_like(pos)
        pairs += int((pos - lo + 1).sum())
    return {"bytes": moved, "flops": 4 * D * Hq * pairs}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------
def _contents(case, seed, n):
    """The cache's keys and values as numbers, [n][Hkv][16][D] in 64 bits, and their fp8 codes' scales."""
    ks, vs = [], []
    for _, k, v, s in _pieces(case, seed, n):
        k, v = k.double(), v.double()
        if case["fmt"] == "int8":
            k, v = k * s[..., :1].double(), v * s[..., 1:].double()
        if case["fmt"] == "fp8":
            k, v = k * s[..., :1, None].double(), v * s[..., 1:, None].double()
        ks.append(k)
        vs.append(v)
    return torch.cat(ks), torch.cat(vs)


def _exact_turn(case, x, w, freq):
    x = x.double()
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * (w.double() + case["offset"])
    z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                    torch.outer(_dev(_positions(case), np.int64).double(), freq.double()))[:, None]
    R = case["rot"]
    i = torch.arange(R // 2, device="cuda")
    a, b = (2 * i, 2 * i + 1) if case["adjacent"] else (i, i + R // 2)
    p = torch.complex(y[..., a], y[..., b]) * z
    y[..., a], y[..., b] = p.real.clone(), p.imag.clone()
    return y


def exact(case, seed):
    kind = case["kind"]
    if kind == "select":
        return None
    lens, new = _lens(case)
    tables, n = _tables(lens, case["seed"])
    D, Hkv = case["D"], case["Hkv"]
    if kind == "rope":
        qkv, wq, wk, freq = _rope_inputs(case, seed)
        q, k, v = _split(case, qkv)
        K, V = _contents(case, seed, n)
        k, row = _exact_turn(case, k, wk, freq), 0
        for b, m in enumerate(lens.tolist()):
            for j in range(0, m, BT):
                c = min(BT, m - j)
                K[tables[b, j // BT], :, :c] = k[row:row + c].transpose(0, 1)
                V[tables[b, j // BT], :, :c] = v[row:row + c].transpose(0, 1).double()
                row += c
        return {"q": _exact_turn(case, q, wq, freq), "k": K, "v": V.transpose(2, 3).contiguous()}
    K, V = _contents(case, seed, n)
    if kind == "compact":
        kept = _kept(case)
        dst, n_dst = _tables(kept, case["seed"] + 7, first_block=n, n_blocks=int((-(-kept // BT)).sum()))
        keep = _keep(case, seed, case["budget"])
        w = _accumulated(case, seed, -(-case["len_hi"] // 64) * 64)
        w_out = torch.zeros((case["B"], Hkv, case["budget"]), dtype=torch.float64, device="cuda")
        k_out = torch.zeros((n_dst, Hkv, BT, D), dtype=torch.float64, device="cuda")
        v_out = torch.zeros_like(k_out)
        for b, m in enumerate(kept.tolist()):
            ids = _dev(tables[b, :-(-int(lens[b]) // BT)], np.int64)
            to = _dev(dst[b, :-(-m // BT)] - n, np.int64)
            for h in range(Hkv):
                p = keep[b, h, :m].long()
                w_out[b, h, :m] = w[b, h, p].double()
                for src, out in ((K, k_out), (V, v_out)):
                    rows = torch.zeros((to.numel() * BT, D), dtype=torch.float64, device="cuda")
                    rows[:m] = src[ids[p // BT], h, p % BT]
                    out[to, h] = rows.view(-1, BT, D)
        out = {"k": k_out, "v": v_out.transpose(2, 3).contiguous(), "weights": w_out}
        if case["fmt"] == "fp8":
            s = torch.stack([x.abs().amax((2, 3)) / 448 for x in (k_out, v_out)], -1)
            for i, name in enumerate("kv"):
                t = s[..., i, None, None]
                out[name] = torch.where(t > 0, out[name] / t, 0.0)
            out["scales"] = s
        if case["fmt"] == "int8":  # codes and their scales are moved, not computed
            out["k"] = out["v"] = None
        return out
    Hq, G = case["Hq"], case["Hq"] // Hkv
    T = int(new.sum())
    q = (_randn(seed, 11, T, Hq, D) * torch.exp(0.3 * _randn(seed, 12, Hq, D))).to(torch.bfloat16).double()
    stride = -(-int(lens.max()) // 64) * 64
    w = _accumulated(case, seed, stride).double()
    out, weights, row = torch.empty_like(q), torch.zeros_like(w), 0
    for b, (m, r) in enumerate(zip(lens.tolist(), new.tolist())):
        ids = _dev(tables[b, :-(-m // BT)], np.int64)
        at = torch.arange(m, device="cuda")
        pos = torch.arange(m - r, m, device="cuda")[:, None]
        on = at <= pos
        if case["window"]:
            on &= at > pos - case["window"]
        for h in range(Hkv):
            k, v = K[ids, h].reshape(-1, D)[:m], V[ids, h].reshape(-1, D)[:m]
            acc = w[b, h, :m] * case["decay"]
            for g in range(h * G, h * G + G):
                s = (q[row:row + r, g] @ k.T.contiguous()) / math.sqrt(D)
                p = torch.softmax(torch.where(on, s, -math.inf), -1)
                out[row:row + r, g] = p @ v
                acc = acc + p.sum(0)
            weights[b, h, :m] = acc
        row += r
    if case["gate"]:
        out = out * torch.sigmoid(_randn(seed, 13, T, Hq, D).to(torch.bfloat16).double())
    return {"out": out, "weights": weights}
