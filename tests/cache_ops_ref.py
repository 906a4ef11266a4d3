"""The operators around an evicting cache in 64 bits, from their formulas (numpy)."""
import numpy as np

import llm_hip
import oracle

FMTS = {"bf16": llm_hip.KV_BF16, "f16": llm_hip.KV_F16, "int8": llm_hip.KV_INT8, "fp8": llm_hip.KV_FP8_E4M3}


def norm_rope(x, pos, freq, weight=None, offset=0.0, eps=1e-6, adjacent=False):
    """x [n][heads][D] (any float), pos [n], freq [R/2] f32 -> f64."""
    y = np.asarray(x, np.float64)
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * (
            np.asarray(weight, np.float64) + offset)
    y = y.copy()
    h = len(freq)
    if h:
        a = np.asarray(pos, np.float64)[:, None] * np.asarray(freq, np.float64)
        c, s = np.cos(a)[:, None], np.sin(a)[:, None]
        i = np.arange(h)
        u, v = (2 * i, 2 * i + 1) if adjacent else (i, i + h)
        yu, yv = y[..., u].copy(), y[..., v].copy()
        y[..., u] = yu * c - yv * s
        y[..., v] = yv * c + yu * s
    return y


def cached(pool, fmt, bt, hkv, d, n_blocks, table, length):
    """K and V of positions [0, length) as the pool holds them, [length][Hkv][D] f64; a block
    outside the pool reads as zeros, and its positions are False in the third array."""
    p = oracle.Pool.from_raw(fmt, bt, hkv, d, n_blocks, pool.raw())
    t = np.asarray(table, np.int64)
    ok = (t >= 0) & (t < n_blocks)
    st, k, v = p.gather_f32(np.where(ok, t, 0), 0, length)
    assert st == oracle.OK
    live = ok[(np.arange(length) // bt) % t.size] if length else np.zeros(0, bool)
    k, v = (x.reshape(length, hkv, d).astype(np.float64) * live[:, None, None] for x in (k, v))
    return k, v, live


def attend(q, k, v, live, scale, window=0):
    """The last len(q) positions' rows q [r][Hq][D] over k, v [n][Hkv][D]: out [r][Hq][D] and the
    weights summed over rows and a kv head's query heads, [Hkv][n]."""
    r, hq, _ = q.shape
    n, hkv, _ = k.shape
    g = hq // hkv
    out, acc = np.zeros(q.shape), np.zeros((hkv, n))
    for i in range(r):
        pos = n - r + i
        lo = max(0, pos - window + 1) if window else 0
        on = np.zeros(n, bool)
        on[lo:pos + 1] = live[lo:pos + 1]
        if not on.any():
            continue
        for h in range(hq):
            s = (k[on, h // g] @ q[i, h]) * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h] = p @ v[on, h // g]
            acc[h // g, on] += p
    return out, acc


def select(w, length, budget, sinks, recent):
    """Kept positions of one row, ascending."""
    if length <= budget:
        return np.arange(length)
    x = np.asarray(w[:length], np.float64)
    key = np.where(np.isnan(x), -np.inf, x)
    nan = np.isnan(x)
    mid = np.arange(sinks, length - recent)
    # NaN below -inf, ties to the lowest position
    order = sorted(mid, key=lambda p: (nan[p], -key[p] if np.isfinite(key[p]) else (-np.inf if key[p] > 0 else np.inf), p))
    picked = order[:budget - sinks - recent]
    return np.sort(np.concatenate([np.arange(sinks), picked, np.arange(length - recent, length)]).astype(np.int64))


def pool_arrays(pool):
    """A pool's raw bytes as arrays in its layout."""
    i, raw = pool.info, pool.raw()
    n, h, bt, d = i.n_blocks, i.kv_heads, i.block_tokens, i.head_dim
    dt = np.uint16 if i.format in (llm_hip.KV_BF16, llm_hip.KV_F16) else np.uint8
    out = {"k": raw["k"].view(dt).reshape(n, h, bt, d), "v": raw["v"].view(dt).reshape(n, h, d, bt)}
    if i.format == llm_hip.KV_INT8:
        out["ks"], out["vs"] = (raw[x].view(np.uint16).reshape(n, h, bt) for x in ("k_scales", "v_scales"))
    if i.format == llm_hip.KV_FP8_E4M3:
        out["ks"], out["vs"] = (raw[x].view(np.float32).reshape(n, h) for x in ("k_scales", "v_scales"))
    return out


def compact(arr, fmt, bt, keep, kept, src, dst):
    """The pool's arrays after the kept tokens' move (valid positions only)."""
    out = {k: a.copy() for k, a in arr.items()}
    hkv = arr["k"].shape[1]
    for b, n in enumerate(kept):
        for j in range(-(-int(n) // bt)):
            m = min(bt, int(n) - j * bt)
            to = dst[b, j]
            for h in range(hkv):
                pos = keep[b, h, j * bt:j * bt + m]
                blk, off = src[b, pos // bt], pos % bt
                for x in ("k", "v"):
                    rows = arr[x][blk, h, off] if x == "k" else arr[x][blk, h, :, off]  # [m][D]
                    new = np.zeros((bt, rows.shape[1]), rows.dtype)
                    if fmt == llm_hip.KV_FP8_E4M3:
                        f = oracle.fp8_decode_table()[rows].astype(np.float32) * arr[x + "s"][blk, h][:, None]
                        mx = np.float32(np.abs(f).max()) if m else np.float32(0)
                        s = np.float32(mx / np.float32(448.0))
                        out[x + "s"][to, h] = s
                        if s > 0:
                            new[:m] = oracle.fp8_encode((f / s).astype(np.float32).ravel()).reshape(m, -1)
                    else:
                        new[:m] = rows
                    out[x][to, h] = new if x == "k" else new.T
                    if fmt == llm_hip.KV_INT8:
                        out[x + "s"][to, h] = 0
                        out[x + "s"][to, h, :m] = arr[x + "s"][blk, h, off]
    return out
