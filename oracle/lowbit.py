"""Plain 64-bit restatements (numpy) of the low-bit operators of include/lbx.h:
the 8-bit integer product, the 4-bit KV cache and its attention, and the
verification of sampled drafts.  Where a definition names a rounding (codes,
steps, least values) it is made here too, in float32 or bfloat16; everything
else is float64."""
from __future__ import annotations

import numpy as np

GROUP = 64
F32_TINY = np.float32(1.1754943508222875e-38)


def bf16_bits(x) -> np.ndarray:
    """Round-to-nearest-even bfloat16 bits of float32 values (NaN -> 0x7fc0)."""
    x = np.asarray(x, np.float32)
    b = x.view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def bf16_value(bits) -> np.ndarray:
    return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


def quantize_tokens(x):
    """float32 x [m, k] -> (int8 codes, float32 scale)."""
    x = np.asarray(x, np.float32)
    a = np.abs(x).max(axis=1)
    fin = np.isfinite(a)
    with np.errstate(all="ignore"):
        inv = np.where(fin & (a > 0), np.float32(127) / a, np.float32(0)).astype(np.float32)
        inv = np.where(np.isfinite(inv), inv, np.float32(0))
        q = np.where(fin[:, None], np.rint(x * inv[:, None]), 0)
        scale = np.where(fin, a * np.float32(1 / 127), np.float32(np.nan)).astype(np.float32)
    return q.astype(np.int8), scale


def linear_int8(x, w, w_scale, bias=None):
    q, s = quantize_tokens(x)
    y = (q.astype(np.float64) @ np.asarray(w, np.float64).T) * s.astype(np.float64)[:, None]
    y = y * np.asarray(w_scale, np.float64)
    return y if bias is None else y + np.asarray(bias, np.float64)


# ---- 4-bit cache -----------------------------------------------------------
def rotate_f32(x, cs):
    """Rotate-half of x [..., d] by (cos, sin) pairs cs [..., d/2, 2], each product and sum rounded to float32."""
    x, cs = np.asarray(x, np.float32), np.asarray(cs, np.float32)
    h = x.shape[-1] // 2
    a, b, c, s = x[..., :h], x[..., h:], cs[..., 0], cs[..., 1]
    return np.concatenate([(a * c) - (b * s), (b * c) + (a * s)], -1)


def kv4_quantize(x):
    """float32 x [..., d] -> codes uint8 [..., d], params uint16 (step, least) bf16 bits [..., d/64, 2]."""
    x = np.asarray(x, np.float32)
    y = x.reshape(*x.shape[:-1], -1, GROUP)
    with np.errstate(all="ignore"):
        fin = np.isfinite(y).all(-1)
        lo, hi = y.min(-1), y.max(-1)
        step = bf16_bits((hi - lo) * np.float32(1 / 15))
        step = np.where(bf16_value(step) < F32_TINY, np.uint16(0), step)
        least = bf16_bits(lo)
        bad = ~fin | ~np.isfinite(bf16_value(step)) | ~np.isfinite(bf16_value(least))
        step, least = np.where(bad, np.uint16(0x7FC0), step), np.where(bad, np.uint16(0x7FC0), least)
        sv, lv = bf16_value(step), bf16_value(least)
        inv = np.where(sv > 0, np.float32(1) / sv, np.float32(0)).astype(np.float32)
        c = np.clip(np.rint((y - lv[..., None]) * inv[..., None]), 0, 15)
        c = np.where(bad[..., None] | (sv == 0)[..., None], 0, c)
    return c.astype(np.uint8).reshape(x.shape), np.stack([step, least], -1)


def kv4_words(d, value):
    """Word index of each block of eight dimensions within a row."""
    b = np.arange(d // 8)
    g, r = b // 8, b % 8
    return r * (d // 64) + g if value else (r % 4) * (d // 32) + 2 * g + r // 4


def kv4_pack(codes, value):
    d = codes.shape[-1]
    c = codes.reshape(*codes.shape[:-1], d // 8, 8).astype(np.uint32)
    w = np.zeros(c.shape[:-1], np.uint32)
    w[..., kv4_words(d, value)] = (c << (4 * np.arange(8, dtype=np.uint32))).sum(-1, dtype=np.uint32)
    return np.ascontiguousarray(w).view(np.uint8)


def kv4_unpack(packed, value):
    w = np.ascontiguousarray(packed).view(np.uint32)
    d = w.shape[-1] * 8
    w = w[..., kv4_words(d, value)]
    return ((w[..., None] >> (4 * np.arange(8, dtype=np.uint32))) & 15).astype(np.uint8).reshape(*w.shape[:-1], d)


def kv4_values(codes, params):
    """float64 values of codes [..., d] and bf16 bits params [..., d/64, 2]."""
    v = bf16_value(params).astype(np.float64)
    c = codes.reshape(*codes.shape[:-1], -1, GROUP).astype(np.float64)
    return (v[..., 1:2] + v[..., 0:1] * c).reshape(codes.shape)


def attention(q, k, v, prefix, scale, rope_cs=None, masks=None):
    """q [n, heads, d], k / v [kv_heads, slots, d] float64 of one sequence whose new tokens sit at slots prefix..;
    masks: list of n integers (bit j: new token j visible) or None (causal).  -> [n, heads, d]"""
    q = np.asarray(q, np.float64)
    n, heads, d = q.shape
    if rope_cs is not None:
        cs = np.asarray(rope_cs, np.float64).reshape(n, 1, d // 2, 2)
        a, b = q[..., : d // 2], q[..., d // 2:]
        q = np.concatenate([a * cs[..., 0] - b * cs[..., 1], b * cs[..., 0] + a * cs[..., 1]], -1)
    rep = heads // k.shape[0]
    out = np.zeros((n, heads, d))
    for i in range(n):
        seen = list(range(prefix)) + [prefix + j for j in range(n)
                                      if ((masks[i] >> j) & 1 if masks is not None else j <= i)]
        if not seen:
            continue
        for h in range(heads):
            s = (k[h // rep, seen] @ q[i, h]) * scale
            p = np.exp(s - s.max())
            out[i, h] = (p / p.sum()) @ v[h // rep, seen]
    return out


# ---- verification of sampled drafts ----------------------------------------
def _prob(x, T):
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, np.float64))
    m = x.max()
    if m == -np.inf:
        return np.zeros_like(x)
    if not T > 0:
        return (np.arange(x.size) == int(np.argmax(x))).astype(np.float64)
    with np.errstate(invalid="ignore"):
        w = np.where(x == m, 1.0, np.exp((x - m) / T))
    return w / w.sum()


def accept_sampled(tokens, target, draft, u, e, T, count):
    """One sequence: tokens [k], target [k+1, V], draft [k, V] or None, u [k], e [V], count <= k drafts ->
    (accepted, next, margin): margin is the least relative distance of any decision from its opposite."""
    a, margin = 0, np.inf
    p = q = None
    while True:
        p = _prob(target[a], T)
        if a >= count:
            break
        d = int(tokens[a])
        inside = 0 <= d < p.size
        if draft is not None:
            q = _prob(draft[a], T)
            qd = q[d] if inside else 0.0
        else:
            q, qd = (np.arange(p.size) == d).astype(np.float64), 1.0
        ratio = min((p[d] if inside else 0.0) / max(qd, 1e-10), 1.0)
        if 0 < ratio < 1:
            margin = min(margin, abs(u[a] - ratio) / ratio)
        if not u[a] < ratio:
            break
        a += 1
    r = p
    if a < count:
        over = np.maximum(p - q, 0)
        if over.max() > 0:
            r = over
            # p and q are softmaxes to about 1e-7 each: where they nearly cancel, the difference is not told
            near = (over > 0) & (over < 1e-4 * p)
            if near.any():
                top = (np.where(near, 0, over) / e).max()
                if (1e-4 * p[near] / e[near]).max() > top:
                    margin = 0.0
    sc = r / np.asarray(e, np.float64)
    if sc.max() <= 0:
        return a, -1, margin
    best = int(np.argmax(sc))
    rest = np.delete(sc, best)
    if T > 0 and rest.size:
        margin = min(margin, (sc[best] - rest.max()) / sc[best])
    return a, best, margin
