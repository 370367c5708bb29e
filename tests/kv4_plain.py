"""Plain 64-bit forms of the q4_0 cache, the attention over it and beam selection, for the tests."""
import numpy as np


def quantise(x):
    """Rows of values -> (codes [n, blocks, 32] uint8, scales [n, blocks] float16), the format's f32 steps."""
    x = np.asarray(x, np.float32).reshape(len(x), -1, 32)
    with np.errstate(all="ignore"):
        mag = np.where(np.isnan(x), np.float32(0), np.abs(x))
        m = np.take_along_axis(x, mag.argmax(-1)[..., None], -1)
        m = np.where(mag.max(-1, keepdims=True) == 0, np.float32(0), m)
        d = (m * np.float32(-0.125)).astype(np.float32)
        inv = np.where(d == 0, np.float32(0), np.float32(1) / d).astype(np.float32)
        t = (x * inv).astype(np.float32) + np.float32(8.5)
        code = np.where(np.isnan(t), np.float32(8), np.clip(np.trunc(np.nan_to_num(t, nan=0.0, posinf=99, neginf=-99)), 0, 15))
        return code.astype(np.uint8), d[..., 0].astype(np.float16)


def pack(code, d):
    """ggml q4_0 rows [n, blocks * 18]."""
    b = np.empty(code.shape[:2] + (18,), np.uint8)
    b[..., :2] = np.ascontiguousarray(d)[..., None].view(np.uint8)
    b[..., 2:] = code[..., :16] | (code[..., 16:] << 4)
    return b.reshape(len(code), -1)


def unpack(rows):
    """ggml q4_0 rows -> values in f64 [n, E]."""
    b = np.ascontiguousarray(rows).reshape(len(rows), -1, 18)
    d = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float64)
    n = np.concatenate([b[..., 2:] & 15, b[..., 2:] >> 4], -1).astype(np.float64)
    with np.errstate(all="ignore"):
        return (d * (n - 8)).reshape(len(rows), -1)


def random_rows(rng, n, E):
    """ggml q4_0 rows of random codes and scales of either sign."""
    code = rng.integers(0, 16, (n, E // 32, 32)).astype(np.uint8)
    d = (rng.uniform(0.05, 0.4, (n, E // 32)) * rng.choice([-1, 1], (n, E // 32))).astype(np.float16)
    return pack(code, d)


def attend(q, kb, vb, n_head_kv, scale, ranges=None, mask=None):
    """q [T, H, D] f64; kb, vb ggml rows; ranges int [T, 2]; mask f16 [T, n]. What is hidden has no effect."""
    T, H, D = q.shape
    k, v = (unpack(b).reshape(len(b), n_head_kv, D) for b in (kb, vb))
    n = len(kb)
    out = np.zeros((T, H, D))
    for t in range(T):
        lo, hi = (0, n) if ranges is None else (max(int(ranges[t][0]), 0), min(int(ranges[t][1]), n))
        seen = np.zeros(n, bool)
        seen[lo:max(lo, hi)] = True
        if mask is not None:
            seen &= ~np.isneginf(mask[t, :n].astype(np.float64))
        at = np.nonzero(seen)[0]
        if not len(at):
            continue
        for h in range(H):
            with np.errstate(all="ignore"):
                s = (k[at, h // (H // n_head_kv)] @ q[t, h]) * scale
                if mask is not None:
                    s = s + mask[t, at].astype(np.float64)
                p = np.exp(s - s.max())
                out[t, h] = (p @ v[at, h // (H // n_head_kv)]) / p.sum()
    return out


def beam(logits, scores, n_out):
    """logits [G, B, V] f64, scores [G, B] -> (scores, beams, tokens), in order, ties to the lowest (beam, token)."""
    G, B, V = logits.shape
    res = np.full((G, n_out), -np.inf), np.full((G, n_out), -1, np.int32), np.full((G, n_out), -1, np.int32)
    with np.errstate(all="ignore"):
        top = np.max(np.where(np.isnan(logits), -np.inf, logits), -1, keepdims=True)
        norm = np.log(np.exp(logits - top).sum(-1, keepdims=True))
        s = scores[..., None] + ((logits - top) - norm)
    s = np.where(np.isnan(s), -np.inf, s)
    for g in range(G):
        flat = s[g].ravel()
        first = np.lexsort((np.arange(B * V), -flat))[:n_out]
        first = first[flat[first] > -np.inf]
        res[0][g, :len(first)], res[1][g, :len(first)], res[2][g, :len(first)] = flat[first], first // V, first % V
    return res


def attend_many(q, kb, vb, n_head_kv, scale, ranges, mask=None):
    """attend() by matrices, for many tokens, and the sums that a tolerance needs: (out, sum p |v|, sum p |d|, the largest
    scale * sum |q||k|, per token and head). Cells with a scale that is no number must be hidden from every token."""
    T, H, D = q.shape
    n = len(kb)
    seen = (np.arange(n) >= np.maximum(np.asarray(ranges)[:, :1], 0)) & (np.arange(n) < np.asarray(ranges)[:, 1:])
    if mask is not None:
        seen &= ~np.isneginf(mask[:, :n].astype(np.float64))
    any_seen = seen.any(0)
    k, v = (np.where(any_seen[:, None], unpack(b), 0.0).reshape(n, n_head_kv, D) for b in (kb, vb))
    d = np.abs(np.ascontiguousarray(vb.reshape(n, -1, 18)[..., :2]).view(np.float16).astype(np.float64)).reshape(n, n_head_kv, D // 32)
    d = np.repeat(np.where(any_seen[:, None, None], d, 0.0), 32, -1)
    out, pv, pd = (np.zeros((T, H, D)) for _ in range(3))
    A = np.zeros((T, H, 1))
    for h in range(H):
        g = h // (H // n_head_kv)
        s = q[:, h] @ k[:, g].T * scale
        if mask is not None:
            s = s + np.where(seen, mask[:, :n].astype(np.float64), 0.0)
        s = np.where(seen, s, -np.inf)
        top = s.max(1, keepdims=True)
        p = np.exp(s - np.where(np.isneginf(top), 0.0, top))
        total = p.sum(1, keepdims=True)
        p = np.divide(p, total, out=np.zeros_like(p), where=total > 0)
        out[:, h], pv[:, h], pd[:, h] = p @ v[:, g], p @ np.abs(v[:, g]), p @ d[:, g]
        A[:, h, 0] = np.where(seen, abs(scale) * (np.abs(q[:, h]) @ np.abs(k[:, g]).T), 0.0).max(1)
    return out, pv, pd, A
