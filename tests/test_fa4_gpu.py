"""Attention over the q4_0 cache on the GPU against numpy in 64 bits.

Tolerance of an output value, from the arithmetic (e = 2^-24, u = the rounding of `type`, half a step):
  scores   products of q and a code are exact or within 2^-22 of their value (two fp16 terms); a sum over D values
           takes D / 16 tensor-core steps, each within 3 e of the running sum of magnitudes, and a few f32 steps for
           the blocks' scales: |ds| <= (3 D / 16 + 16) e A, A = scale * max_c sum |q||k|, plus e times the mask
           value's size where a mask is added and 2 e |s| for the change of base;
  weights  dp / p <= |ds| + |ds of the maximum| + 2^-21 (the exponential);
  output   sum p v / sum p: (2 |ds| + 2^-20 + 64 e) * sum p |v|; values enter the products as d n, n = 0..15, and
           8 sum p d is taken off at the end, so a rounding is relative to 16 sum p |d| also where v = d (n - 8) is
           near 0. A tensor-core step adds 16 products and the sum so far, each cut at a unit (2 e) of the largest;
           a warp takes a step for 16 cells of its share (a quarter, and a tile's rest) of the n cells, and four
           f32 steps follow: (34 (n / 64 + 2) + 4) e * 16 sum p |d| more; and u |out| for the last rounding (fp16: at least
           2^-25, half the step of its subnormal numbers).
bf16 outputs allow the kernels one fp16 rounding (2^-11) of each weight, each key and each value: 2^-10 (A + 1) sum p |v| more.
"""
import numpy as np
import pytest

import kv4_plain as P
import tsrc

pytestmark = pytest.mark.gpu

HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def _tolerance(q, kb, vb, Hk, scale, ranges, mask, dtype, want):
    T, H, D = q.shape
    n = len(kb)
    k, v = (np.abs(P.unpack(b).reshape(n, Hk, D)) for b in (kb, vb))
    tol = np.zeros_like(want)

    def scales(rows):
        return np.abs(np.ascontiguousarray(rows.reshape(n, -1, 18)[..., :2]).view(np.float16).astype(np.float64)).reshape(n, Hk, D // 32)

    e = 2.0 ** -24
    for t in range(T):
        lo, hi = (0, n) if ranges is None else (max(int(ranges[t][0]), 0), min(int(ranges[t][1]), n))
        seen = np.zeros(n, bool)
        seen[lo:max(lo, hi)] = True
        if mask is not None:
            seen &= ~np.isneginf(mask[t, :n].astype(np.float64))
        if not seen.any():
            continue
        spread = 0.0
        if mask is not None:
            m = mask[t, :n][seen].astype(np.float64)
            spread = min(float(m.max() - m.min()), 200.0)      # weights further down than e^-200 are 0
        for h in range(H):
            kk, vv = k[seen, h // (H // Hk)], v[seen, h // (H // Hk)]
            A = abs(scale) * float((kk @ np.abs(q[t, h])).max())
            ds = ((3 * D / 16 + 16) + 2) * e * A + 4 * e * spread
            s = (P.unpack(kb).reshape(n, Hk, D)[seen, h // (H // Hk)] @ q[t, h]) * scale
            if mask is not None:
                s = s + mask[t, :n][seen].astype(np.float64)
            p = np.exp(s - s.max())
            pv = (p @ vv) / p.sum()
            pd = np.repeat((p @ scales(vb)[seen, h // (H // Hk)]) / p.sum(), 32)
            tol[t, h] = (2 * ds + 2.0 ** -20 + 64 * e) * pv + (34 * (n / 64 + 2) + 4) * e * 16 * pd + np.maximum(HALF[dtype] * np.abs(want[t, h]), 2.0 ** -25 if dtype == "float16" else 0.0)
            if dtype == "bfloat16":
                tol[t, h] += 2.0 ** -10 * (A + 1) * pv
    return tol + 1e-30


def _run(dev, q, kb, vb, Hk, scale, ranges=None, mask=None, group=0, max_len=0, n_kv=None, extra=0):
    """q: torch [T, H, D] on the GPU; -> [T, H, D] in f64."""
    import torch
    T, H, D = q.shape
    n = len(kb) if n_kv is None else n_kv
    kv = dev.kv4_create(Hk, D, len(kb) + extra)
    try:
        kv.set_bytes(tsrc.KV_K, kb)
        kv.set_bytes(tsrc.KV_V, vb)
        out = torch.full_like(q, float("nan"))
        dev.flash_attn_q4(kv, q, out, T=T, n_head=H, n_kv=n, scale=scale, group=group, max_len=max_len,
                          ranges=None if ranges is None else torch.from_numpy(np.asarray(ranges, np.int32)).cuda(),
                          mask=None if mask is None else torch.from_numpy(np.ascontiguousarray(mask)).cuda())
        dev.sync()
        return out.double().cpu().numpy()
    finally:
        kv.free()


def _inputs(seed, T, H, Hk, D, n, dtype):
    import torch
    rng = np.random.default_rng(seed)
    q = torch.from_numpy(rng.standard_normal((T, H, D)).astype(np.float32)).to(getattr(torch, dtype)).cuda()
    return rng, q, P.random_rows(rng, n, Hk * D), P.random_rows(rng, n, Hk * D)


def _check(dev, q, kb, vb, Hk, dtype, ranges=None, mask=None, scale=None, **kw):
    scale = float(np.float32(1 / np.sqrt(q.shape[2]))) if scale is None else scale
    q64 = q.double().cpu().numpy()
    n = kw.get("n_kv", len(kb))
    want = P.attend(q64, kb[:n], vb[:n], Hk, scale, ranges, mask)
    got = _run(dev, q, kb, vb, Hk, scale, ranges, mask, **kw)
    tol = _tolerance(q64, kb[:n], vb[:n], Hk, scale, ranges, mask, dtype, want)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), bad.size, float(np.nanmax(np.abs(got - want) / tol)), np.argwhere(bad)[:3].tolist())


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("H,Hk,D,n", [(1, 1, 64, 1), (4, 1, 64, 31), (14, 2, 64, 640), (32, 8, 128, 257), (8, 1, 128, 64), (3, 3, 128, 65),
                                      (16, 1, 128, 100), (5, 1, 256, 77), (8, 2, 256, 130), (4, 2, 512, 33), (9, 1, 512, 200), (64, 1, 64, 40),
                                      (40, 8, 128, 2049)])
def test_one_token(dev, dtype, H, Hk, D, n):
    _, q, kb, vb = _inputs(H * 1000 + n, 1, H, Hk, D, n, dtype)
    _check(dev, q, kb, vb, Hk, dtype)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("H,Hk,D,T,past", [(4, 1, 128, 2, 30), (8, 2, 64, 17, 0), (4, 4, 128, 40, 100), (14, 2, 64, 129, 3), (8, 2, 128, 150, 0),
                                           (8, 1, 128, 63, 500), (2, 1, 256, 70, 60), (4, 1, 512, 35, 9), (32, 8, 128, 64, 64), (7, 1, 64, 300, 40)])
def test_causal_prompt(dev, dtype, H, Hk, D, T, past):
    n = past + T
    _, q, kb, vb = _inputs(T * 100 + past, T, H, Hk, D, n, dtype)
    ranges = [[0, past + t + 1] for t in range(T)]
    _check(dev, q, kb, vb, Hk, dtype, ranges)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_windows_and_odd_ranges(dev, dtype, D):
    """Sliding windows, ranges cut to the cache, empty and inverted ranges, a first cell off every tile."""
    n, T = 333, 12
    _, q, kb, vb = _inputs(D, T, 4, 2, D, n, dtype)
    ranges = [[0, 0], [5, 5], [9, 3], [-7, 4], [300, 999], [331, 333], [332, 333], [17, 18], [63, 66], [1, 333], [333, 400], [-9, -1]]
    for group in (1, 3, 12):
        _check(dev, q, kb, vb, 2, dtype, ranges, group=group)
    _check(dev, q, kb, vb, 2, dtype, [[max(0, 20 * t - 70), 20 * t + 1] for t in range(T)], n_kv=250)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("H,Hk,D", [(8, 2, 128), (7, 1, 64), (4, 2, 256)])
@pytest.mark.parametrize("group", [1, 3])
def test_many_sequences(dev, dtype, H, Hk, D, group):
    """A decode step of ragged sequences in one cache, with one or a few tokens each; max_len too small is only slow."""
    S, cap = 9, 150
    _, q, kb, vb = _inputs(group, S * group, H, Hk, D, S * cap, dtype)
    lens = [1, 150, 64, 65, 3, 149, 32, 100, 127]
    ranges = [[s * cap, s * cap + max(1, lens[s] - group + j + 1)] for s in range(S) for j in range(group)]
    for max_len in (0, 150, 10):
        _check(dev, q, kb, vb, Hk, dtype, ranges, group=group, max_len=max_len)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("T,n,D", [(1, 70, 128), (5, 200, 128), (13, 515, 64), (90, 260, 128), (66, 100, 256), (200, 264, 64), (130, 700, 128)])
def test_masks(dev, dtype, T, n, D):
    """Hidden cells at random, a slope, a row that sees nothing, one that sees one cell, rows of the type's lowest value."""
    rng, q, kb, vb = _inputs(T + n, T, 8, 2, D, n, dtype)
    mask = np.where(rng.random((T, n)) < 0.4, -np.inf, -0.01 * rng.random((T, n)) * n).astype(np.float16)
    lowest = np.finfo(np.float16).min
    if T > 4:
        mask[0] = -np.inf
        mask[1] = -np.inf
        mask[1, n // 2] = 3.0
        mask[2] = lowest
        mask[3, : n // 2] = lowest                              # lowest, then ordinary values: weights of exactly 0
        mask[4, n // 2:] = lowest
    _check(dev, q, kb, vb, 2, dtype, mask=mask)
    ranges = [[3 * (t % 5), n - (t % 7)] for t in range(T)]
    _check(dev, q, kb, vb, 2, dtype, ranges, mask=mask)


def _compare_many(got, want, pv, pd, A, D, n, dtype, spread):
    e = 2.0 ** -24
    ds = ((3 * D / 16 + 16) + 2) * e * A + 4 * e * spread
    tol = (2 * ds + 2.0 ** -20 + 64 * e) * pv + (34 * (n / 64 + 2) + 4) * e * 16 * pd
    tol += np.maximum(HALF[dtype] * np.abs(want), 2.0 ** -25 if dtype == "float16" else 0.0) + 1e-30
    if dtype == "bfloat16":
        tol += 2.0 ** -10 * (A + 1) * pv
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), bad.size, float(np.nanmax(np.abs(got - want) / tol)), np.argwhere(bad)[:3].tolist())


def _check_many(dev, q, kb, vb, Hk, dtype, ranges, scale=None):
    """_check by matrices."""
    T, H, D = q.shape
    scale = float(np.float32(1 / np.sqrt(D))) if scale is None else scale
    want, pv, pd, A = P.attend_many(q.double().cpu().numpy(), kb, vb, Hk, scale, ranges)
    got = _run(dev, q, kb, vb, Hk, scale, ranges)
    _compare_many(got, want, pv, pd, A, D, len(kb), dtype, 0.0)


# (T, n, H, Hk, D): a last row tile of a few rows, all cells in a split; splits over the cells; one tile of rows; a short prompt;
# enough rows for CTAs of 256, their second half filled, with a few rows, empty
MANY = [(70, 1500, 32, 8, 128), (70, 4200, 32, 8, 64), (64, 6000, 8, 1, 128), (301, 301, 32, 8, 128), (513, 513, 14, 2, 64), (40, 9000, 32, 8, 128),
        (1300, 1400, 44, 11, 64), (300, 333, 120, 120, 128), (333, 500, 150, 75, 128)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("T,n,H,Hk,D", MANY)
def test_many_rows_causal(dev, dtype, T, n, H, Hk, D):
    _, q, kb, vb = _inputs(T + n, T, H, Hk, D, n, dtype)
    _check_many(dev, q, kb, vb, Hk, dtype, [[0, n - T + t + 1] for t in range(T)])


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("T,n,H,Hk,D", MANY)
def test_many_rows_masks_windows_and_hidden_cells(dev, dtype, T, n, H, Hk, D):
    """A mask with hidden cells, empty rows and rows of the type's lowest value; windows; what hides, and the mask beside
    the ranges, holds NaN, infinities and huge scales. Also a mask whose rows start off every wide boundary."""
    import torch
    rng, q, kb, vb = _inputs(T * 3 + n, T, H, Hk, D, n, dtype)
    mask = np.where(rng.random((T, n)) < 0.3, -np.inf, -0.001 * np.arange(n)[::-1]).astype(np.float16)
    mask[1] = -np.inf
    mask[2] = np.finfo(np.float16).min
    mask[3, : n // 2] = np.finfo(np.float16).min
    ranges = np.array([[max(0, n - T + t + 1 - (700 if t % 3 else n)), n - T + t + 1] for t in range(T)])
    ranges[5] = [9, 9]
    ranges[6] = [n + 5, n + 9]
    ranges[7] = [-5, n + 100]
    hidden = np.arange(20, n, 97)
    mask[:, hidden] = -np.inf
    for rows in (kb, vb):
        b = rows.reshape(n, -1, 18)
        for i, c in enumerate(hidden):
            bits = (0x7E00, 0x7C00, 0xFC00, 0x7BFF)[i % 4]
            b[c, :, :2] = np.array([bits & 255, bits >> 8], np.uint8)
    beside = (np.arange(n) < ranges[:, :1]) | (np.arange(n) >= ranges[:, 1:])
    mask[beside] = np.where(rng.random(int(beside.sum())) < 0.5, np.nan, np.inf).astype(np.float16)
    clean = np.where(beside, np.float16(-np.inf), mask)
    q64 = q.double().cpu().numpy()
    want, pv, pd, A = P.attend_many(q64, kb, vb, Hk, float(np.float32(1 / np.sqrt(D))), ranges, clean)
    got = _run(dev, q, kb, vb, Hk, float(np.float32(1 / np.sqrt(D))), ranges, mask)
    _compare_many(got, want, pv, pd, A, D, n, dtype, 0.001 * n)
    wide = np.full((T, n + 3), 7.0, np.float16)
    wide[:, :n] = clean
    kv = dev.kv4_create(Hk, D, n)
    try:
        kv.set_bytes(tsrc.KV_K, kb)
        kv.set_bytes(tsrc.KV_V, vb)
        out = torch.full_like(q, float("nan"))
        dev.flash_attn_q4(kv, q, out, T=T, n_head=H, n_kv=n, scale=float(np.float32(1 / np.sqrt(D))), mask=torch.from_numpy(wide).cuda(),
                          ranges=torch.from_numpy(ranges.astype(np.int32)).cuda())
        dev.sync()
        _compare_many(out.double().cpu().numpy(), want, pv, pd, A, D, n, dtype, 0.001 * n)
    finally:
        kv.free()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("T,D", [(300, 64), (300, 128), (1300, 64), (1300, 128)])
def test_many_rows_magnitudes(dev, dtype, T, D):
    """Scales from tiny to far above the common ones, differing from cell to cell, in tiles of the kernel for many rows."""
    import torch
    n, H, Hk = 300, 32, 8
    for qs, ks, vs, scale in ((1e3, 1e-3, 1e-4, 0.09), (1e-3, 3e2, 2e3, 0.05), (3e2, 1.0, 1.0, 0.0003), (1.0, 1.0, 6e-6, 0.0), (1.0, 20.0, 60.0, -0.004)):
        rng, q, kb, vb = _inputs(int(10 * ks) + D, T, H, Hk, D, n, "float32")
        q = (q * qs).to(getattr(torch, dtype))
        for rows, f in ((kb, ks), (vb, vs)):
            b = rows.reshape(n, -1, 18)
            d = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float32) * f
            d *= np.where(rng.random(d.shape) < 0.1, 8.0, 1.0)
            b[..., :2] = d.astype(np.float16).view(np.uint8).reshape(b[..., :2].shape)
        _check_many(dev, q, kb, vb, Hk, dtype, [[t % 3, n] for t in range(T)], scale=scale)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T", [1, 80])
def test_what_is_hidden_has_no_effect(dev, dtype, T):
    """NaN and infinite scales and huge values in cells outside the ranges or under the mask; NaN in the mask outside the range."""
    n, D = 200, 128
    rng, q, kb, vb = _inputs(T, T, 4, 2, D, n, dtype)
    mask = np.zeros((T, n), np.float16)
    mask[:, 40:60] = -np.inf
    ranges = [[10, 150]] * T
    for rows in (kb, vb):
        b = rows.reshape(n, -1, 18)
        for cells, bits in (((0, 9, 45, 199), 0x7E00), ((3, 50, 150), 0x7C00), ((8, 59, 151), 0xFC00), ((55, 180), 0x7BFF)):
            for c in cells:
                b[c, :, :2] = np.array([bits & 255, bits >> 8], np.uint8)
    mask[:, :10] = np.nan
    mask[:, 160:] = np.inf
    _check(dev, q, kb, vb, 2, dtype, ranges, mask=mask)
    _check(dev, q, kb, vb, 2, dtype, [[10, 40]] * T)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("T,D", [(3, 128), (3, 256), (300, 64), (1300, 128)])
def test_visible_scale_of_v_that_is_not_finite(dev, dtype, T, D):
    """Its block is not finite for the tokens that see the cell, whatever weight they give it; nothing else changes."""
    n, H, Hk = 200, 32, 8
    _, q, kb, vb = _inputs(T + D, T, H, Hk, D, n, dtype)
    ranges = [[0, 200] if t % 2 else [0, 100] if t % 4 else [131, 200] for t in range(T)]
    clean = _run(dev, q, kb, vb, Hk, 0.1, ranges)
    b = vb.reshape(n, Hk, D // 32, 18)
    b[130, 3, 1, :2] = np.array([0x00, 0x7C], np.uint8)
    b[120, 5, 0, :2] = np.array([0x01, 0x7E], np.uint8)
    got = _run(dev, q, kb, vb, Hk, 0.1, ranges)
    lost = np.zeros(got.shape, bool)
    lost[1::2, 12:16, 32:64] = lost[1::2, 20:24, :32] = True
    assert not np.isfinite(got[lost]).any()
    assert np.isfinite(got[~lost]).all()
    others = [h for h in range(H) if h // 4 not in (3, 5)]
    assert (got[:, others] == clean[:, others]).all()


def test_visible_nan_makes_its_row_nan(dev):
    n = 130
    _, q, kb, vb = _inputs(3, 3, 4, 2, 128, n, "float32")
    kb.reshape(n, -1, 18)[70, 0, :2] = np.array([0x00, 0x7E], np.uint8)      # head 0, block 0
    q[1, 3, 5] = float("nan")
    got = _run(dev, q, kb, vb, 2, 0.1, [[0, 130], [0, 60], [71, 130]])
    assert np.isnan(got[0, :2]).all() and np.isfinite(got[0, 2:]).all()
    assert np.isfinite(got[1, :3]).all() and np.isnan(got[1, 3]).all()
    assert np.isfinite(got[2]).all()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("T", [1, 70])
def test_scales_and_magnitudes(dev, dtype, T):
    """Large and small queries, keys and values: no overflow or loss inside the kernels' narrower terms."""
    import torch
    n, D = 300, 128
    for qs, ks, vs, scale in ((1e3, 1e-3, 1e-4, 0.09), (1e-3, 3e2, 2e3, 0.05), (3e2, 1.0, 1.0, 0.0003), (1.0, 1.0, 1.0, -0.3), (1.0, 1.0, 6e-6, 0.0)):
        rng, q, kb, vb = _inputs(T + 7, T, 8, 2, D, n, "float32")
        q = (q * qs).to(getattr(torch, dtype))
        for rows, f in ((kb, ks), (vb, vs)):
            b = rows.reshape(n, -1, 18)
            d = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float32) * f
            # values of very different sizes side by side
            d *= np.where(rng.random(d.shape) < 0.1, 8.0, 1.0)
            b[..., :2] = d.astype(np.float16).view(np.uint8).reshape(b[..., :2].shape)
        _check(dev, q, kb, vb, 2, dtype, scale=scale, ranges=[[t % 3, n] for t in range(T)])


@pytest.mark.parametrize("T,D", [(1, 128), (3, 64), (80, 128), (66, 512)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_strides_and_odd_addresses(dev, dtype, T, D):
    """q inside a fused projection's rows, off every wide boundary; out rows apart; nothing beside them is written."""
    import torch
    H, Hk, n = 4, 2, 90
    rng, q, kb, vb = _inputs(T, T, H, Hk, D, n, dtype)
    qs, os_ = H * D + 5, H * D + 3
    wide = torch.zeros(T * qs + 8, dtype=q.dtype, device="cuda")
    src = wide[1:]
    torch.as_strided(src, (T, H, D), (qs, D, 1), 1).copy_(q)
    out = torch.full((T * os_ + 8,), 3.0, dtype=q.dtype, device="cuda")
    kv = dev.kv4_create(Hk, D, n)
    try:
        kv.set_bytes(tsrc.KV_K, kb)
        kv.set_bytes(tsrc.KV_V, vb)
        dev.flash_attn_q4(kv, src, out[3:], T=T, n_head=H, n_kv=n, scale=0.1, q_stride=qs, out_stride=os_)
        dev.sync()
    finally:
        kv.free()
    got = torch.as_strided(out, (T, H, D), (os_, D, 1), 3).double().cpu().numpy()
    q64 = q.double().cpu().numpy()
    want = P.attend(q64, kb, vb, Hk, float(np.float32(0.1)))
    assert (np.abs(got - want) <= _tolerance(q64, kb, vb, Hk, 0.1, None, None, dtype, want)).all()
    rest = torch.ones_like(out, dtype=torch.bool)
    torch.as_strided(rest, (T, H, D), (os_, D, 1), 3).fill_(False)
    assert (out[rest] == 3.0).all()


@pytest.mark.parametrize("T", [1, 80])
def test_captured_replayed_and_on_two_streams(dev, T):
    """A captured call follows the ranges on the device; two graphs with a workspace each run side by side."""
    import torch
    H, Hk, D, n = 8, 2, 128, 3000
    _, q, kb, vb = _inputs(T, T, H, Hk, D, n, "float32")
    kv = dev.kv4_create(Hk, D, n)
    try:
        kv.set_bytes(tsrc.KV_K, kb)
        kv.set_bytes(tsrc.KV_V, vb)
        size = max(256, tsrc.lib().tsrc_flash_attn_q4_workspace(tsrc.TYPE_F32, Hk, D, T, H, n, 0, 0))
        jobs = []
        for i in range(2):
            r = torch.zeros(T, 2, dtype=torch.int32, device="cuda")
            out = torch.zeros_like(q)
            ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")      # NaN in every word
            g, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
            with torch.cuda.graph(g, stream=st):
                dev.flash_attn_q4(kv, q, out, T=T, n_head=H, n_kv=n, scale=0.1, ranges=r, workspace=ws)
            jobs.append((g, st, r, out))
        q64 = q.double().cpu().numpy()
        for step in (1, 900, 3000):
            for i, (g, st, r, out) in enumerate(jobs):
                r.copy_(torch.tensor([[i * (step // 2), max(1, step - t % 3)] for t in range(T)], dtype=torch.int32))
            torch.cuda.synchronize()
            for _ in range(5):
                for g, st, r, out in jobs:
                    with torch.cuda.stream(st):
                        g.replay()
            torch.cuda.synchronize()
            for g, st, r, out in jobs:
                ranges = r.cpu().numpy()
                want = P.attend(q64, kb, vb, Hk, float(np.float32(0.1)), ranges)
                tol = _tolerance(q64, kb, vb, Hk, 0.1, ranges, None, "float32", want)
                assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()
        jobs.clear()
    finally:
        kv.free()


def test_same_call_same_bits(dev):
    """The order of every sum is fixed: repeated calls agree bit for bit, and a token's result does not depend on the others."""
    import torch
    for T, dtype in ((1, "float32"), (70, "float32"), (70, "bfloat16")):
        _, q, kb, vb = _inputs(T, T, 8, 2, 128, 1500, dtype)
        a, b = (_run(dev, q, kb, vb, 2, 0.1) for _ in range(2))
        np.testing.assert_array_equal(a, b)


def test_last_cells_of_a_long_cache(dev):
    """Code offsets past 32 bits: the last cells of the last head, and a range over the end."""
    import torch
    Hk, D, cells = 8, 512, 2_200_000
    rng, q, kb, vb = _inputs(1, 2, Hk, Hk, D, 100, "float32")
    kv = dev.kv4_create(Hk, D, cells)
    try:
        kv.set_bytes(tsrc.KV_K, kb, cell0=cells - 100)
        kv.set_bytes(tsrc.KV_V, vb, cell0=cells - 100)
        out = torch.zeros_like(q)
        r = torch.tensor([[cells - 100, cells], [cells - 100, 2 ** 31 - 1]], dtype=torch.int32).cuda()
        dev.flash_attn_q4(kv, q, out, T=2, n_head=Hk, n_kv=cells, scale=0.05, ranges=r, max_len=100)
        dev.sync()
        q64 = q.double().cpu().numpy()
        want = P.attend(q64, kb, vb, Hk, float(np.float32(0.05)))
        assert (np.abs(out.double().cpu().numpy() - want) <= _tolerance(q64, kb, vb, Hk, 0.05, None, None, "float32", want)).all()
    finally:
        kv.free()


def test_refusals(dev):
    import torch
    kv = dev.kv4_create(2, 64, 100)
    try:
        q = torch.zeros(4, 4, 64, device="cuda")
        out = torch.full_like(q, 5.0)

        def call(**kw):
            a = dict(T=4, n_head=4, n_kv=100, scale=0.1) | kw
            dev.flash_attn_q4(kv, a.pop("q", q), a.pop("out", out), **a)

        for kw in (dict(n_kv=101), dict(n_head=3), dict(n_head=0), dict(q_stride=255), dict(out_stride=255), dict(group=3),
                   dict(scale=float("nan")), dict(scale=float("inf")), dict(q=q.half()), dict(q=q.double(), out=out.double()),
                   dict(ranges=torch.zeros(4, 2, dtype=torch.int64, device="cuda")),
                   dict(mask=torch.zeros(4, 99, dtype=torch.float16, device="cuda")),
                   dict(mask=torch.zeros(4, 100, device="cuda"))):
            with pytest.raises(tsrc.TsrcError) as e:
                call(**kw)
            assert e.value.code in (tsrc.E_ARG, tsrc.E_SHAPE)
        call(T=0)
        dev.sync()
        assert (out == 5).all()
        call(n_kv=0)                                              # no cells: zeros
        dev.sync()
        assert (out == 0).all()
    finally:
        kv.free()


def test_beam_search_over_the_cache(dev):
    """Store, attend, select and reorder as a beam search strings them together, beside a plain one, for three steps."""
    import torch
    rng = np.random.default_rng(11)
    B, cap, H, Hk, D, V = 4, 40, 4, 2, 64, 700
    E = Hk * D
    head = rng.standard_normal((H * D, V)).astype(np.float32) * 0.4
    embed = rng.standard_normal((V, 2 * E + H * D)).astype(np.float32)
    kv = dev.kv4_create(Hk, D, B * cap)
    try:
        n = 20
        prompt = rng.standard_normal((2, B, n, E)).astype(np.float32)
        cells = (np.arange(B)[:, None] * cap + np.arange(n)).reshape(-1)
        kv.set_rows(*(torch.from_numpy(prompt[w].reshape(B * n, E)).cuda() for w in (0, 1)), cells=torch.from_numpy(cells).cuda())
        plain = [[P.unpack(P.pack(*P.quantise(prompt[w, b]))) for b in range(B)] for w in (0, 1)]
        tokens, scores = np.arange(B) * 7, -rng.random(B).astype(np.float32)
        for step in range(3):
            row = embed[tokens]
            k, v, q = (torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in (row[:, :E], row[:, E:2 * E], row[:, 2 * E:]))
            kv.set_rows(k, v, cells=torch.arange(B, device="cuda") * cap + n)
            r = torch.tensor([[b * cap, b * cap + n + 1] for b in range(B)], dtype=torch.int32).cuda()
            out = torch.empty(B, H * D, device="cuda")
            dev.flash_attn_q4(kv, q, out, T=B, n_head=H, n_kv=B * cap, scale=0.125, ranges=r, group=1, max_len=n + 1)
            logits = out @ torch.from_numpy(head).cuda()
            s = torch.empty(1, B, device="cuda")
            beam, tok = (torch.empty(1, B, dtype=torch.int32, device="cuda") for _ in range(2))
            dev.beam_select(logits, torch.from_numpy(scores).cuda(), s, beam, tok, n_group=1, n_beam=B, n_vocab=V, n_out=B)
            kv.reorder(beam, 1, B, cap, n + 1)
            dev.sync()
            want = np.zeros((B, H, D))
            for b in range(B):
                for w, x in ((0, row[b, :E]), (1, row[b, E:2 * E])):
                    plain[w][b] = np.concatenate([plain[w][b], P.unpack(P.pack(*P.quantise(x[None])))])
                kk, vv = (plain[w][b].reshape(-1, Hk, D) for w in (0, 1))
                for h in range(H):
                    z = kk[:, h // 2] @ row[b, 2 * E:].astype(np.float64).reshape(H, D)[h] * 0.125
                    p = np.exp(z - z.max())
                    want[b, h] = p @ vv[:, h // 2] / p.sum()
            np.testing.assert_allclose(out.cpu().numpy(), want.reshape(B, -1), rtol=0, atol=1e-5 * np.abs(want).max())
            ws, wb, wt = P.beam((want.reshape(B, -1) @ head.astype(np.float64))[None], scores[None].astype(np.float64), B)
            np.testing.assert_array_equal(beam.cpu().numpy(), wb)
            np.testing.assert_array_equal(tok.cpu().numpy(), wt)
            plain = [[plain[w][p] for p in wb[0]] for w in (0, 1)]
            tokens, scores = wt[0], s.cpu().numpy()[0]
            n += 1
            got = torch.empty(n, E, device="cuda")
            for b in range(B):
                kv.get_rows(None, got, n=n, cell0=b * cap)
                np.testing.assert_array_equal(got.double().cpu().numpy(), plain[1][b])
    finally:
        kv.free()
