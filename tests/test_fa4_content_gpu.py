"""Attention over the q4_0 cache on the GPU: any content that the cache's format can hold, against 64 bits.

Tolerance of an output value (e = 2^-24), for few visible cells or long rows alike:
  scores   q is within 2^-22 of its value in two fp16 terms (bf16 and f16: exact in one); d (n - 8) is exact in two terms,
           and the product of the two small terms, 2^-22, is left out; a sum over D values takes D / 16 tensor-core
           steps for each of three products at most, each within 2 e of the running sum of magnitudes, and a few f32 steps for
           the blocks' scales: |ds| <= (2^-21 + (6 D / 16 + 16) e) A, A = scale * max_c sum |q||k|;
  weights  dp / p <= 2 |ds| + 2^-20 (the exponentials of a weight and of the sum) + 2^-21 (two fp16 terms and the product left out);
  output   a chain of tensor-core sums, each cut by 2 e of its size at most: f32 prompts 4 tiles x 12 products, then one f32
           step for 4 tiles; decode warps two products for 16 cells of a quarter of the cells, and a few f32 steps for the joins:
           (96 + n / 256 + 64) e or (4 (n / 64 + 2) + 64) e; together and rounded up, C e with C = 160 + n / 16;
           and half a step of `type` for the last rounding.
All this is relative to sum p |v| of the output's own channel, so nothing that a row does not see, and no other block's scale,
widens it. 16-bit outputs of the kernel for few rows take codes n = 0..15 as subnormal numbers n 2^-24, which the tensor cores
align as 2^-14, so that a step is cut by 2^-14 2^-24 of the other operand, 2^-18 of a product with n = 15; a block takes two steps
for each of two terms, and starts from -8 sum q: 2^-16 of 15 sum |q| |d_K| for a score, and likewise up to 2^-16 of 15 sum p |d|
for an output, besides; bf16 outputs round weights, and in the kernel for many rows K and V, to one fp16: 2^-10 (A + 1) sum p |v|.
Where a weight is far below the row's largest it is held to 2^-30 of that, which matters only beside scales of
V that differ by as much: 2^-28 max |d| over the visible cells. However far off the scores are, an output is a mean of the
visible values, none of them above 8 max |d|: it is never off by more than twice that.
"""
import numpy as np
import pytest

import kv4_plain as P
import tsrc

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def _attend(q, kb, vb, Hk, scale, ranges, mask, dtype):
    """(values, tolerances) in f64."""
    T, H, D = q.shape
    n = len(kb)
    want, pv, pd, A = P.attend_many(q, kb, vb, Hk, scale, ranges, mask)
    seen = (np.arange(n) >= np.maximum(np.asarray(ranges)[:, :1], 0)) & (np.arange(n) < np.asarray(ranges)[:, 1:])
    if mask is not None:
        seen &= ~np.isneginf(mask.astype(np.float64))
    d = np.abs(np.ascontiguousarray(vb.reshape(n, -1, 18)[..., :2]).view(np.float16).astype(np.float64)).reshape(n, Hk, D // 32)
    most = np.zeros((T, H, D))
    for t in range(T):
        if seen[t].any():
            most[t] = np.repeat(np.repeat(np.nan_to_num(d[seen[t]].max(0), posinf=0.0), 32, -1), H // Hk, 0)
    ds = (2.0 ** -21 + (6 * D / 16 + 16) * E) * A
    if dtype != "float32":
        dk = np.repeat(np.nan_to_num(np.abs(_scales(kb, Hk, D).astype(np.float64)), posinf=0.0), 32, -1)
        for h in range(H):
            ds[:, h, 0] += 2.0 ** -16 * 15 * np.where(seen, abs(scale) * (np.abs(q[:, h]) @ dk[:, h // (H // Hk)].T), 0.0).max(1)
    tol = (2 * ds + 2.0 ** -20 + 2.0 ** -21 + (160 + n / 16) * E) * pv + 2.0 ** -28 * most
    if mask is not None:
        spread = np.zeros((T, 1, 1))
        for t in range(T):
            m = mask[t][seen[t]].astype(np.float64)
            spread[t] = min(float(m.max() - m.min()), 200.0) if len(m) else 0.0
        tol += 8 * E * spread * pv
    if dtype == "float16":
        tol += 2.0 ** -16 * 15 * pd
    if dtype == "bfloat16":
        tol += 2.0 ** -10 * (A + 1) * pv + 2.0 ** -16 * 15 * pd
    return want, np.minimum(tol, 16 * most) + np.maximum(HALF[dtype] * np.abs(want), 2.0 ** -25 if dtype == "float16" else 0.0) + 1e-30


def _run(dev, q, kb, vb, Hk, scale, ranges=None, mask=None, group=0, max_len=0):
    import torch
    T, H, D = q.shape
    kv = dev.kv4_create(Hk, D, len(kb))
    try:
        kv.set_bytes(tsrc.KV_K, kb)
        kv.set_bytes(tsrc.KV_V, vb)
        out = torch.full_like(q, float("nan"))
        dev.flash_attn_q4(kv, q, out, T=T, n_head=H, n_kv=len(kb), scale=scale, group=group, max_len=max_len,
                          ranges=None if ranges is None else torch.from_numpy(np.asarray(ranges, np.int32)).cuda(),
                          mask=None if mask is None else torch.from_numpy(np.ascontiguousarray(mask)).cuda())
        dev.sync()
        return out.double().cpu().numpy()
    finally:
        kv.free()


def _inputs(seed, T, H, Hk, D, n, dtype, q_size=1.0):
    import torch
    rng = np.random.default_rng(seed)
    q = torch.from_numpy((q_size * rng.standard_normal((T, H, D))).astype(np.float32)).to(getattr(torch, dtype)).cuda()
    return rng, q, P.random_rows(rng, n, Hk * D), P.random_rows(rng, n, Hk * D)


def _scales(rows, Hk, D):
    """The rows' scales as f16 [n, Hk, D / 32], to be written back by _set."""
    return np.ascontiguousarray(rows.reshape(len(rows), Hk, D // 32, 18)[..., :2]).view(np.float16)[..., 0].copy()


def _set(rows, Hk, D, d):
    rows.reshape(len(rows), Hk, D // 32, 18)[..., :2] = np.ascontiguousarray(d.astype(np.float16))[..., None].view(np.uint8)


def _check(dev, q, kb, vb, Hk, dtype, ranges, mask=None, scale=0.05, **kw):
    scale = float(np.float32(scale))
    want, tol = _attend(q.double().cpu().numpy(), kb, vb, Hk, scale, ranges, mask, dtype)
    got = _run(dev, q, kb, vb, Hk, scale, ranges, mask, **kw)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), bad.size, float(np.nanmax(np.abs(got - want) / tol)), np.argwhere(bad)[:3].tolist())


# tokens and heads that reach the kernel for few rows, and those for 128 and (bf16) 256 rows
SHAPES = [(1, 8, 2), (5, 32, 8), (300, 32, 8), (1300, 32, 8)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("T,H,Hk", SHAPES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_blocks_of_very_different_scales(dev, dtype, T, H, Hk, D):
    """V's and K's scales fall by 2^0, 2^10, 2^16, 2^13 from block to block of every cell, and by a random power besides; rows
    that see one cell, a few or all."""
    if D == 256 and T == 1300:
        T = 100
    n = 200
    rng, q, kb, vb = _inputs(T + D, T, H, Hk, D, n, dtype, 0.2)
    fall = np.array([0, 10, 16, 13, 5, 11, 15, 3], np.float64)[:D // 32]
    for rows, by in ((kb, fall[::-1]), (vb, fall)):
        _set(rows, Hk, D, 4 * _scales(rows, Hk, D).astype(np.float64) * 2.0 ** -by)
    ranges = [[t % n, t % n + 1] if t % 3 == 0 else [t % (n - 5), t % (n - 5) + 3] if t % 3 == 1 else [0, n] for t in range(T)]
    _check(dev, q, kb, vb, Hk, dtype, ranges)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("T,H,Hk,D,n", [(1, 8, 2, 128, 200), (3, 8, 2, 64, 200), (3, 4, 2, 256, 77), (2, 2, 1, 512, 90), (1, 8, 2, 128, 5000),
                                        (1, 4, 1, 64, 40000), (1, 2, 1, 256, 40000), (300, 32, 8, 64, 200), (1300, 32, 8, 128, 200)])
@pytest.mark.parametrize("bits", [0x7C00, 0xFC00, 0x7E01])
def test_scale_of_v_that_is_not_finite_shows_at_any_weight(dev, dtype, T, H, Hk, D, n, bits):
    """A visible cell whose weight is 0 in any arithmetic, by its score or by a mask of the type's lowest value, in tiles that
    all rows see whole and in others: its block is not finite, and no other output changes."""
    low = np.float16(np.finfo(np.float16).min)
    for masked in (False, True):
        rng, q, kb, vb = _inputs(T + D, T, H, Hk, D, n, dtype)
        q[:] = 1.0
        at = n // 2 + 1
        mask = None
        b = kb.reshape(n, Hk, D // 32, 18)
        b[..., 2:] = 0x88                                             # scores of 0
        if masked:
            mask = np.zeros((T, n), np.float16)
            mask[:, at] = low
        else:
            b[at, ..., 2:] = 0x00                                     # n - 8 = -8, 32 times a block
            _set(kb, Hk, D, np.where((np.arange(n) == at)[:, None, None], 1.0, _scales(kb, Hk, D)))
        ranges = [[0, n - 3] if t % 2 == 0 else [3, n // 2] for t in range(T)]
        clean = _run(dev, q, kb, vb, Hk, 0.5, ranges, mask)
        vb.reshape(n, Hk, D // 32, 18)[at, Hk - 1, 1, :2] = np.array([bits & 255, bits >> 8], np.uint8)
        got = _run(dev, q, kb, vb, Hk, 0.5, ranges, mask)
        lost = np.zeros(got.shape, bool)
        lost[::2, H - H // Hk:, 32:64] = True
        assert not np.isfinite(got[lost]).any()
        np.testing.assert_array_equal(got[~lost], clean[~lost])


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("T,H,Hk", SHAPES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_size_of_what_is_hidden_has_no_effect(dev, dtype, T, H, Hk, D, masked):
    """Small cells seen beside hidden cells of large finite scales, each row with cells of its own."""
    if D == 256 and T == 1300:
        T = 100
    n = 160
    for large in (20.0, 1000.0, 65504.0):
        rng, q, kb, vb = _inputs(T + D, T, H, Hk, D, n, dtype)
        q *= 64
        big = np.arange(n) % 5 == 4
        for rows in (kb, vb):
            d = _scales(rows, Hk, D).astype(np.float64) * 2.0 ** -9
            d[big] = large
            _set(rows, Hk, D, d)
        if masked:
            mask = np.where(rng.random((T, n)) < 0.5, -np.inf, 0.0).astype(np.float16)
            mask[:, big] = -np.inf
            _check(dev, q, kb, vb, Hk, dtype, [[0, n]] * T, mask)
        else:
            ranges = [[5 * (t % (n // 5)) + t % 3, 5 * (t % (n // 5)) + 4] for t in range(T)]
            _check(dev, q, kb, vb, Hk, dtype, ranges)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T,H,Hk", SHAPES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_largest_and_smallest_queries(dev, dtype, T, H, Hk, D):
    """Queries near the type's largest and smallest values, with a scale that makes ordinary scores of them, and with keys of 0."""
    if D == 256 and T == 1300:
        T = 100
    n = 90
    ranges = [[t % 7, n] for t in range(T)]
    for size, scale in ((2.0 ** 120, 2.0 ** -123), (2.0 ** 124, 2.0 ** -60), (2.0 ** -70, 2.0 ** 66), (2.0 ** -84, 2.0 ** 81)):
        _, q, kb, vb = _inputs(T + D, T, H, Hk, D, n, dtype)
        q *= size
        if scale == 2.0 ** -60:                                      # scores of 0, whatever the factor
            kb.reshape(n, -1, 18)[..., 2:] = 0x88
            for s in (scale, 2.0 ** 100, -2.0 ** 100):
                _check(dev, q, kb, vb, Hk, dtype, ranges, scale=s)
        else:
            _check(dev, q, kb, vb, Hk, dtype, ranges, scale=scale)
