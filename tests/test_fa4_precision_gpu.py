"""f32 outputs of the attention over the q4_0 cache held to f32's own arithmetic, short windows and long rows, and shapes that no other
test reaches: prompts at head sizes 256 and 512, several groups of 256-row CTAs."""
import numpy as np
import pytest

import kv4_bounds as B
import kv4_plain as P
import test_fa4_content_gpu as C

pytestmark = pytest.mark.gpu


def _check(dev, q, kb, vb, Hk, ranges, chain, mask=None, scale=0.05, spread=0.0, **kw):
    scale = float(np.float32(scale))
    want, pv, A = B.attend64(q, kb, vb, Hk, scale, ranges, mask)
    got = C._run(dev, q, kb, vb, Hk, scale, ranges, mask, **kw)
    tol = B.bound_f32(pv, A, q.shape[2], chain, spread) + B.E * np.abs(want) + 1e-30
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), bad.size, float(np.nanmax(np.abs(got - want) / tol)), np.argwhere(bad)[:3].tolist())


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("T,H,Hk", C.SHAPES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_short_windows_of_a_long_cache(dev, T, H, Hk, D, masked):
    """A few cells each: every weight's second term counts. Without a mask windows anywhere; with one, the visible cells lie in
    a stretch of 64, apart."""
    n = 4200 if T < 300 else 2100
    T = min(T, 300) if D == 256 else T
    rng, q, kb, vb = C._inputs(T + D, T, H, Hk, D, n, "float32", 0.2)
    lo = rng.integers(0, n - 64, T)
    if masked:
        mask = np.full((T, n), -np.inf, np.float16)
        for t in range(T):
            mask[t, lo[t] + rng.choice(64, 1 + t % 12, replace=False)] = -rng.random(1 + t % 12)
        _check(dev, q, kb, vb, Hk, [[0, n]] * T, B.chain_many(64), mask, spread=1.0)
    else:
        _check(dev, q, kb, vb, Hk, np.stack([lo, lo + 2 + rng.integers(0, 7, T)], 1), B.chain_many(64))


def _one_sign(vb):
    b = vb.reshape(len(vb), -1, 18)
    b[..., 2:] |= 0x99
    b[..., 1] &= 0x7F


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("H,Hk,D,T,n", [(75, 75, 64, 150, 4500), (40, 40, 128, 500, 3000), (32, 8, 128, 100, 9000)])
def test_long_rows_of_one_sign_many(dev, H, Hk, D, T, n, masked):
    """Flat weights over all cells, values of one sign: every cut of a sum adds to the last. All cells in one split, or some."""
    rng, q, kb, vb = C._inputs(n, T, H, Hk, D, n, "float32", 0.2)
    _one_sign(vb)
    mask = np.where(rng.random((T, n)) < 0.2, -np.inf, 0.0).astype(np.float16) if masked else None
    _check(dev, q, kb, vb, Hk, [[0, n]] * T, B.chain_many(n), mask, scale=1e-3)


@pytest.mark.parametrize("H,Hk,D,T,group,n", [(8, 8, 128, 80, 1, 9000), (8, 1, 64, 1, 1, 9000), (32, 8, 128, 1, 0, 20000), (1, 1, 64, 1, 0, 70000),
                                              (16, 4, 256, 40, 1, 3000), (8, 2, 512, 80, 1, 2000)])
def test_long_rows_of_one_sign_few(dev, H, Hk, D, T, group, n):
    """The same for few rows: one CTA for all cells, clusters, and splits with a merge."""
    _, q, kb, vb = C._inputs(n, T, H, Hk, D, n, "float32", 0.2)
    _one_sign(vb)
    _check(dev, q, kb, vb, Hk, [[0, n - t % 3] for t in range(T)], B.chain_few(n), scale=1e-3, group=group)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("H,Hk,D,T,n", [(16, 4, 256, 300, 400), (8, 2, 512, 300, 300), (6, 1, 256, 513, 513)])
def test_prompts_at_large_head_sizes(dev, dtype, H, Hk, D, T, n):
    _, q, kb, vb = C._inputs(T + D, T, H, Hk, D, n, dtype)
    C._check(dev, q, kb, vb, Hk, dtype, [[0, n - T + t + 1] for t in range(T)])


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("S,g,H,Hk,D,cap", [(4, 300, 32, 8, 128, 310), (3, 500, 28, 4, 64, 500), (5, 131, 32, 8, 64, 200)])
def test_several_prompts_in_a_call(dev, dtype, S, g, H, Hk, D, cap, masked):
    """Groups of one length over stretches of their own, causal, with CTAs of 128 and 256 rows whose last rows are another group's
    nothing."""
    T, n = S * g, S * cap
    rng, q, kb, vb = C._inputs(T, T, H, Hk, D, n, dtype)
    ranges = [[s * cap, s * cap + cap - g + j + 1 - 3 * s] for s in range(S) for j in range(g)]
    mask = np.where(rng.random((T, n)) < 0.3, -np.inf, -rng.random((T, n))).astype(np.float16) if masked else None
    C._check(dev, q, kb, vb, Hk, dtype, ranges, mask, group=g, max_len=cap)
