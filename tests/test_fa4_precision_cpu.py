"""What the bound on f32 outputs notices, with the mistake planted in the 64-bit form: a weight, a value or a query held to one
fp16 term, sums of tensor-core steps that no f32 addition relieves."""
import numpy as np
import pytest

import kv4_bounds as B
import kv4_plain as P

torch = pytest.importorskip("torch")


def _case(seed, T, H, D, n, window):
    rng = np.random.default_rng(seed)
    q = torch.from_numpy((0.2 * rng.standard_normal((T, H, D))).astype(np.float32))
    kb, vb = (P.random_rows(rng, n, H * D) for _ in range(2))
    lo = rng.integers(0, n - window, T)
    ranges = np.stack([lo, lo + rng.integers(2, window + 1, T)], 1)
    return q, kb, vb, ranges


def _one(x):
    return x.astype(np.float32).astype(np.float16).astype(np.float64)


@pytest.mark.parametrize("what", ["nothing", "weights", "values", "queries"])
@pytest.mark.parametrize("D", [64, 128])
def test_a_missing_second_term_is_noticed(what, D):
    T, H, n, scale = 60, 2, 500, 0.05
    q, kb, vb, ranges = _case(D, T, H, D, n, 8)
    want, pv, A = B.attend64(q, kb, vb, H, scale, ranges)
    tol = B.bound_f32(pv, A, D, B.chain_few(64)) + B.E * np.abs(want)
    got = np.zeros_like(want)
    k, v = (P.unpack(b).reshape(n, H, D) for b in (kb, vb))
    x = q.double().numpy()
    for t, (lo, hi) in enumerate(ranges):
        for h in range(H):
            qh = _one(x[t, h]) if what == "queries" else x[t, h]
            s = k[lo:hi, h] @ qh * scale
            p = np.exp(s - s.max())
            vh = _one(v[lo:hi, h]) if what == "values" else v[lo:hi, h]
            got[t, h] = (_one(64 * p) / 64 if what == "weights" else p) @ vh / p.sum()
    off = (np.abs(got - want) > tol).mean()
    assert off == 0 if what == "nothing" else off > 0.03, off


@pytest.mark.parametrize("D", [64, 128])
def test_an_unrelieved_sum_is_noticed(D):
    """4500 cells without a total: 71 tiles of 12 products, each cut by 2^-25 in the mean."""
    q, kb, vb, _ = _case(D, 4, 1, D, 4500, 8)
    vb.reshape(4500, -1, 18)[..., 2:] |= 0x99                        # codes 9 and above: values of one sign
    vb.reshape(4500, -1, 18)[..., 1] &= 0x7F
    want, pv, A = B.attend64(q, kb, vb, 1, 1e-4, [[0, 4500]] * 4)
    tol = B.bound_f32(pv, A, D, B.chain_many(4500)) + B.E * np.abs(want)
    assert (np.abs(want * 71 * 12 * 2.0 ** -25) > tol).all()
