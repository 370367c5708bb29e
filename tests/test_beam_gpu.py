"""Beam selection on the GPU against numpy in 64 bits.

Beams, tokens and their order are equal. A score's error is that of the normaliser: a sum of positive terms, each
exponential within 2^-21 of its value (its argument, up to 2^5, is rounded to 2^-24 of itself, and the function
itself is within 2^-22), added in at most 37 f32 steps of 2^-24, so log(sum) is within 2^-18; then one rounding of
the score to f32. Inputs are drawn so that neighbouring scores lie further apart than that, or are exactly equal.
"""
import numpy as np
import pytest

import kv4_plain as P
import tsrc

pytestmark = pytest.mark.gpu


def _select(dev, x, scores, G, B, V, n_out, stride=0, stream=None):
    import torch
    s = torch.full((G, n_out), 99.0, device="cuda")
    b, t = (torch.full((G, n_out), 99, dtype=torch.int32, device="cuda") for _ in range(2))
    dev.beam_select(x, scores, s, b, t, n_group=G, n_beam=B, n_vocab=V, n_out=n_out, stride=stride, stream=stream)
    dev.sync()
    return s.cpu().numpy(), b.cpu().numpy(), t.cpu().numpy()


def _check(got, want):
    np.testing.assert_array_equal(got[1], want[1])
    np.testing.assert_array_equal(got[2], want[2])
    fin = np.isfinite(want[0])
    np.testing.assert_array_equal(np.isneginf(got[0]), ~fin)
    assert np.all(np.abs(got[0][fin] - want[0][fin]) <= 2.0 ** -18 + np.abs(want[0][fin]) * 2.0 ** -24)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("G,B,V,n_out", [(1, 1, 1, 1), (1, 1, 5, 8), (2, 3, 31, 6), (1, 4, 8192, 8), (3, 2, 8193, 64), (2, 5, 20001, 10),
                                         (1, 64, 300, 64), (1, 4, 151936, 8), (5, 8, 32000, 16), (1, 33, 1000, 33)])
def test_against_numpy(dev, dtype, G, B, V, n_out):
    import torch
    rng = np.random.default_rng(G * 1000 + V)
    x = torch.from_numpy((3 * rng.standard_normal((G, B, V))).astype(np.float32)).to(getattr(torch, dtype)).cuda()
    scores = torch.from_numpy((-10 * rng.random((G, B))).astype(np.float32)).cuda()
    got = _select(dev, x, scores, G, B, V, n_out)
    _check(got, P.beam(x.double().cpu().numpy(), scores.double().cpu().numpy(), n_out))


def test_no_scores_strides_and_odd_rows(dev):
    import torch
    rng = np.random.default_rng(3)
    G, B, V, stride = 2, 3, 1001, 1007
    flat = torch.from_numpy(rng.standard_normal(G * B * stride + 1).astype(np.float32)).cuda()
    x = flat[1:]                                                   # rows start off every wide boundary
    got = _select(dev, x, None, G, B, V, 7, stride=stride)
    rows = x.double().cpu().numpy().reshape(G, B, stride)[..., :V]
    _check(got, P.beam(rows, np.zeros((G, B)), 7))


def test_ties_go_to_the_lowest_beam_and_token(dev):
    """All logits equal (every key ties), rows that repeat, and a first step whose beams are all alike."""
    import torch
    for V in (3, 300, 20000):
        x = torch.full((1, 4, V), 1.5, device="cuda")
        s, b, t = _select(dev, x, None, 1, 4, V, 10)
        k = np.arange(10)
        np.testing.assert_array_equal(b[0], k // V)
        np.testing.assert_array_equal(t[0], k % V)
    x = torch.randn(1, 1, 9000, device="cuda").repeat(1, 4, 1).contiguous()
    x[..., 17] = x[..., 8999] = 9.0
    s, b, t = _select(dev, x, torch.full((1, 4), -2.0, device="cuda"), 1, 4, 9000, 8)
    np.testing.assert_array_equal(b[0], [0, 0, 1, 1, 2, 2, 3, 3])
    np.testing.assert_array_equal(t[0], [17, 8999] * 4)
    x = torch.zeros(1, 2, 40, device="cuda")
    x[0, 0, 5] = -0.0                                              # -0 ties with 0
    s, b, t = _select(dev, x, None, 1, 2, 40, 6)
    np.testing.assert_array_equal(t[0], np.arange(6))


def test_sorted_rows_overflow_the_first_bound(dev):
    """Ascending and descending logits put all of a part's best into few threads."""
    import torch
    up = torch.linspace(-4, 4, 16384, device="cuda")
    x = torch.stack([up, up.flip(0), up.view(32, -1).t().flatten()])[None].contiguous()
    for n_out in (1, 3, 64):
        got = _select(dev, x, torch.tensor([[0.0, -1e-3, -2e-3]], device="cuda"), 1, 3, 16384, n_out)
        want = P.beam(x.double().cpu().numpy(), np.array([[0.0, np.float32(-1e-3), np.float32(-2e-3)]]), n_out)
        _check(got, want)


def test_banned_tokens_dead_beams_and_bad_rows(dev):
    import torch
    rng = np.random.default_rng(4)
    x = rng.standard_normal((2, 4, 500)).astype(np.float32)
    x[0, 0, :] = -np.inf                                           # a beam whose every token is banned
    x[0, 1, 3:] = -np.inf                                          # three tokens left
    x[0, 2, 7] = np.nan                                            # a broken row
    x[0, 3, 9] = np.inf
    scores = np.zeros((2, 4), np.float32)
    scores[1, 1:] = -np.inf                                        # a first step: one live beam
    scores[1, 2] = np.nan
    got = _select(dev, torch.from_numpy(x).cuda(), torch.from_numpy(scores).cuda(), 2, 4, 500, 8)
    _check(got, P.beam(x.astype(np.float64), scores.astype(np.float64), 8))
    assert (got[1][0, 3:] == -1).all() and (got[1][1] == 0).all()
    x[:] = np.float32(-3e38)                                       # far from 0, all alike
    x[0, 1, 6] = np.float32(-2.9e38)
    got = _select(dev, torch.from_numpy(x).cuda(), None, 2, 4, 500, 2)
    np.testing.assert_array_equal(got[1][0], [1, 0])
    np.testing.assert_array_equal(got[2][0], [6, 0])


def test_large_offsets_do_not_lose_the_sum(dev):
    """Parts that are all -inf beside parts far below 0."""
    import torch
    x = np.full((1, 2, 20000), -np.inf, np.float32)
    x[0, :, 8192:] = np.random.default_rng(5).standard_normal((2, 20000 - 8192)).astype(np.float32) - 900.0
    got = _select(dev, torch.from_numpy(x).cuda(), None, 1, 2, 20000, 9)
    _check(got, P.beam(x.astype(np.float64), np.zeros((1, 2)), 9))


def test_captured_and_replayed_on_another_stream(dev):
    import torch
    G, B, V, n_out = 2, 4, 9001, 8
    x = torch.randn(G, B, V, device="cuda")
    scores = torch.zeros(G, B, device="cuda")
    s = torch.zeros(G, n_out, device="cuda")
    b, t = (torch.zeros(G, n_out, dtype=torch.int32, device="cuda") for _ in range(2))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        dev.beam_select(x, scores, s, b, t, n_group=G, n_beam=B, n_vocab=V, n_out=n_out)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dev.beam_select(x, scores, s, b, t, n_group=G, n_beam=B, n_vocab=V, n_out=n_out)
    for seed in (1, 2):
        x.copy_(torch.randn(G, B, V, generator=torch.Generator().manual_seed(seed)))
        scores.copy_(torch.randn(G, B, generator=torch.Generator().manual_seed(seed)))
        g.replay()
        torch.cuda.synchronize()
        _check((s.cpu().numpy(), b.cpu().numpy(), t.cpu().numpy()), P.beam(x.double().cpu().numpy(), scores.double().cpu().numpy(), n_out))
    del g


def test_refusals(dev):
    import torch
    x = torch.zeros(4, 100, device="cuda")
    s = torch.zeros(1, 8, device="cuda")
    b, t = (torch.zeros(1, 8, dtype=torch.int32, device="cuda") for _ in range(2))

    def call(**kw):
        a = dict(n_group=1, n_beam=4, n_vocab=100, n_out=8) | kw
        x_ = a.pop("x", x)
        dev.beam_select(x_, None, a.pop("s", s), b, t, **a)

    call()
    for kw in (dict(n_out=0), dict(n_out=65), dict(n_beam=0), dict(n_beam=65), dict(n_vocab=0), dict(stride=99), dict(x=x.double()),
               dict(s=s.double()), dict(n_group=20000), dict(workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(tsrc.TsrcError) as e:
            call(**kw)
        assert e.value.code in (tsrc.E_ARG, tsrc.E_SHAPE)
    call(n_group=0)
    dev.sync()
