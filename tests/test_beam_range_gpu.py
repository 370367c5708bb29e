"""Beam selection over its whole range of vocabularies and row addresses, against 64 bits.

Order and tokens are equal; scores within test_beam_gpu's bound: 2^-18 for the normaliser and one rounding to f32.
"""
import numpy as np
import pytest

import kv4_plain as P

pytestmark = pytest.mark.gpu


def _select(dev, x, scores, G, B, V, n_out, stride=0):
    import torch
    s = torch.full((G, n_out), 99.0, device="cuda")
    b, t = (torch.full((G, n_out), 99, dtype=torch.int32, device="cuda") for _ in range(2))
    dev.beam_select(x, scores, s, b, t, n_group=G, n_beam=B, n_vocab=V, n_out=n_out, stride=stride)
    dev.sync()
    return s.cpu().numpy(), b.cpu().numpy(), t.cpu().numpy()


@pytest.mark.parametrize("dtype,V", [("float16", 50257), ("bfloat16", 1001), ("float32", 9001), ("float16", 20003), ("bfloat16", 33)])
def test_alike_rows_tie_wherever_they_lie(dev, dtype, V):
    """Rows of an odd length, all alike with alike scores: every row starts at another offset from a wide boundary, and the
    candidates of one token still tie, so that they come out by ascending beam with the same score."""
    import torch
    B, n_out = 8, 24
    row = torch.from_numpy(3 * np.random.default_rng(V).standard_normal(V).astype(np.float32)).to(getattr(torch, dtype))
    x = row.repeat(B).view(1, B, V).cuda()
    scores = torch.full((1, B), -2.0, device="cuda")
    got = _select(dev, x, scores, 1, B, V, n_out)
    want = P.beam(x.double().cpu().numpy(), scores.double().cpu().numpy(), n_out)
    np.testing.assert_array_equal(got[1], want[1])
    np.testing.assert_array_equal(got[2], want[2])
    same = got[0].reshape(-1, 8)
    if len(set(row.double().topk(4)[0].tolist())) == 4:             # the best tokens' logits differ: eights of one score
        np.testing.assert_array_equal(same, np.repeat(same[:, :1], 8, 1))
    # one row at a time, at every offset from a wide boundary, gives the same bits
    flat = torch.zeros(V + 16, dtype=row.dtype, device="cuda")
    alone = None
    for off in range(8):
        flat[off:off + V] = row.cuda()
        one = _select(dev, flat[off:], None, 1, 1, V, 8)
        alone = alone or one
        for a, b in zip(one, alone):
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("V", [262137, 262138, 262145, 524282, 524288, 1048569, 1048570, 1 << 20])
@pytest.mark.parametrize("kind", ["scattered", "ascending", "tied"])
def test_largest_vocabularies(dev, V, kind):
    """Where groups of 32 neighbours become groups of 64 and 128; rows on and off a wide boundary."""
    import torch
    if kind == "scattered":
        row = 3 * torch.randn(V, generator=torch.Generator().manual_seed(V))
    elif kind == "ascending":
        row = torch.linspace(-8, 8, V)
    else:
        row = torch.zeros(V)
    buf = torch.zeros(V + 16, device="cuda")
    value, at = row.double().sort(descending=True, stable=True)
    norm = row.double().logsumexp(0)
    want = (value[:64] - norm).numpy()
    for off in (0, 3):
        buf[off:off + V] = row.cuda()
        for n_out in (1, 32, 33, 64):
            s, b, t = _select(dev, buf[off:], None, 1, 1, V, n_out)
            np.testing.assert_array_equal(t[0], at[:n_out].numpy())
            assert (b == 0).all()
            assert (np.abs(s[0] - want[:n_out]) <= 2.0 ** -18 + np.abs(want[:n_out]) * 2.0 ** -24).all()
    for dtype in (torch.float16, torch.bfloat16):
        x = row.to(dtype)
        value, at = x.double().sort(descending=True, stable=True)
        _, _, t = _select(dev, x.cuda(), None, 1, 1, V, 64)
        np.testing.assert_array_equal(t[0], at[:64].numpy())
