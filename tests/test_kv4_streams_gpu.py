"""The q4_0 cache's attention and beam selection on a stream that the call names, as an object and as a raw handle."""
import numpy as np
import pytest

import kv4_plain as P
import tsrc

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("raw", [False, True])
def test_named_streams(dev, raw):
    """Results as on the current stream, while work queued on the current stream still writes into blocks freed before."""
    import torch
    rng = np.random.default_rng(12)
    T, H, Hk, D, n, V = 70, 32, 8, 128, 3000, 9001
    kb, vb = (P.random_rows(rng, n, Hk * D) for _ in range(2))
    q = torch.from_numpy(rng.standard_normal((T, H, D)).astype(np.float32)).cuda()
    x = torch.from_numpy(rng.standard_normal((4, V)).astype(np.float32)).cuda()
    need = tsrc.lib().tsrc_flash_attn_q4_workspace(tsrc.TYPE_F32, Hk, D, T, H, n, 0, 0)
    assert need > 0
    side = torch.cuda.Stream()
    kv = dev.kv4_create(Hk, D, n)
    try:
        kv.set_bytes(tsrc.KV_K, kb)
        kv.set_bytes(tsrc.KV_V, vb)

        def both(stream):
            out = torch.zeros_like(q)
            s = torch.zeros(1, 8, device="cuda")
            b, t = (torch.zeros(1, 8, dtype=torch.int32, device="cuda") for _ in range(2))
            torch.cuda.synchronize()
            if stream is not None:
                junk = [torch.empty(need, dtype=torch.uint8, device="cuda") for _ in range(2)]
                for _ in range(50):
                    for j in junk:
                        j.fill_(255)
                del junk, j                                        # free for the current stream, whose fills still run
            dev.flash_attn_q4(kv, q, out, T=T, n_head=H, n_kv=n, scale=0.1, stream=stream)
            dev.beam_select(x, None, s, b, t, n_group=1, n_beam=4, n_vocab=V, n_out=8, stream=stream)
            torch.cuda.synchronize()
            return out, s, b, t

        want = both(None)
        for _ in range(3):
            for a, b in zip(both(side.cuda_stream if raw else side), want):
                assert torch.equal(a, b)
        dev.sync()
    finally:
        kv.free()
