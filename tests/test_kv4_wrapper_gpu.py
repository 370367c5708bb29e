"""The q4_0 cache's calls on tensors that are rows of a wider matrix: the same bits as on dense copies, nothing else written."""
import numpy as np
import pytest

import kv4_plain as P
import tsrc

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T", [3, 200])
def test_rows_of_a_fused_projection(dev, dtype, T):
    import torch
    H, Hk, D, V = 4, 2, 64, 1001
    E = Hk * D
    torch.manual_seed(T)
    fused = torch.randn(T, H * D + 2 * E, device="cuda").to(getattr(torch, dtype))
    q, k, v = fused.split([H * D, E, E], 1)
    res = []
    for dense in (False, True):
        kv = dev.kv4_create(Hk, D, T)
        try:
            f = (lambda t: t.contiguous()) if dense else (lambda t: t)
            kv.set_rows(f(k), f(v))
            wide = torch.full((T, 2, H, D), 5.0, dtype=q.dtype, device="cuda")
            out = wide[:, 1] if not dense else torch.empty(T, H, D, dtype=q.dtype, device="cuda")
            dev.flash_attn_q4(kv, f(q), out, T=T, n_head=H, n_kv=T, scale=0.1)
            back = torch.full((T, 3, E), 5.0, dtype=q.dtype, device="cuda")
            kb, vb = (back[:, 0], back[:, 2]) if not dense else (torch.empty(T, E, dtype=q.dtype, device="cuda") for _ in range(2))
            kv.get_rows(kb, vb)
            padded = torch.randn(4, V + 23, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")[:, :V]
            s = torch.zeros(1, 8, device="cuda")
            b, t = (torch.zeros(1, 8, dtype=torch.int32, device="cuda") for _ in range(2))
            dev.beam_select(f(padded), None, s, b, t, n_group=1, n_beam=4, n_vocab=V, n_out=8)
            dev.sync()
            res.append([x.clone() for x in (out, kb, vb, s, b, t)])
            assert (wide[:, 0] == 5).all() and (back[:, 1] == 5).all()
        finally:
            kv.free()
    for a, b in zip(*res):
        assert torch.equal(a, b)


def test_reorder_by_a_selection_of_twice_the_beams(dev):
    """Several groups, n_out = 2 n_beam: the first n_beam entries of each group go on, gathered."""
    import torch
    rng = np.random.default_rng(8)
    G, B, V, cap = 3, 4, 500, 8
    kv = dev.kv4_create(1, 64, G * B * cap)
    try:
        img = rng.integers(0, 256, (G * B * cap, kv.row_bytes), dtype=np.uint8)
        kv.set_bytes(tsrc.KV_K, img)
        x = torch.from_numpy(rng.standard_normal((G, B, V)).astype(np.float32)).cuda()
        s = torch.empty(G, 2 * B, device="cuda")
        b, t = (torch.empty(G, 2 * B, dtype=torch.int32, device="cuda") for _ in range(2))
        dev.beam_select(x, None, s, b, t, n_group=G, n_beam=B, n_vocab=V, n_out=2 * B)
        with pytest.raises(tsrc.TsrcError):
            kv.reorder(b, G, B, cap, cap)
        kv.reorder(b[:, :B].contiguous(), G, B, cap, cap)
        dev.sync()
        parent = P.beam(x.double().cpu().numpy(), np.zeros((G, B)), 2 * B)[1][:, :B]
        want = img.reshape(G, B, -1)[np.arange(G)[:, None], parent].reshape(img.shape)
        np.testing.assert_array_equal(kv.get_bytes(tsrc.KV_K), want)
    finally:
        kv.free()
