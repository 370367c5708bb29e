"""The q4_0 KV cache on the GPU: stored rows, rows read back, the ggml image and the reordering, against numpy.

Codes and scales are compared bit for bit: every step of the format is one f32 rounding. Values read back are
d (n - 8), exact in f32 (11 + 4 bits), so they too are equal after their one rounding.
"""
import numpy as np
import pytest

import kv4_plain as P
import tsrc

pytestmark = pytest.mark.gpu

GEOMETRIES = [(1, 64), (3, 64), (8, 128), (1, 128), (2, 256), (1, 512)]
DTYPES = ["float32", "float16", "bfloat16"]


def _rows(seed, n, E, dtype):
    import torch
    x = torch.from_numpy(np.random.default_rng(seed).standard_normal((n, E)).astype(np.float32))
    return x.to(getattr(torch, dtype)).cuda()


def _f32(t):
    return t.float().cpu().numpy()


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_store_and_read(dev, heads, dim, dtype):
    import torch
    E, cells = heads * dim, 77
    kv = dev.kv4_create(heads, dim, cells)
    try:
        for n, cell0 in ((1, 0), (1, 76), (33, 5), (77, 0)):
            k, v = (_rows(s + n, n, E, dtype) for s in (1, 2))
            kv.set_rows(k, v, cell0=cell0)
            for which, x in ((tsrc.KV_K, k), (tsrc.KV_V, v)):
                want = P.pack(*P.quantise(_f32(x)))
                np.testing.assert_array_equal(kv.get_bytes(which, cell0, n), want)
                got = torch.full((n, E), float("nan"), dtype=x.dtype, device="cuda")
                kv.get_rows(*((got, None) if which == tsrc.KV_K else (None, got)), cell0=cell0)
                exact = torch.from_numpy(P.unpack(want)).float().to(x.dtype)
                assert torch.equal(got.cpu(), exact)
        dev.sync()
    finally:
        kv.free()


def test_scattered_cells_strides_and_odd_addresses(dev):
    """Cells in any order, rows inside a wider matrix, rows that start off a four-value boundary."""
    import torch
    heads, dim, cells, n = 2, 64, 50, 21
    E = heads * dim
    rng = np.random.default_rng(5)
    cell = torch.from_numpy(rng.permutation(cells)[:n].astype(np.int64)).cuda()
    for off, stride in ((0, E), (4, E + 12), (1, E + 3), (3, 2 * E)):
        kv = dev.kv4_create(heads, dim, cells)
        try:
            wide = _rows(off + 9, n + 1, stride, "float32").flatten()
            k = wide[off:]
            kv.set_rows(k, None, n=n, cells=cell, row_stride=stride)
            x = np.lib.stride_tricks.as_strided(_f32(wide)[off:], (n, E), (stride * 4, 4)).copy()
            img = kv.get_bytes(tsrc.KV_K)
            np.testing.assert_array_equal(img[cell.cpu().numpy()], P.pack(*P.quantise(x)))
            rest = np.setdiff1d(np.arange(cells), cell.cpu().numpy())
            assert not img[rest].any() and not kv.get_bytes(tsrc.KV_V).any()
            again = torch.cat([cell, cell[:2]])                  # a cell may be read twice
            out = torch.full(((n + 3) * stride,), 7.0, device="cuda")
            kv.get_rows(out[off:], None, n=n + 2, cells=again, row_stride=stride)
            got = out[off:].cpu().numpy()
            vals = P.unpack(P.pack(*P.quantise(x)))
            for i in range(n + 2):
                np.testing.assert_array_equal(got[i * stride:i * stride + E], vals[i % n].astype(np.float32))
                assert (got[i * stride + E:(i + 1) * stride] == 7.0).all()        # nothing between rows is written
            dev.sync()
        finally:
            kv.free()


def test_special_values(dev):
    """NaN, infinities, zeros, subnormals, overflowing scales and ties of opposite sign."""
    import torch
    x = np.random.default_rng(6).standard_normal((8, 64)).astype(np.float32)
    x[0, 3] = np.nan
    x[1, 5] = np.inf
    x[2, :32] = 0.0
    x[3, :32] = np.float32(1e-41)
    x[4, :] = np.float32(3e38)
    x[4, 7] = -x[4, 7]
    x[5, 2], x[5, 20] = -9.0, 9.0
    x[6, 9], x[6, 10] = 9.0, -9.0
    x[7, :] = np.nan
    kv = dev.kv4_create(1, 64, 8)
    try:
        kv.set_rows(torch.from_numpy(x).cuda(), torch.from_numpy(x).cuda())
        want = P.pack(*P.quantise(x))
        np.testing.assert_array_equal(kv.get_bytes(tsrc.KV_K), want)
        np.testing.assert_array_equal(kv.get_bytes(tsrc.KV_V), want)
        got = torch.zeros(8, 64, device="cuda")
        kv.get_rows(got, None)
        np.testing.assert_array_equal(got.cpu().numpy(), P.unpack(want).astype(np.float32))
    finally:
        kv.free()


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_bytes_round_trip(dev, heads, dim):
    import torch
    rng = np.random.default_rng(7)
    kv = dev.kv4_create(heads, dim, 70)
    try:
        img = rng.integers(0, 256, (70, kv.row_bytes), dtype=np.uint8)
        kv.set_bytes(tsrc.KV_V, img)
        np.testing.assert_array_equal(kv.get_bytes(tsrc.KV_V), img)
        part = rng.integers(0, 256, (5, kv.row_bytes), dtype=np.uint8)
        kv.set_bytes(tsrc.KV_V, torch.from_numpy(part).cuda(), cell0=64)
        img[64:69] = part
        np.testing.assert_array_equal(kv.get_bytes(tsrc.KV_V), img)
        np.testing.assert_array_equal(kv.get_bytes(tsrc.KV_V, 63, 4), img[63:67])
        assert not kv.get_bytes(tsrc.KV_K).any()
    finally:
        kv.free()


@pytest.mark.parametrize("heads,dim", [(2, 64), (3, 128), (1, 512)])
@pytest.mark.parametrize("groups,beams,cell0,stride,n", [(1, 1, 0, 4, 4), (1, 4, 3, 9, 7), (2, 8, 1, 5, 5), (3, 12, 0, 3, 1), (1, 32, 2, 2, 2)])
def test_reorder(dev, heads, dim, groups, beams, cell0, stride, n):
    import torch
    rng = np.random.default_rng(groups * 100 + beams)
    cells = cell0 + groups * beams * stride + 5
    kv = dev.kv4_create(heads, dim, cells)
    try:
        for parents in (rng.integers(0, beams, (groups, beams)), np.tile(np.roll(np.arange(beams), 1), (groups, 1)),
                        np.zeros((groups, beams), int), np.where(rng.random((groups, beams)) < 0.5, -1, rng.integers(0, beams, (groups, beams)))):
            img = {w: rng.integers(0, 256, (cells, kv.row_bytes), dtype=np.uint8) for w in (tsrc.KV_K, tsrc.KV_V)}
            for w, b in img.items():
                kv.set_bytes(w, b)
            kv.reorder(torch.from_numpy(parents.astype(np.int32)).cuda(), groups, beams, stride, n, cell0=cell0)
            dev.sync()
            for w, b in img.items():
                want = b.copy()
                for g in range(groups):
                    for s in range(beams):
                        if parents[g, s] >= 0:
                            to, fr = (cell0 + (g * beams + x) * stride for x in (s, parents[g, s]))
                            want[to:to + n] = b[fr:fr + n]
                np.testing.assert_array_equal(kv.get_bytes(w), want)
    finally:
        kv.free()


def test_bad_device_side_indexes_are_reported_and_harmless(dev):
    import torch
    kv = dev.kv4_create(1, 64, 10)
    try:
        img = np.random.default_rng(8).integers(0, 256, (10, kv.row_bytes), dtype=np.uint8)
        kv.set_bytes(tsrc.KV_K, img)
        rows = torch.randn(3, 64, device="cuda")
        kv.set_rows(rows, None, cells=torch.tensor([10, -1, 4], device="cuda"))
        with pytest.raises(tsrc.TsrcError) as e:
            dev.sync()
        assert e.value.code == tsrc.E_ARG and "set_rows" in str(e.value)
        dev.sync()                                                # the report was cleared
        img[4] = P.pack(*P.quantise(rows.cpu().numpy()))[2]
        np.testing.assert_array_equal(kv.get_bytes(tsrc.KV_K), img)
        out = torch.full((3, 64), 5.0, device="cuda")
        kv.get_rows(out, None, cells=torch.tensor([1 << 40, 4, 12], device="cuda"))
        with pytest.raises(tsrc.TsrcError):
            dev.sync()
        assert (out[0] == 5).all() and (out[2] == 5).all()
        np.testing.assert_array_equal(out[1].cpu().numpy(), P.unpack(img[4:5])[0].astype(np.float32))
        kv.reorder(torch.tensor([7, 0], dtype=torch.int32, device="cuda"), 1, 2, 5, 5)
        with pytest.raises(tsrc.TsrcError) as e:
            dev.sync()
        assert "parent" in str(e.value)
        want = img.copy()
        want[5:] = img[:5]
        np.testing.assert_array_equal(kv.get_bytes(tsrc.KV_K), want)
    finally:
        kv.free()


def test_refusals(dev):
    import torch
    with pytest.raises(tsrc.TsrcError):
        dev.kv4_create(1, 96, 10)
    with pytest.raises(tsrc.TsrcError):
        dev.kv4_create(1, 64, 0)
    kv = dev.kv4_create(2, 64, 10)
    try:
        rows = torch.zeros(4, 128, device="cuda")
        bad = [lambda: kv.set_rows(rows, None, cell0=7), lambda: kv.set_rows(rows, None, row_stride=127),
               lambda: kv.set_rows(None, None), lambda: kv.set_rows(rows, rows.half()), lambda: kv.set_rows(rows.double(), None),
               lambda: kv.set_rows(rows, None, cells=torch.zeros(4, dtype=torch.int32, device="cuda")),
               lambda: kv.get_rows(rows, None, cell0=10), lambda: kv.set_bytes(tsrc.KV_K, np.zeros((11, kv.row_bytes), np.uint8)),
               lambda: kv.set_bytes(2, np.zeros((1, kv.row_bytes), np.uint8)),
               lambda: kv.reorder(torch.zeros(2, dtype=torch.int32, device="cuda"), 1, 2, 6, 6),
               lambda: kv.reorder(torch.zeros(2, dtype=torch.int32, device="cuda"), 1, 2, 3, 4),
               lambda: kv.reorder(torch.zeros(33, dtype=torch.int32, device="cuda"), 1, 33, 0, 0),
               lambda: kv.reorder(torch.zeros(2, dtype=torch.int64, device="cuda"), 1, 2, 5, 5)]
        for call in bad:
            with pytest.raises(tsrc.TsrcError) as e:
                call()
            assert e.value.code in (tsrc.E_ARG, tsrc.E_SHAPE)
        kv.set_rows(rows, None, n=0)                               # nothing to do is no error
        kv.reorder(torch.zeros(2, dtype=torch.int32, device="cuda"), 0, 2, 5, 5)
        dev.sync()
        assert not kv.get_bytes(tsrc.KV_K).any()
    finally:
        kv.free()


def test_offsets_past_32_bits(dev):
    """A cache whose planes pass 4 GiB: the last cells of the last head."""
    import torch
    heads, dim, cells = 8, 512, 2_200_000                         # 2 x 4.5 GB of codes
    kv = dev.kv4_create(heads, dim, cells)
    try:
        rows = torch.randn(3, heads * dim, device="cuda")
        at = torch.tensor([cells - 1, 0, cells - 64], device="cuda")
        kv.set_rows(rows, rows, cells=at)
        out = torch.zeros_like(rows)
        kv.get_rows(None, out, cells=at)
        want = P.pack(*P.quantise(rows.cpu().numpy()))
        np.testing.assert_array_equal(out.cpu().numpy(), P.unpack(want).astype(np.float32))
        np.testing.assert_array_equal(kv.get_bytes(tsrc.KV_K, cells - 1, 1), want[:1])
        kv.reorder(torch.tensor([1, -1], dtype=torch.int32, device="cuda"), 1, 2, cells - 1, 1)
        np.testing.assert_array_equal(kv.get_bytes(tsrc.KV_V, 0, 1), want[:1])
        dev.sync()
    finally:
        kv.free()
