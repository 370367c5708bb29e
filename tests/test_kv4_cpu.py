"""The q4_0 cache's entry points, its attention and beam selection without a GPU: refusals, workspace sizes."""
import pytest

import tsrc

F32, F16, BF16 = tsrc.TYPE_F32, tsrc.TYPE_F16, tsrc.TYPE_BF16


def test_null_arguments_are_errors_not_crashes():
    L = tsrc.lib()
    assert L.tsrc_kv4_create(None, 1, 64, 16, None) == tsrc.E_ARG
    assert b"NULL" in L.tsrc_last_error()
    assert L.tsrc_kv4_free(None) == tsrc.E_ARG
    assert L.tsrc_kv4_set_rows(None, None, F32, None, None, 1, 0, None, 0, None) == tsrc.E_ARG
    assert L.tsrc_kv4_get_rows(None, None, F32, None, None, 1, 0, None, 0, None) == tsrc.E_ARG
    assert L.tsrc_kv4_set_bytes(None, 0, None, 0, 1) == tsrc.E_ARG
    assert L.tsrc_kv4_get_bytes(None, 0, None, 0, 1) == tsrc.E_ARG
    assert L.tsrc_kv4_reorder(None, None, None, 1, 4, 0, 16, 16, None) == tsrc.E_ARG
    assert L.tsrc_flash_attn_q4(None, None, F32, None, 0, 1, 4, 1, None, 0, 0, None, 0, 0.125, None, 0, None, 0, None) == tsrc.E_ARG
    assert L.tsrc_beam_select(None, F32, None, 0, None, 1, 4, 100, 4, None, None, None, None, 0, None) == tsrc.E_ARG


@pytest.mark.parametrize("kind,n_head_kv,dim,n_head,ok", [
    (F32, 8, 128, 32, True), (F16, 2, 64, 14, True), (BF16, 1, 512, 64, True), (2, 8, 128, 32, False),
    (F32, 8, 96, 32, False), (F32, 0, 128, 0, False), (F32, 8, 128, 0, False), (F32, 8, 128, 12, False),
    (F32, 1, 128, 65, False), (F32, 512, 64, 512, False), (F32, 511, 64, 511, True),
    (F32, 0x80000000, 128, 0x80000000, False)])
def test_attention_refusals(kind, n_head_kv, dim, n_head, ok):
    why = tsrc.flash_attn_q4_unsupported(kind, n_head_kv, dim, n_head)
    assert (why is None) == ok, why
    assert ok or why.startswith("FLASH_ATTN")


@pytest.mark.parametrize("kind,beams,vocab,out,ok", [
    (F32, 4, 151936, 8, True), (BF16, 64, 1 << 20, 64, True), (F16, 1, 1, 1, True), (8, 4, 100, 4, False),
    (F32, 0, 100, 4, False), (F32, 65, 100, 4, False), (F32, 4, 0, 4, False), (F32, 4, (1 << 20) + 1, 4, False),
    (F32, 4, 100, 0, False), (F32, 4, 100, 65, False)])
def test_beam_refusals(kind, beams, vocab, out, ok):
    why = tsrc.beam_select_unsupported(kind, beams, vocab, out)
    assert (why is None) == ok, why
    assert ok or why.startswith("beam_select")


def test_workspace_sizes():
    L = tsrc.lib()
    assert L.tsrc_beam_select_workspace(0, 4, 1000, 4) == 0
    one, two = (L.tsrc_beam_select_workspace(g, 4, 151936, 8) for g in (1, 2))
    assert 0 < one < two < 1 << 20
    assert L.tsrc_beam_select_workspace(1, 65, 1000, 4) == 0       # refused shapes need none
    assert L.tsrc_flash_attn_q4_workspace(F32, 8, 128, 0, 32, 100, 0, 0) == 0
    # partial results: of the order of the outputs times the split, never of the cache
    assert L.tsrc_flash_attn_q4_workspace(F32, 8, 128, 1, 32, 1 << 20, 1, 0) < 1 << 24
    assert L.tsrc_flash_attn_q4_workspace(F32, 8, 128, 2048, 32, 1 << 20, 0, 0) < 1 << 30
    assert L.tsrc_flash_attn_q4_workspace(F32, 8, 96, 1, 32, 100, 1, 0) == 0


@pytest.mark.parametrize("T,group", [(4, 5), (4, 3), (1, 1 << 31), ((1 << 20) + 1, 1), (0xFFFFFFFF, 0), (0, 7)])
@pytest.mark.parametrize("dim", [128, 256])
def test_refused_groups_and_token_counts_need_no_workspace(T, group, dim):
    assert tsrc.lib().tsrc_flash_attn_q4_workspace(F32, 1, dim, T, 64, 1 << 16, group, 0) == 0


@pytest.mark.parametrize("dim", [64, 128, 256, 512])
@pytest.mark.parametrize("n_kv", [0, 1, 0xFFFFFFFF])
@pytest.mark.parametrize("group", [0, 1])
def test_workspace_at_the_largest_sizes(dim, n_kv, group):
    """The largest token count and heads, no cell and the largest cell number: a size, and no division by nothing."""
    for T, kv_heads, heads in ((1, 1, 1), (1, 1, 64), (1 << 20, 1, 64), (1 << 20, 256 * 64 // dim, 256 * 64 // dim), (1 << 20, 256 * 64 // dim, 256 * 4096 // dim)):
        assert tsrc.lib().tsrc_flash_attn_q4_workspace(F32, kv_heads, dim, T, heads, n_kv, group, 0) < 1 << 40


def test_wrapper_checks_types():
    torch = pytest.importorskip("torch")
    a, b = torch.zeros(2, 64), torch.zeros(2, 64, dtype=torch.float16)
    assert tsrc._type_of(a, None) == F32 and tsrc._type_of(b, b) == F16
    for bad in ((a, b), (torch.zeros(2, dtype=torch.float64),), (None, None)):
        with pytest.raises(tsrc.TsrcError) as e:
            tsrc._type_of(*bad)
        assert e.value.code == tsrc.E_ARG
    with pytest.raises(tsrc.TsrcError):
        tsrc._expect(torch.zeros(4, dtype=torch.int64), "int32", "parent")
