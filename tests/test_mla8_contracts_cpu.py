"""What the library says on the host about calls over the 8-bit cache and under windows: numbers of splits, sizes of workspaces, refusals."""
import pytest

import helios_glm53flash_b200 as hk
from test_mla8_cpu import A, DENSE, WINDOW, call, lib  # noqa: F401


def test_numbers_of_keys_of_all_31_bits_choose_as_many_splits_as_smaller_ones(lib):  # noqa: F811
    for m in (1, 3, 100):
        for keys in (2 ** 31 - 1, 2 ** 31 - 63, 2 ** 31 - 64):
            assert lib.hk_mla_auto_splits(m, keys) == lib.hk_mla_auto_splits(m, 1 << 30), (m, keys)
            assert lib.hk_mla8_dense_workspace_bytes(m, 64, 0, keys, 0, 0, 1) == lib.hk_mla8_dense_workspace_bytes(m, 64, 0, 1 << 30, 0, 0, 1)
            assert lib.hk_mla8_dense_workspace_bytes(m, 64, 0, keys, keys, keys, 1) == lib.hk_mla8_dense_workspace_bytes(m, 64, 0, 1 << 30, 0, 0, 1)


def test_a_chunk_that_is_refused_has_no_workspace(lib):  # noqa: F811
    """positions past 31 bits: the size is 0, as the call is HK_ERR_INVALID"""
    for pos, m in ((2 ** 31 - 1, 1), (2 ** 31 - 100, 101), (2 ** 31 - 1, 2 ** 31 - 1)):
        assert lib.hk_mla8_dense_workspace_bytes(m, 64, pos, 0, 0, 0, 0) == 0
        assert call(lib, "hk_mla8_dense", DENSE, m=m, pos_start=pos, kv_len=None, row_seq=None, ws=A, ws_bytes=1 << 60) == hk.HK_ERR_INVALID
    assert lib.hk_mla8_dense_workspace_bytes(100, 64, 2 ** 31 - 101, 0, 0, 0, 0) >= (2 ** 31 - 1) * 1024


@pytest.mark.parametrize("heads", [64, 16, 4, 100])
@pytest.mark.parametrize("window,sinks", [(104, 0), (128, 0), (512, 0), (1016, 0), (1, 0), (4096, 4), (3, 700), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_a_window_asks_for_the_workspace_that_is_said(lib, heads, window, sinks):  # noqa: F811
    """one byte less is refused before any launch, and where none is said the form of one split is chosen"""
    for m, n, per_row in ((1, 128, False), (1, 5000, False), (3, 700, True), (24, 5000, True), (200, 1000, False), (1, 0, True), (2, 2 ** 31 - 1, True)):
        need = lib.hk_mla_window_workspace_bytes(m, heads, n, window, sinks)
        args = dict(m=m, n_heads=heads, pos_start=n if per_row else n - m, kv_len=A if per_row else None, ckv_rows=0, window=window, sinks=sinks)
        if per_row and n + m > 2 ** 31 - 1:
            assert call(lib, "hk_mla_window", WINDOW, **args) == hk.HK_ERR_INVALID
        elif need:
            splits = 2
            while lib.hk_mla_partial_bytes(splits, m * heads) < need:
                splits += 1
            assert lib.hk_mla_partial_bytes(splits, m * heads) == need
            assert call(lib, "hk_mla_window", WINDOW, **args, ws=A, ws_bytes=need - 1) == hk.HK_ERR_WORKSPACE
            assert call(lib, "hk_mla_window", WINDOW, **args, ws=None, ws_bytes=need) == hk.HK_ERR_WORKSPACE
            assert call(lib, "hk_mla_window", WINDOW, **args, ws=A + 16, ws_bytes=need) == hk.HK_ERR_INVALID     # it is enough, and looked at further
        assert hk.mla_window_workspace_bytes(m, heads, n, window, sinks) >= 0


def test_sizes_of_windows_that_are_refused_are_none(lib):  # noqa: F811
    for bad in ((0, 64, 500, 100, 0), (-1, 64, 500, 100, 0), (1, 0, 500, 100, 0), (1, 64, 500, 0, 0), (1, 64, 500, 100, -1)):
        assert lib.hk_mla_window_workspace_bytes(*bad) == 0
    assert lib.hk_mla_window_keys(500, 0, 0) == lib.hk_mla_window_keys(500, 3, -1) == 0
    assert lib.hk_mla_window_keys(500, 100, 0) == lib.hk_mla_window_keys(0, 100, 0) == 192 and lib.hk_mla_window_keys(100, 1000, 5) == 128
    assert lib.hk_mla_window_keys(2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1) == 2 ** 31 - 1


def test_tables_and_blocks_whose_sizes_do_not_fit_31_bits_raise(lib):  # noqa: F811
    """(the library takes ints: 2^32 + 4 would arrive as 4)"""
    import torch
    from helios_glm53flash_b200 import _binding as nb
    ckv8, scales = torch.zeros(4, 16, 512, dtype=torch.int8), torch.zeros(4)
    for shape in ((1, 2 ** 32 + 4), (2 ** 32 + 4, 1), (2 ** 31,), (2, 2 ** 31)):
        with pytest.raises(ValueError):
            nb.cache8(ckv8, scales, torch.empty(shape, dtype=torch.int32, device="meta"))
    with pytest.raises(ValueError):
        nb.cache8(torch.empty(0, 2 ** 32 + 16, 512, dtype=torch.int8), torch.zeros(0), None)
    assert nb.cache8(ckv8, scales, torch.empty(2 ** 31 - 1, 1, dtype=torch.int32, device="meta")) == (hk.HK_I8, 4, 16, 1, 2 ** 31 - 1)
