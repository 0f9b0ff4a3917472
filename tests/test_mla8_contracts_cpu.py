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
