"""What the 8-bit cache and windowed attention refuse, without a GPU: every refusal is a status before any launch."""
import pytest

import helios_glm53flash_b200 as hk

A = 1 << 20                      # an address that is never used


@pytest.fixture(scope="module")
def lib():
    from helios_glm53flash_b200 import build as hk_build
    hk_build.build()
    return hk.load_library()


def call(lib, name, args, **changed):
    return getattr(lib, name)(*{**args, **changed}.values())


CACHE = dict(ckv8=A, scales=A, dtype=hk.HK_I8, n_blocks=8, block=64, table=A, stride=4)
APPEND = dict(kv_pre=A, ln_w=A, **CACHE, n_seqs=2, seq_start=A, pos=A, n=0, eps=1e-6, new=None, stream=None)
READ = dict(**CACHE, pos=0, n=0, out=A, stream=None)
ROWS = dict(q=A, **CACHE, n_seqs=2, row_seq=A)
TAIL = dict(out=A, m=0, n_heads=64, scale=0.0625, n_split=0)
DENSE = dict(**ROWS, kv_len=A, pos_start=0, window=0, sinks=0, **TAIL, hint=0, ws=None, ws_bytes=0, stream=None)
SPARSE = dict(**ROWS, raw_idx=A, kidx=8, **TAIL, ws=None, ws_bytes=0, stream=None)
WINDOW = dict(q=A, ckv=A, ckv_rows=100, kv_base=None, kv_len=None, pos_start=0, window=8, sinks=0, **TAIL, ws=None, ws_bytes=0, stream=None)

BAD_CACHE = [dict(ckv8=None), dict(scales=None), dict(dtype=hk.HK_F16), dict(dtype=7), dict(n_blocks=0), dict(n_blocks=1 << 31), dict(block=0),
             dict(block=48), dict(block=8), dict(block=256), dict(ckv8=A + 8), dict(stride=0), dict(stride=-1)]
BAD_ROWS = [dict(q=None), dict(out=None), dict(q=A + 2), dict(out=A + 8), dict(n_heads=0), dict(n_heads=6), dict(m=-1), dict(n_seqs=0)]


@pytest.mark.parametrize("name,args,bad", [
    ("hk_mla8_append", APPEND, BAD_CACHE + [dict(kv_pre=None), dict(ln_w=None), dict(pos=None), dict(n=-1), dict(kv_pre=A + 4), dict(ln_w=A + 8),
                                            dict(new=A + 2), dict(n_seqs=0), dict(n_seqs=70000), dict(n=5, seq_start=None), dict(table=None)]),
    ("hk_mla8_read", READ, BAD_CACHE + [dict(out=None), dict(out=A + 2), dict(pos=-1), dict(n=-1), dict(pos=2 ** 31 - 1, n=1)]),
    ("hk_mla8_dense", DENSE, BAD_CACHE + BAD_ROWS + [dict(pos_start=-1), dict(window=-1), dict(sinks=-1), dict(pos_start=2 ** 31 - 1, m=1), dict(table=None),
                                                    dict(kv_len=None, row_seq=None, pos_start=250, m=7),
                                                    dict(kv_len=None, row_seq=None, table=None, n_seqs=1, pos_start=500, m=13)]),
    ("hk_mla8_sparse", SPARSE, BAD_CACHE + BAD_ROWS + [dict(raw_idx=None), dict(kidx=-1), dict(table=None)]),
    ("hk_mla_window", WINDOW, [dict(q=None), dict(ckv=None), dict(out=None), dict(window=0), dict(window=-3), dict(sinks=-1), dict(n_heads=6), dict(m=-1),
                               dict(ckv_rows=-1), dict(pos_start=-1), dict(m=101), dict(q=A + 2), dict(ckv=A + 2), dict(out=A + 2),
                               dict(pos_start=2 ** 31 - 1, m=1, ckv_rows=0)])], ids=["append", "read", "dense", "sparse", "window"])
def test_refusals(lib, name, args, bad):
    assert call(lib, name, args) == hk.HK_OK, "no rows: nothing to do"
    for change in bad:
        assert call(lib, name, args, **change) == hk.HK_ERR_INVALID, change


def test_workspace_too_small(lib):
    need = lib.hk_mla_partial_bytes(3, 2 * 64)
    for name, args in (("hk_mla8_dense", DENSE), ("hk_mla8_sparse", SPARSE), ("hk_mla_window", WINDOW)):
        assert call(lib, name, args, m=2, n_split=3, ws=A, ws_bytes=need - 1) == hk.HK_ERR_WORKSPACE
        assert call(lib, name, args, m=2, n_split=3, ws=None, ws_bytes=need) == hk.HK_ERR_WORKSPACE
        assert call(lib, name, args, m=2, n_split=3, ws=A + 16, ws_bytes=need) == hk.HK_ERR_INVALID
        assert call(lib, name, args, m=2, n_split=2000, ws=A, ws_bytes=1 << 60) in (hk.HK_ERR_UNSUPPORTED, hk.HK_ERR_WORKSPACE)


def test_tensors_that_are_no_cache_raise(lib):
    import torch
    from helios_glm53flash_b200 import _binding as nb
    ok = torch.zeros(4, 16, 512, dtype=torch.int8)
    scales, table = torch.zeros(4), torch.zeros(2, 2, dtype=torch.int32)
    assert nb.cache8(ok, scales, None) == (hk.HK_I8, 4, 16, 0, 1)
    assert nb.cache8(ok.view(torch.float8_e4m3fn), scales, table) == (hk.HK_E4M3, 4, 16, 2, 2)
    assert nb.cache8(ok, scales, table[0]) == (hk.HK_I8, 4, 16, 2, 1)
    for args in ((ok.view(torch.uint8), scales, None), (ok[:, :, :256], scales, None), (ok.view(-1), scales, None), (ok[:, ::2], scales, None),
                 (ok, scales[:3], None), (ok, scales.double(), None), (ok, torch.zeros(8)[::2], None), (ok, scales, table.long()),
                 (ok, scales, table[:, :1]), (ok, scales, table.view(1, 2, 2)), (ok, scales, table[:, :0]), (ok, scales, torch.tensor(3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            nb.cache8(*args)
    for args in ((ok, scales), (ok, None, None), (3, scales, None), (ok, scales, 5)):
        with pytest.raises(TypeError):
            nb.cache8(*args)


def test_workspaces_are_enough_and_no_more(lib):
    """sizes that the calls then ask for, on the host: one byte less is refused before any launch"""
    per_row = lib.hk_mla8_dense_workspace_bytes(2, 64, 0, 5000, 0, 0, 1)
    chunk = lib.hk_mla8_dense_workspace_bytes(100, 64, 1000, 0, 0, 0, 0)
    sparse = lib.hk_mla8_sparse_workspace_bytes(1, 64, 2052, 256, 1)
    gathered = lib.hk_mla8_sparse_workspace_bytes(300, 64, 70, 256, 0)                 # 82 keys a position
    assert per_row > 64 * 2056 and chunk >= 1100 * 1024 and sparse > 64 * 2056
    assert call(lib, "hk_mla8_dense", DENSE, m=2, hint=5000, ws=A, ws_bytes=per_row - 1) == hk.HK_ERR_WORKSPACE
    assert call(lib, "hk_mla8_dense", DENSE, m=100, kv_len=None, row_seq=None, pos_start=1000, stride=20, ws=A, ws_bytes=chunk - 1) == hk.HK_ERR_WORKSPACE
    assert call(lib, "hk_mla8_sparse", SPARSE, m=1, kidx=2052, ws=A, ws_bytes=sparse - 1) == hk.HK_ERR_WORKSPACE
    assert call(lib, "hk_mla8_sparse", SPARSE, m=1, kidx=2052, ws=A + 64, ws_bytes=sparse) == hk.HK_ERR_INVALID
    assert lib.hk_mla8_dense_workspace_bytes(2, 64, 0, 5000, 64, 4, 1) < per_row, "fewer keys under a window"
    assert gathered >= 256 * 1024 + 300 * 70 * 4
    assert call(lib, "hk_mla8_sparse", SPARSE, m=300, kidx=70, row_seq=None, ws=A, ws_bytes=gathered - 1) == hk.HK_ERR_WORKSPACE
    assert lib.hk_mla8_sparse_workspace_bytes(5000, 64, 2052, 256, 1) == 0 and lib.hk_mla8_sparse_workspace_bytes(1, 64, 64, 256, 1) == 0


def test_tables_of_more_positions_than_31_bits_need_no_less_workspace(lib):
    for m in (1, 3, 300):
        want = lib.hk_mla8_sparse_workspace_bytes(m, 64, 2052, 1 << 30, 0)
        assert lib.hk_mla8_sparse_workspace_bytes(m, 64, 2052, 1 << 33, 0) == lib.hk_mla8_sparse_workspace_bytes(m, 64, 2052, 2 ** 63 - 1, 0) == want
    assert lib.hk_mla8_sparse_workspace_bytes(1, 64, 2052, 1 << 33, 0) > 64 * 2056
    need = lib.hk_mla8_sparse_workspace_bytes(1, 64, 2052, 1 << 33, 0)
    assert call(lib, "hk_mla8_sparse", SPARSE, m=1, kidx=2052, row_seq=None, stride=1 << 27, ws=A, ws_bytes=need - 1) == hk.HK_ERR_WORKSPACE


def test_tensors_of_another_type_layout_or_size_raise(lib):
    import torch
    from helios_glm53flash_b200 import _binding as nb
    names = ("half", "single", "ints", "longs")
    ok = [torch.zeros(4, 8).half(), 32, torch.zeros(3), 3, torch.zeros(5, dtype=torch.int32), 4, torch.zeros(2, dtype=torch.int64), 0]
    assert nb.tensors("hfil", names, *ok) is None
    assert nb.tensors("hfil", names, *[x if k % 2 else None for k, x in enumerate(ok)]) is None
    cache = (torch.zeros(4, 16, 512, dtype=torch.int8), torch.zeros(4), None)
    assert nb.cache8(*cache, "hfil", names, *ok) == nb.cache8(*cache)
    for k, bad in ((0, torch.zeros(4, 8)), (0, torch.zeros(8, 4).half().t()), (0, torch.zeros(31).half()), (0, torch.zeros(4, 8).bfloat16()), (0, 5),
                   (2, torch.zeros(2)), (2, torch.zeros(6)[::2]), (4, torch.zeros(5, dtype=torch.int64)), (4, torch.zeros(3, dtype=torch.int32)),
                   (6, torch.zeros(2, dtype=torch.int32)), (6, [1, 2])):
        args = ok[:k] + [bad] + ok[k + 1:]
        for call_ in (lambda: nb.tensors("hfil", names, *args), lambda: nb.cache8(*cache, "hfil", names, *args)):
            with pytest.raises(ValueError, match=names[k // 2]):
                call_()
    for args in (("hfil", names, *ok[:-1]), ("hfi", names, *ok), (3, names, *ok), ("hfil", list(names), *ok), ()):
        with pytest.raises(TypeError):
            nb.tensors(*args)


def test_more_rows_than_the_cuda_core_kernel_takes(lib):
    """heads other than 64 over the fp16 cache: refused on the host, not by a launch that fails"""
    assert call(lib, "hk_mla_window", WINDOW, m=70000, n_heads=16, kv_len=A, kv_base=A, n_split=1) == hk.HK_ERR_UNSUPPORTED
