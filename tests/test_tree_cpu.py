"""No-GPU checks of the calls on trees of drafted tokens and on pages: what is refused is refused on the host, before any launch."""
import pytest

import helios_glm53flash_b200 as hk

A = 1 << 20                                                  # an address, never dereferenced
BAD = hk.HK_ERR_INVALID


@pytest.fixture(scope="module")
def lib():
    from helios_glm53flash_b200 import build as hk_build
    hk_build.build()
    return hk.load_library()


def call(fn, names, good, **changes):
    args = {**good, **changes}
    return fn(*[args[n] for n in names.split()])


TREE = "q ckv rows base len pos kv parent start seqs out m heads scale split ws bytes stream"
TREE_GOOD = dict(q=A, ckv=A, rows=100, base=None, len=None, pos=10, kv=A, parent=A, start=A, seqs=2, out=A, m=8, heads=64, scale=1.0, split=2, ws=None, bytes=0, stream=None)


@pytest.mark.parametrize("changes,status", [
    (dict(q=None), BAD), (dict(ckv=None), BAD), (dict(kv=None), BAD), (dict(parent=None), BAD), (dict(out=None), BAD), (dict(q=A + 8), BAD), (dict(kv=A + 2), BAD),
    (dict(seqs=0), BAD), (dict(seqs=65536), BAD), (dict(m=-1), BAD), (dict(heads=0), BAD), (dict(heads=62), BAD), (dict(pos=-1), BAD), (dict(pos=101), BAD),
    (dict(rows=-1), BAD), (dict(start=None, m=7), BAD), (dict(start=None, m=130), BAD), (dict(split=1025), hk.HK_ERR_UNSUPPORTED),
    (dict(), hk.HK_ERR_WORKSPACE), (dict(ws=A, bytes=1000), hk.HK_ERR_WORKSPACE), (dict(ws=A + 16, bytes=1 << 40), BAD),
])
def test_tree_attention_refuses(lib, changes, status):
    assert call(lib.hk_mla_tree, TREE, TREE_GOOD, **changes) == status


TREE8 = "q ckv8 scales dtype blocks block table stride len pos kv parent start seqs out m heads scale split ws bytes stream"
TREE8_GOOD = dict(q=A, ckv8=A, scales=A, dtype=hk.HK_I8, blocks=8, block=64, table=A, stride=4, len=None, pos=10, kv=A, parent=A, start=A, seqs=2, out=A, m=8, heads=64,
                  scale=1.0, split=2, ws=None, bytes=0, stream=None)


@pytest.mark.parametrize("changes,status", [
    (dict(ckv8=A + 8), BAD), (dict(scales=None), BAD), (dict(dtype=hk.HK_F16), BAD), (dict(block=48), BAD), (dict(table=None), BAD), (dict(stride=0), BAD),
    (dict(blocks=0), BAD), (dict(blocks=1 << 30), BAD), (dict(kv=None), BAD), (dict(m=7, start=None), BAD), (dict(heads=5), BAD), (dict(), hk.HK_ERR_WORKSPACE),
    (dict(split=2000), hk.HK_ERR_UNSUPPORTED),
])
def test_tree_attention_over_8_bits_refuses(lib, changes, status):
    assert call(lib.hk_mla8_tree, TREE8, TREE8_GOOD, **changes) == status


def test_empty_calls_and_workspaces(lib):
    assert call(lib.hk_mla_tree, TREE, TREE_GOOD, m=0) == hk.HK_OK
    assert call(lib.hk_mla8_tree, TREE8, TREE8_GOOD, m=0) == hk.HK_OK
    assert lib.hk_mla_tree_workspace_bytes(0, 64, 1, 100) == 0 and lib.hk_mla_tree_workspace_bytes(4, 64, 1, -1) == 0
    for m in (1, 8, 64, 700):
        for keys in (0, 1, 5001, 1 << 20, (1 << 31) - 1):
            for heads in (4, 64):
                need = lib.hk_mla_tree_workspace_bytes(m, heads, 3, keys)
                assert need == 0 or need >= lib.hk_mla_partial_bytes(2, m * heads)
            assert lib.hk_mla8_tree_workspace_bytes(m, 64, 3, keys, 1 << 17) >= 0
    assert lib.hk_mla8_pages_workspace_bytes(0, 4) == 0 and lib.hk_mla8_pages_workspace_bytes(8, -1) == 0
    assert lib.hk_mla8_pages_workspace_bytes(1000, 5) >= 3 * 4000 and lib.hk_mla8_pages_workspace_bytes(5, 1000) >= 3 * 4000


def test_tables_of_more_positions_than_31_bits_need_no_less_workspace(lib):
    for m, heads, keys in ((8, 64, 5001), (64, 64, 32768), (7, 20, 900), (96, 16, 3000)):
        for seqs in (1, 2, 65535):
            want = lib.hk_mla8_tree_workspace_bytes(m, heads, seqs, keys, 1 << 30)
            for positions in (1 << 31, 1 << 38, 2 ** 63 - 1):
                assert lib.hk_mla8_tree_workspace_bytes(m, heads, seqs, keys, positions) == want
    # 5,001 keys in a table of 2^31 positions, and the call itself: what is less than the size is refused
    need = lib.hk_mla8_tree_workspace_bytes(8, 64, 2, 5001, 1 << 31)
    assert need >= lib.hk_mla_partial_bytes(2, 8 * 64)
    wide = dict(block=128, stride=1 << 24, pos=5001, split=0)
    assert call(lib.hk_mla8_tree, TREE8, TREE8_GOOD, **wide) == hk.HK_ERR_WORKSPACE
    assert call(lib.hk_mla8_tree, TREE8, TREE8_GOOD, **wide, len=A, ws=A, bytes=lib.hk_mla_partial_bytes(2, 8 * 64) - 1) == hk.HK_ERR_WORKSPACE


ACCEPT = "kv ckv rows base len pos parent start seqs leaf m told stream"
ACCEPT_GOOD = dict(kv=A, ckv=A, rows=9, base=None, len=A, pos=0, parent=A, start=A, seqs=2, leaf=A, m=4, told=None, stream=None)


@pytest.mark.parametrize("changes", [dict(kv=None), dict(ckv=A + 8), dict(leaf=None), dict(parent=None), dict(rows=-1), dict(pos=-2), dict(told=A), dict(seqs=0),
                                     dict(start=None, m=5)])
def test_accepting_latents_refuses(lib, changes):
    assert call(lib.hk_mla_tree_accept, ACCEPT, ACCEPT_GOOD, **changes) == BAD


KDA = "qkv g beta dt a lb state slots parent start seqs out f32 m heads most stream"
KDA_GOOD = dict(qkv=A, g=A, beta=A, dt=None, a=None, lb=-5.0, state=A, slots=None, parent=A, start=A, seqs=2, out=A, f32=None, m=8, heads=4, most=0, stream=None)


@pytest.mark.parametrize("changes", [dict(qkv=None), dict(qkv=A + 4), dict(g=A + 8), dict(beta=None), dict(dt=A), dict(a=A), dict(state=A + 8), dict(parent=None), dict(out=None),
                                     dict(most=65), dict(most=-1), dict(heads=0), dict(heads=20000), dict(seqs=0), dict(start=None, m=9), dict(m=-1)])
def test_the_recurrence_of_nodes_refuses(lib, changes):
    assert call(lib.hk_kda_tree, KDA, KDA_GOOD, **changes) == BAD
    assert call(lib.hk_kda_tree, KDA, KDA_GOOD, m=0) == hk.HK_OK


KACC = "x conv qkv g beta dt a lb state slots parent start seqs leaf m heads stream"
KACC_GOOD = dict(KDA_GOOD, x=A, conv=A, leaf=A)


@pytest.mark.parametrize("changes", [dict(x=None), dict(conv=None), dict(conv=A + 4), dict(leaf=None), dict(g=None), dict(state=None), dict(a=A)])
def test_accepting_states_refuses(lib, changes):
    assert call(lib.hk_kda_tree_accept, KACC, KACC_GOOD, **changes) == BAD


CONV = "x conv slots w bias parent start seqs out m dim act stream"
CONV_GOOD = dict(x=A, conv=A, slots=None, w=A, bias=None, parent=A, start=A, seqs=2, out=A, m=4, dim=8, act=1, stream=None)


@pytest.mark.parametrize("changes", [dict(x=A + 4), dict(conv=None), dict(w=A + 4), dict(out=A + 4), dict(dim=6), dict(dim=0), dict(parent=None), dict(start=None, m=5)])
def test_the_convolution_of_nodes_refuses(lib, changes):
    assert call(lib.hk_kda_tree_conv, CONV, CONV_GOOD, **changes) == BAD


POOL = dict(ckv8=A, scales=A, dtype=hk.HK_E4M3, blocks=8, block=16, refs=A, table=A, stride=4, seqs=2, a=A, b=A, c=A, n=1, told=None, ws=A, bytes=1 << 20, stream=None)
FORK = "ckv8 scales dtype blocks block refs table stride seqs a b c n told ws bytes stream"
RESERVE = "ckv8 scales dtype blocks block refs table stride seqs a b n told ws bytes stream"
FREE = "ckv8 scales dtype blocks block refs table stride seqs a b n stream"
COMPACT = "ckv8 scales dtype blocks block refs table stride seqs told ws bytes stream"


@pytest.mark.parametrize("changes,status", [(dict(refs=None), BAD), (dict(table=None), BAD), (dict(stride=0), BAD), (dict(seqs=0), BAD), (dict(blocks=0), BAD), (dict(block=24), BAD),
                                            (dict(ckv8=None), BAD), (dict(dtype=9), BAD), (dict(ws=None), hk.HK_ERR_WORKSPACE), (dict(bytes=300), hk.HK_ERR_WORKSPACE),
                                            (dict(ws=A + 64), BAD)])
def test_pages_refuse(lib, changes, status):
    assert call(lib.hk_mla8_pages_fork, FORK, POOL, **changes) == status
    assert call(lib.hk_mla8_pages_reserve, RESERVE, POOL, **changes) == status
    assert call(lib.hk_mla8_pages_compact, COMPACT, POOL, **changes) == status
    if not {"ws", "bytes"} & set(changes):
        assert call(lib.hk_mla8_pages_free, FREE, POOL, **changes) == status


def test_pages_refuse_lists(lib):
    for name in "abc":
        assert call(lib.hk_mla8_pages_fork, FORK, POOL, **{name: None}) == BAD
    assert call(lib.hk_mla8_pages_reserve, RESERVE, POOL, b=None) == BAD and call(lib.hk_mla8_pages_free, FREE, POOL, a=None) == BAD
    for fn, names in ((lib.hk_mla8_pages_fork, FORK), (lib.hk_mla8_pages_reserve, RESERVE), (lib.hk_mla8_pages_free, FREE)):
        assert call(fn, names, POOL, n=-1) == BAD and call(fn, names, POOL, n=0) == hk.HK_OK
    assert call(lib.hk_mla8_pages_fork, FORK, POOL, n=0, a=None, b=None, c=None) == hk.HK_OK
    assert call(lib.hk_mla8_pages_reserve, RESERVE, POOL, n=0, a=None, b=None) == call(lib.hk_mla8_pages_free, FREE, POOL, n=0, a=None) == hk.HK_OK
    copy = "ckv8 scales blocks ckv8 scales blocks dtype block a b n stream"
    assert call(lib.hk_mla8_pages_copy, copy, POOL, n=0) == call(lib.hk_mla8_pages_copy, copy, POOL, n=0, a=None, b=None) == hk.HK_OK
    for changes in (dict(a=None), dict(n=-1), dict(block=8), dict(dtype=0), dict(blocks=0)):
        assert call(lib.hk_mla8_pages_copy, copy, POOL, **changes) == BAD
