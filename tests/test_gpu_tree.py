"""Trees of drafted tokens: attention over both latent caches, the KDA convolution and recurrence, and the steps to an accepted node, against
64 bits and against the calls that decode token by token."""
import math
import os
import subprocess
import sys

import pytest
import torch

import helios_glm53flash_b200 as hk
import latent8_ref as ref8
from latent8_ref import attend, cache, rows_of, table_for
from tree_ref import TREES, ints, kda_token, layout, path, tree_of

pytestmark = pytest.mark.gpu

NAN, INF = math.nan, math.inf


def gen_of(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def finish():
    torch.cuda.synchronize()
    assert hk.read_device_status() == 0


def check_rows(out, want):
    for r, (o, tol) in enumerate(want):
        off = (out[r].double() - o).abs()
        assert bool((off <= tol).all()), "row %d: off %.3e of %.3e" % (r, float((off - tol).max()), float(tol.max()))


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------
def wanted(q, past, tree_kv, first, tree, scale):
    """(output, bound) of a tree's rows; past: the sequence's keys in 64 bits"""
    return [attend(q[first + j].double(), torch.cat((past, tree_kv[[first + i for i in path(tree, j)]].double())), scale) for j in range(len(tree))]


@pytest.mark.parametrize("trees,lens", [
    (["one"], [0]), (["one"], [1]), (["chain5"], [63]), (["binary15"], [64]), (["wide63"], [65]), (["chain64"], [200]),
    (["star7", "two_roots", "one"], [0, 129, 1000]), ([(31, 1), (8, 2), (64, 3), (1, 4)], [500, 64, 3, 128]), ([(64, 5)], [2500]), ([(5, 6)] * 9, [777] * 9),
    ([(16, 7)], [4100]), (["chain5", [], "chain5"], [40, 50, 60]),
])
@pytest.mark.parametrize("heads,n_split", [(64, 0), (64, 1), (64, 3), (16, 0), (32, 2), (8, 1), (4, 5), (20, 0), (128, 2)])
def test_nodes_over_the_fp16_cache(trees, lens, heads, n_split):
    trees = [tree_of(t) for t in trees]
    gen = gen_of(len(trees) + sum(lens))
    starts, parent, tree_start = layout(trees)
    m, n = starts[-1], len(trees)
    gap = 3                                                   # rows between the sequences, of which nobody may see any
    base = [sum(lens[:i]) + gap * (i + 1) for i in range(n)]
    ckv = torch.full((sum(lens) + gap * (n + 1), 512), NAN, dtype=torch.float16, device="cuda")
    for b, k in zip(base, lens):
        ckv[b:b + k] = randn(gen, k, 512).half()
    q, tree_kv = (randn(gen, m, heads, 512) * 0.7).half(), randn(gen, m, 512).half()
    out = torch.full((m, heads, 512), 7.0, dtype=torch.float16, device="cuda")
    hk.mla_tree_decode(q, ckv, tree_kv, parent, out, m, n_seqs=n, tree_start=tree_start, kv_base=torch.tensor(base, device="cuda"), kv_len=ints(lens),
                       n_heads=heads, n_split=n_split, n_keys_hint=max(lens))
    finish()
    check_rows(out, [w for s in range(n) for w in wanted(q, ckv[base[s]:base[s] + lens[s]].double(), tree_kv, starts[s], trees[s], 0.0625)])


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("block", [16, 64, 128])
@pytest.mark.parametrize("trees,lens,heads,n_split", [
    (["one"], [0], 64, 0), (["binary15"], [64], 64, 0), (["wide63", "chain5"], [65, 1000], 64, 0), ([(31, 1), (64, 2), (1, 3)], [500, 3, 128], 16, 0),
    ([(12, 5)], [3000], 64, 0), (["star7"], [700], 20, 3), (["chain64"], [200], 128, 1), ([(5, 6)] * 9, [777] * 9, 64, 2),
    (["chain64", (60, 3), "one"], [3000, 2100, 900], 64, 0), (["chain5"] * 12, [3000 - 100 * i for i in range(12)], 16, 0), ([(64, 3)] * 3, [2000, 1999, 300], 32, 0),
    (["star7", "one"], [90, 0], 4, 2),
])
def test_nodes_over_the_8_bit_cache(kind, block, trees, lens, heads, n_split):
    trees = [tree_of(t) for t in trees]
    gen = gen_of(block + sum(lens) + heads)
    starts, parent, tree_start = layout(trees)
    m, n = starts[-1], len(trees)
    blocks = max(1, max((k + block - 1) // block for k in lens))
    ckv8, scales = cache(gen, kind, n * blocks + 2, block, spread=0.5)
    table = table_for(gen, n, blocks, n * blocks + 2)
    q, tree_kv = (randn(gen, m, heads, 512) * 0.7).half(), randn(gen, m, 512).half()
    out = torch.full((m, heads, 512), 7.0, dtype=torch.float16, device="cuda")
    hk.mla8_tree_decode(q, ckv8, scales, tree_kv, parent, out, m, n_seqs=n, tree_start=tree_start, block_table=table, kv_len=ints(lens), n_heads=heads,
                        n_split=n_split, n_keys_hint=max(lens))
    finish()
    want = []
    for s in range(n):
        past = rows_of(ckv8, scales, table[s], torch.arange(lens[s], device="cuda"))
        want += wanted(q, past, tree_kv, starts[s], trees[s], 0.0625)
    check_rows(out, want)


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("heads,seqs,nodes,n,factor", [(64, 3, 33, 1153, 1.0), (32, 3, 52, 802, 1.0), (64, 3, 33, 1153, 2.0 ** 11), (32, 3, 52, 802, 2.0 ** -16), (64, 2, 64, 1500, 0.0)])
def test_scales_where_many_nodes_share_the_keys(kind, heads, seqs, nodes, n, factor):
    """positions that are read first lose nothing, whatever their scales; outputs follow a common factor of all keys and queries' inverse"""
    gen, block = gen_of(12), 32
    blocks = (n + block - 1) // block
    ckv8, scales = cache(gen, kind, seqs * blocks, block, spread=0.7)
    scales *= factor
    table = table_for(gen, seqs, blocks, seqs * blocks)
    trees = [tree_of((nodes, i)) for i in range(seqs)]
    starts, parent, tree_start = layout(trees)
    m, back = starts[-1], 1.0 / factor if factor else 1.0
    q, tree_kv = (randn(gen, m, heads, 512) * 0.7).half(), (randn(gen, m, 512) * min(factor, 1.0)).half()
    out = torch.empty(m, heads, 512, dtype=torch.float16, device="cuda")
    scale = 0.0625 * back
    hk.mla8_tree_decode(q, ckv8, scales, tree_kv, parent, out, m, n_seqs=seqs, tree_start=tree_start, block_table=table, kv_len=ints([n] * seqs), n_heads=heads, scale=scale,
                        n_keys_hint=n)
    finish()
    want = [w for s in range(seqs) for w in wanted(q, rows_of(ckv8, scales, table[s], torch.arange(n, device="cuda")), tree_kv, starts[s], trees[s], scale)]
    # values of 65,520 (half a step above the largest of fp16) or more are infinities in fp16: where one is within the bound, infinity is right too
    for r, (o, tol) in enumerate(want):
        beyond = (o.abs() + tol >= 65520) & torch.isinf(out[r]) & (torch.sign(out[r]) == torch.sign(o))
        out[r] = torch.where(beyond, o.clamp(-65504, 65504).half(), out[r])
        want[r] = (torch.where(beyond, o.clamp(-65504, 65504), o), tol)
    check_rows(out, want)


@pytest.mark.parametrize("nodes,stride", [(3, 30), (64, 30), (64, 60)])
def test_positions_without_a_block_and_behind_the_table(nodes, stride):
    """an entry that names no block is a latent of zeros, positions behind the table are none; the same whether the positions are read first or not"""
    gen, block = gen_of(9), 64
    ckv8, scales = cache(gen, "i8", 64, block)
    table = table_for(gen, 1, stride, 64)
    table[0, 3], table[0, 11] = -1, 64
    q, rows, tree = (randn(gen, nodes, 64, 512) * 0.7).half(), randn(gen, nodes, 512).half(), list(range(-1, nodes - 1))
    out = torch.full((nodes, 64, 512), 7.0, dtype=torch.float16, device="cuda")
    n = stride * block + 500 if stride < 60 else stride * block - 37
    hk.mla8_tree_decode(q, ckv8, scales, rows, ints(tree), out, nodes, block_table=table, kv_len=ints([n]), n_keys_hint=n)
    also = torch.empty_like(out)
    hk.mla8_tree_decode(q, ckv8, scales, rows, ints(tree), also, nodes, n, block_table=table)
    finish()
    p = torch.arange(min(n, stride * block), device="cuda")
    named = torch.where((table[0] >= 0) & (table[0] < 64), table[0], 0).long()[p // block]
    past = ref8.as_f64(ckv8.view(torch.uint8)[named, p % block].view(ckv8.dtype)) * scales[named].double()[:, None]
    past[(p // block == 3) | (p // block == 11)] = 0
    for got in (out, also):
        check_rows(got, [attend(q[j].double(), torch.cat((past, rows[:j + 1].double())), 0.0625) for j in range(nodes)])


@pytest.mark.parametrize("over", ["f16", "i8", "f16 of 4", "f16 of 16", "f16 of 32", "f16 of 20", "i8 of 16", "i8 of 8", "i8 of 20"])
def test_what_a_node_does_not_see_has_no_effect(over):
    """NaN and infinities in other branches, in rows of no tree and behind a sequence's keys; a key that is not finite shows in the rows that see it"""
    heads = int(over.split(" of ")[1]) if " of " in over else 64
    tree = tree_of("binary15")
    gen = gen_of(3)
    starts, parent, tree_start = layout([tree, tree], front=2)
    m = starts[-1] + 3                                        # rows behind the last tree
    parent = torch.cat((parent, ints([0, 1, 2])))
    n = 70
    q, clean = (randn(gen, m, heads, 512) * 0.7).half(), randn(gen, m, 512).half()
    ckv = torch.full((4 * n, 512), INF, dtype=torch.float16, device="cuda")
    base = [1, 2 * n]
    for b in base:
        ckv[b:b + n] = randn(gen, n, 512).half()
    ckv8, scales = cache(gen, "i8", 12, 16)
    scales[5] = NAN                                          # in nobody's table
    table = ints([[0, 1, 2, 3, 4, 5], [6, 7, 8, 9, 10, 5]])

    def call(rows):
        out = torch.full((m, heads, 512), 7.0, dtype=torch.float16, device="cuda")
        tree_args = dict(n_seqs=2, tree_start=tree_start, kv_len=ints([n, n]), n_heads=heads, n_keys_hint=n)
        if over.startswith("i8"):
            hk.mla8_tree_decode(q, ckv8, scales, rows, parent, out, m, block_table=table, **tree_args)
        else:
            hk.mla_tree_decode(q, ckv, rows, parent, out, m, kv_base=torch.tensor(base, device="cuda"), **tree_args)
        finish()
        return out

    good = call(clean)
    assert bool(torch.isfinite(good).all())
    assert bool((good[:2] == 7).all()) and bool((good[starts[-1]:] == 7).all()), "rows of no tree are left as they were"
    bad = clean.clone()
    bad[:2], bad[starts[-1]:] = NAN, -INF
    for node, value in ((4, NAN), (6, INF), (14, -INF)):
        bad[starts[0] + node] = value
    out = call(bad)
    for s in range(2):
        for j in range(len(tree)):
            r = starts[s] + j
            if s == 0 and {4, 6, 14} & set(path(tree, j)):
                assert bool(torch.isnan(out[r]).any()), (s, j)
            else:
                assert torch.equal(out[r], good[r]), (s, j)


@pytest.mark.parametrize("told", [True, False])
def test_two_nodes_by_a_pair_of_ctas(told):
    """enough nodes and keys that two of a tree go together: odd trees, an empty one, ragged lengths, splits, branches and gaps that hold NaN"""
    trees = [tree_of(t) for t in ((33, 1), (64, 2), "one", [], "chain5", (40, 6), "star7")]
    lens = [2000, 1531, 3001, 5, 64, 2879, 0]
    gen = gen_of(31)
    starts, parent, tree_start = layout(trees, front=1)
    m, n = starts[-1] + 2, len(trees)
    parent = torch.cat((parent, ints([0, 0])))
    base = [sum(lens[:i]) + 2 * (i + 1) for i in range(n)]
    ckv = torch.full((sum(lens) + 2 * (n + 1) + 64, 512), NAN, dtype=torch.float16, device="cuda")
    for b, k in zip(base, lens):
        ckv[b:b + k] = randn(gen, k, 512).half()
    q, rows = (randn(gen, m, 64, 512) * 0.7).half(), randn(gen, m, 512).half()
    bad = {starts[1] + 60: NAN, starts[0] + 31: INF, starts[6] + 3: -INF, 0: NAN, m - 1: NAN}
    for r, value in bad.items():
        rows[r] = value
    out = torch.full((m, 64, 512), 7.0, dtype=torch.float16, device="cuda")
    hk.mla_tree_decode(q, ckv, rows, parent, out, m, n_seqs=n, tree_start=tree_start, kv_base=torch.tensor(base, device="cuda"), kv_len=ints(lens),
                       n_keys_hint=max(lens), ckv_rows=None if told else 0)
    finish()
    for s, tree in enumerate(trees):
        for j in range(len(tree)):
            r, seen = starts[s] + j, [starts[s] + i for i in path(tree, j)]
            if set(seen) & set(bad):
                assert bool(torch.isnan(out[r]).any()), (s, j)
            else:
                o, tol = attend(q[r].double(), torch.cat((ckv[base[s]:base[s] + lens[s]].double(), rows[seen].double())), 0.0625)
                assert bool(((out[r].double() - o).abs() <= tol).all()), (s, j)
    for r in (0, m - 2, m - 1):
        assert bool((out[r] == 7).all())


@pytest.mark.parametrize("switch", ["HK_MLA_FORCE_SIMT", "HK_MLA_NO_TMA"])
def test_trees_on_the_cuda_cores(switch):
    """asked for, and where there is no encoder of tensor maps, when positions of the 8-bit cache are read first all the same; in a process of its own"""
    names = ("test_nodes_over", "test_scales_where_many_nodes_share_the_keys", "test_positions_without_a_block_and_behind_the_table", "test_what_a_node_does_not_see_has_no_effect",
             "test_two_nodes_by_a_pair_of_ctas", "test_parents_that_are_no_earlier_node", "test_a_sequence_of_more_rows", "test_a_chain_agrees_with_a_causal_chunk")
    run = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-m", "gpu", "-p", "no:cacheprovider", "-k", " or ".join(names), os.path.abspath(__file__)],
                         env={**os.environ, switch: "1"}, capture_output=True, text=True, timeout=600)
    assert run.returncode == 0, run.stdout[-3000:] + run.stderr[-2000:]


@pytest.mark.parametrize("behind", [0, 1, 13, 40, 200])
def test_caches_at_the_end_of_their_memory_whose_rows_are_not_told(behind):
    """a cache that ends `behind` rows before the end of its allocation, several of them (what follows an allocation may be nothing): the same bits as with its rows told"""
    torch.cuda.empty_cache()
    gen, held, rows = gen_of(51 + behind), 200, 17 << 11         # 34 MB, an allocation of its own
    trees = [tree_of((46, 1)), tree_of((27, 3))]
    starts, parent, tree_start = layout(trees)
    m, base = starts[-1], torch.tensor([10, 90], device="cuda")
    kv = randn(gen, m, 512).half()
    whole = [torch.empty(rows, 512, dtype=torch.float16, device="cuda") for _ in range(4)]
    idx = torch.full((3, 64), -1, dtype=torch.int32, device="cuda")
    idx[:, :5] = ints([[0, 7, 199, 100, 199], [198, 199, -1, 5, 5], [199, -1, -1, -1, -1]])
    for ckv in (w[rows - behind - held:rows - behind] for w in whole):
        ckv.copy_(randn(gen, held, 512))
        for lens in ([0, 3], [64, 110], [70, 1], [128, 96]):
            for heads, n_split in ((64, 0), (64, 3), (16, 0), (4, 24)):
                q = (randn(gen, m, heads, 512) * 0.7).half()
                got = [torch.empty_like(q) for _ in range(2)]
                for out, told in zip(got, (0, None)):
                    hk.mla_tree_decode(q, ckv, kv, parent, out, m, n_seqs=2, tree_start=tree_start, kv_base=base, kv_len=ints(lens), n_heads=heads, n_split=n_split,
                                       n_keys_hint=128, ckv_rows=told)
                finish()
                assert torch.equal(*got), (lens, heads)
            q = (randn(gen, 3, 64, 512) * 0.7).half()
            for call in (lambda o, told: hk.mla_dense_prefill(q, ckv, o, 3, 0, kv_base=torch.tensor([10, 90, 199], device="cuda"), kv_len=ints(lens + [1]), n_keys_hint=128, ckv_rows=told),
                         lambda o, told: hk.mla_window_prefill(q, ckv, o, 3, 0, 60, 3, kv_base=torch.tensor([10, 90, 199], device="cuda"), kv_len=ints(lens + [1]), n_keys_hint=128, ckv_rows=told),
                         lambda o, told: hk.mla_dense_prefill(q, ckv, o, 3, held - 3, ckv_rows=told),
                         lambda o, told: hk.mla_sparse_decode(q, ckv, idx, 64, o, 3, ckv_rows=told)):
                got = [torch.empty_like(q) for _ in range(2)]
                call(got[0], 0)
                call(got[1], None)
                finish()
                assert torch.equal(*got), lens


def test_parents_that_are_no_earlier_node_hang_on_the_sequence():
    gen = gen_of(4)
    m, n = 6, 90
    q, tree_kv, ckv = (randn(gen, m, 64, 512) * 0.7).half(), randn(gen, m, 512).half(), randn(gen, n, 512).half()
    outs = []
    for tree in ([0, 5, -7, 2, 1 << 30, 4], [-1, -1, -1, 2, -1, 4]):
        out = torch.empty(m, 64, 512, dtype=torch.float16, device="cuda")
        hk.mla_tree_decode(q, ckv, tree_kv, ints(tree), out, m, n)
        outs.append(out)
    finish()
    assert torch.equal(*outs)
    check_rows(outs[0], wanted(q, ckv.double(), tree_kv, 0, [-1, -1, -1, 2, -1, 4], 0.0625))


def test_a_sequence_of_more_rows_than_a_tree_has():
    """rows from the 65th on belong to no tree; lengths are cut at the cache's end"""
    gen = gen_of(5)
    m, n = 70, 50
    tree = list(range(-1, m - 1))
    q, tree_kv, ckv = (randn(gen, m, 64, 512) * 0.7).half(), randn(gen, m, 512).half(), randn(gen, n, 512).half()
    out = torch.full((m, 64, 512), 7.0, dtype=torch.float16, device="cuda")
    hk.mla_tree_decode(q, ckv, tree_kv, ints(tree), out, m, tree_start=ints([0, m]), kv_len=ints([1 << 30]), n_keys_hint=n)
    finish()
    check_rows(out[:64], wanted(q, ckv.double(), tree_kv, 0, tree[:64], 0.0625))
    assert bool((out[64:] == 7).all())


@pytest.mark.parametrize("m,n", [(1, 5001), (12, 9000), (64, 3000)])
def test_a_chain_agrees_with_a_causal_chunk(m, n):
    """the nodes of a chain are the rows of a chunk whose keys lie in the cache"""
    gen = gen_of(6)
    ckv = randn(gen, n + m, 512).half()
    q = (randn(gen, m, 64, 512) * 0.7).half()
    out, chunk = (torch.empty(m, 64, 512, dtype=torch.float16, device="cuda") for _ in range(2))
    hk.mla_tree_decode(q, ckv, ckv[n:].contiguous(), ints(list(range(-1, m - 1))), out, m, n)
    hk.mla_dense_prefill(q, ckv, chunk, m, n)
    finish()
    want = wanted(q, ckv[:n].double(), ckv[n:], 0, list(range(-1, m - 1)), 0.0625)
    check_rows(out, want)
    check_rows(chunk, want)


@pytest.mark.parametrize("kind", ["f16", "i8"])
def test_the_accepted_rows_go_behind_the_cached_ones(kind, monkeypatch):
    trees = [tree_of(t) for t in ("binary15", "chain64", "one", "star7", (20, 3))]
    leaves = [13, 63, 0, -1, 99]
    lens = [30, 61, 5, 40, 7]
    gen = gen_of(7)
    starts, parent, tree_start = layout(trees)
    m, n = starts[-1], len(trees)
    rows = randn(gen, m, 512).half()
    len_out = torch.zeros(n, dtype=torch.int32, device="cuda")
    paths = [path(t, j) if 0 <= j < len(t) else [] for t, j in zip(trees, leaves)]
    picked = [starts[s] + j for s in range(n) for j in paths[s]]
    if kind == "f16":
        room = 130
        ckv = randn(gen, n * room, 512).half()
        want = ckv.clone()
        for s in range(n):
            want[s * room + lens[s]:s * room + lens[s] + len(paths[s])] = rows[[starts[s] + j for j in paths[s]]]
        hk.mla_tree_accept(rows, ckv, parent, ints(leaves), m, n_seqs=n, tree_start=tree_start, kv_base=torch.arange(n, device="cuda") * room, kv_len=ints(lens),
                           len_out=len_out)
        finish()
        assert torch.equal(ckv, want)
    else:
        for block in (16, 32, 64, 128):
            blocks = (130 + block - 1) // block
            ckv8, scales = cache(gen, "i8", n * blocks + 1, block)
            scales *= 0.5 + torch.rand(n * blocks + 1, device="cuda", generator=gen)
            table = table_for(gen, n, blocks, n * blocks + 1)
            before, before_scales = ckv8.clone(), scales.clone()
            hk.mla8_tree_accept(rows, ckv8, scales, parent, ints(leaves), m, n_seqs=n, tree_start=tree_start, block_table=table, kv_len=ints(lens), len_out=len_out)
            finish()
            monkeypatch.setattr(ref8, "normed", lambda x, w, eps: x.double())
            at = [0]
            for p in paths:
                at.append(at[-1] + len(p))
            ref8.check_append(before, before_scales, ckv8, scales, rows[picked], None, table.cpu(), lens, at, "i8")
    assert len_out.tolist() == [k + len(p) for k, p in zip(lens, paths)]


def test_accepted_rows_beyond_the_cache_are_dropped():
    gen = gen_of(8)
    rows, ckv = randn(gen, 5, 512).half(), randn(gen, 12, 512).half()
    want = ckv.clone()
    want[7:10] = rows[:3]
    hk.mla_tree_accept(rows, ckv, ints(TREES["chain5"]), ints([4]), 5, 7, ckv_rows=10)
    finish()
    assert torch.equal(ckv, want)


# ---------------------------------------------------------------------------------------------
# KDA
# ---------------------------------------------------------------------------------------------
def kda_inputs(gen, m, heads, n_states, g_low=-5.0):
    return dict(qkv=randn(gen, m, 3 * heads * 128).bfloat16(), g=(g_low * torch.sigmoid(2 * randn(gen, m, heads, 128))).contiguous(),
                beta=torch.sigmoid(randn(gen, m, heads)).bfloat16(), state=0.3 * randn(gen, n_states, heads, 128, 128))


def kda_wanted(x, heads, starts, trees, slots):
    """outputs in 64 bits, and what they may be off by: sums of 128 products, then the chain of a node's path in fp32 - 200 roundings a token of
    relative 2^-24 of the magnitudes, 8 ulp for exponentials of arguments down to -5 and the norms - of states, values and their sums that are at most M"""
    out = torch.zeros(x["qkv"].shape[0], heads, 128, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    for s, tree in enumerate(trees):
        made = {-1: x["state"][slots[s]].double()}
        for j in range(len(tree)):
            r = starts[s] + j
            q, k, v = x["qkv"][r].double().view(3, heads, 128)
            steps = path(tree, j)
            made[j], out[r] = kda_token(made[steps[-2] if len(steps) > 1 else -1], q, k, v, x["g"][r].double(), x["beta"][r].double())
            big = 128 ** 0.5 * x["state"][slots[s]].abs().max().double() + sum(x["qkv"][starts[s] + i].double().abs().max() for i in steps)
            tol[r] = (200 * 2.0 ** -24 + 64 * 2.0 ** -24) * len(steps) * big
    return out, tol


@pytest.mark.parametrize("trees", [["one"], ["chain5"], ["chain64"], ["wide63", "binary15"], ["star7", "one", "two_roots", (33, 1)], [(16, 2)] * 5, ["one", [], "chain5"]])
@pytest.mark.parametrize("heads", [1, 6, 40])
def test_recurrence_of_nodes(trees, heads):
    trees = [tree_of(t) for t in trees]
    gen = gen_of(heads + len(trees))
    starts, parent, tree_start = layout(trees, front=1)
    m = starts[-1] + 2
    parent = torch.cat((parent, ints([0, 0])))
    n = len(trees)
    slots = [(3 * s + 1) % (n + 2) if n < 3 else n + 1 - s for s in range(n)]
    x = kda_inputs(gen, m, heads, n + 2)
    held = x["state"].clone()
    out = torch.full((m, heads, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    f32 = torch.full((m, heads, 128), 7.0, device="cuda")
    hk.kda_tree_decode(x["qkv"], x["g"], x["beta"], x["state"], parent, out, m, heads, n_seqs=n, tree_start=tree_start, slots=ints(slots), out_f32=f32)
    finish()
    assert torch.equal(x["state"], held), "states stay as they are"
    want, tol = kda_wanted(x, heads, starts, trees, slots)
    mine = slice(1, starts[-1])
    off = (f32.double() - want).abs()
    assert bool((off <= tol)[mine].all()), float(off[mine].max())
    toward_zero = (f32.view(torch.int32) & -65536).view(torch.float32)
    assert torch.equal(out[mine].float(), toward_zero[mine])
    for r in [0] + list(range(starts[-1], m)):
        assert bool((f32[r] == 7).all()) and bool((out[r] == 7).all()), "rows of no tree are left as they were"


@pytest.mark.parametrize("nodes", [1, 2, 15, 16, 17, 31, 32, 33, 64])
@pytest.mark.parametrize("heads", [2, 20, 60])
def test_recurrence_of_trees_of_a_told_size(nodes, heads):
    """the forms for up to 16, 32 and 64 nodes, with 32, 64 and 128 columns a CTA"""
    trees = [tree_of((nodes, 1)), tree_of((max(1, nodes - 3), 2)), tree_of((nodes, 5))]
    gen = gen_of(nodes + heads)
    starts, parent, tree_start = layout(trees)
    m = starts[-1]
    x = kda_inputs(gen, m, heads, 3)
    out, f32 = torch.empty(m, heads, 128, dtype=torch.bfloat16, device="cuda"), torch.empty(m, heads, 128, device="cuda")
    hk.kda_tree_decode(x["qkv"], x["g"], x["beta"], x["state"], parent, out, m, heads, n_seqs=3, tree_start=tree_start, out_f32=f32, max_nodes=nodes)
    finish()
    want, tol = kda_wanted(x, heads, starts, trees, [0, 1, 2])
    off = (f32.double() - want).abs()
    assert bool((off <= tol).all()), float((off - tol).max())


@pytest.mark.parametrize("most", [1, 7, 16, 20, 40])
def test_nodes_beyond_the_told_number_are_left_as_they_were(most):
    gen, heads, tree = gen_of(21), 3, tree_of((50, 4))
    x = kda_inputs(gen, 50, heads, 1)
    all_of, some = (torch.full((50, heads, 128), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    a = (x["qkv"], x["g"], x["beta"], x["state"], ints(tree))
    hk.kda_tree_decode(*a, all_of, 50, heads, tree_start=ints([0, 50]))
    hk.kda_tree_decode(*a, some, 50, heads, tree_start=ints([0, 50]), max_nodes=most)
    finish()
    assert bool((some[most:] == 7).all())
    # the same sums in other orders, rounded to bf16 toward zero: a step of bf16 and 1e-5 of the largest
    off = (some[:most].double() - all_of[:most].double()).abs()
    assert bool((off <= 2.0 ** -7 * all_of[:most].double().abs() + 1e-5 * all_of.double().abs().max()).all())


def test_rows_and_states_beyond_four_gigabytes():
    """caches of 4.3 million rows and 70,000 blocks, states in slot 70,000"""
    gen, n, rows = gen_of(22), 700, 4_300_000
    tree = tree_of("binary15")
    q, kv = (randn(gen, 15, 64, 512) * 0.7).half(), randn(gen, 15, 512).half()
    ckv = torch.empty(rows, 512, dtype=torch.float16, device="cuda")
    first = rows - n - 20
    ckv[first:first + n] = randn(gen, n, 512).half()
    base, lens, leaf, told = torch.tensor([first], device="cuda"), ints([n]), ints([14]), ints([0])
    want = wanted(q, ckv[first:first + n].double(), kv, 0, tree, 0.0625)
    for splits in (0, 1, 4):
        out = torch.empty(15, 64, 512, dtype=torch.float16, device="cuda")
        hk.mla_tree_decode(q, ckv, kv, ints(tree), out, 15, kv_base=base, kv_len=lens, n_keys_hint=n, n_split=splits)
        finish()
        check_rows(out, want)
    hk.mla_tree_accept(kv, ckv, ints(tree), leaf, 15, kv_base=base, kv_len=lens, len_out=told)
    finish()
    steps = path(tree, 14)
    assert int(told) == n + len(steps) and torch.equal(ckv[first + n:first + n + len(steps)], kv[steps])
    del ckv
    blocks = 70_000                                          # of 128 tokens: 4.6 GB
    ckv8 = torch.empty(blocks, 128, 512, dtype=torch.int8, device="cuda")
    scales = torch.ones(blocks, device="cuda")
    some, s = cache(gen, "i8", 6, 128)
    ckv8[-6:], scales[-6:] = some, s
    table = ints([list(range(blocks - 6, blocks))])
    want = wanted(q, rows_of(ckv8, scales, table[0], torch.arange(n, device="cuda")), kv, 0, tree, 0.0625)
    out = torch.empty(15, 64, 512, dtype=torch.float16, device="cuda")
    hk.mla8_tree_decode(q, ckv8, scales, kv, ints(tree), out, 15, block_table=table, kv_len=lens, n_keys_hint=n)
    finish()
    check_rows(out, want)
    hk.mla8_tree_accept(kv, ckv8, scales, ints(tree), leaf, 15, block_table=table, kv_len=lens)
    finish()
    got = rows_of(ckv8, scales, table[0], torch.arange(n, n + len(steps), device="cuda"))
    assert bool(((got - kv[steps].double()).abs() <= 0.5 * scales[-1].double() * 1.01 + 0.5 * float(s[-1])).all()), "half a step of the block's scale, before and after it grew"
    del ckv8
    x = kda_inputs(gen, 15, 1, 1)
    state = torch.empty(70_001, 1, 128, 128, device="cuda")
    state[-1] = x["state"][0]
    near, far = (torch.empty(15, 1, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    a = (x["qkv"], x["g"], x["beta"])
    hk.kda_tree_decode(*a, x["state"], ints(tree), near, 15, 1)
    hk.kda_tree_decode(*a, state, ints(tree), far, 15, 1, slots=ints([70_000]))
    hk.kda_tree_accept(None, None, *a, x["state"], ints(tree), leaf, 15, 1)
    hk.kda_tree_accept(None, None, *a, state, ints(tree), leaf, 15, 1, slots=ints([70_000]))
    finish()
    assert torch.equal(near, far) and torch.equal(state[-1], x["state"][0])


def test_hard_resets_and_gates_of_zero():
    """log decays of 0, -100 and minus infinity on a long chain: nothing overflows, what is forgotten is nothing"""
    gen, heads, tree = gen_of(11), 2, TREES["chain64"]
    x = kda_inputs(gen, 64, heads, 1)
    x["g"][::3], x["g"][1::7], x["g"][2::9] = 0.0, -100.0, -INF
    f32 = torch.empty(64, heads, 128, device="cuda")
    hk.kda_tree_decode(x["qkv"], x["g"], x["beta"], x["state"], ints(tree), torch.empty(64, heads, 128, dtype=torch.bfloat16, device="cuda"), 64, heads, out_f32=f32)
    finish()
    want, tol = kda_wanted(x, heads, [0], [tree], [0])
    assert bool(((f32.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("nodes", [9, 30, 60])
@pytest.mark.parametrize("heads", [2, 60, 200])
def test_states_of_the_largest_numbers(nodes, heads):
    """states up to the largest number of fp32, which bf16 has no neighbour above for; one that is not finite shows in its column of every node, and nowhere else"""
    gen, tree = gen_of(nodes), tree_of((nodes, 1))
    x = kda_inputs(gen, nodes, heads, 1)

    def call():
        f32 = torch.empty(nodes, heads, 128, device="cuda")
        hk.kda_tree_decode(x["qkv"], x["g"], x["beta"], x["state"], ints(tree), torch.empty(nodes, heads, 128, dtype=torch.bfloat16, device="cuda"), nodes, heads, out_f32=f32)
        finish()
        return f32

    x["state"][0, :, [5, 100, 3, 64], [7, 70, 127, 0]] = 0.0
    base = call()
    x["state"][0, :, [5, 100, 3, 64], [7, 70, 127, 0]] = torch.tensor([3.4e38, -3.395e38, torch.finfo(torch.float32).max, -3.38953139e38], device="cuda")
    out, (want, tol) = call(), kda_wanted(x, heads, [0], [tree], [0])
    large = [0, 7, 70, 127]
    rest = [c for c in range(128) if c not in large]
    assert bool(torch.isfinite(out).all()) and torch.equal(out[..., rest], base[..., rest])
    assert bool(((out.double() - want).abs() <= tol)[..., large].all())
    x["state"][0, :, [5, 100, 3, 64], [7, 70, 127, 0]] = torch.tensor([INF, -INF, NAN, INF], device="cuda")
    out = call()
    assert not bool(torch.isfinite(out[..., large]).any()) and torch.equal(out[..., rest], base[..., rest])


@pytest.mark.parametrize("nodes", [1, 16, 17, 33, 64])
@pytest.mark.parametrize("heads", [3, 40, 90])
def test_how_precise_the_products_with_the_state_are(nodes, heads):
    """Children of the sequence alone, so that out_f32 is (q E)^T S + (q k) u, u = beta (v - (k E)^T S).  A number is two of bf16 and at most 2^-16 of it: of a product's
    four parts the smallest may be left out, 3 * 2^-16 of the product at most, and 384 additions in fp32 lose 2^-23 of the magnitudes each (the tensor cores may cut off).
    Rows are fp32: norm, product and exponential of an argument down to -5 are within 16 roundings of 2^-24.  q k is a sum of 128 products of such rows."""
    gen = gen_of(nodes + heads)
    x = kda_inputs(gen, nodes, heads, 1)
    f32 = torch.empty(nodes, heads, 128, device="cuda")
    hk.kda_tree_decode(x["qkv"], x["g"], x["beta"], x["state"], ints([-1] * nodes), torch.empty(nodes, heads, 128, dtype=torch.bfloat16, device="cuda"), nodes, heads, out_f32=f32)
    finish()
    q, k, v = x["qkv"].double().view(nodes, 3, heads, 128).unbind(1)
    q, k = (r / torch.sqrt(r.pow(2).sum(-1, keepdim=True) + 1e-6) for r in (q, k))
    e, s, beta = torch.exp(x["g"].double()), x["state"][0].double(), x["beta"].double()[..., None]
    dot = lambda a, b: torch.einsum("nhk,hkv->nhv", a, b)  # noqa: E731
    row = 16 * 2.0 ** -24
    part = 3 * 2.0 ** -16 + 384 * 2.0 ** -23 + row
    u = beta * (v - dot(k * e, s))
    u_mag = beta * (v.abs() + dot((k * e).abs(), s.abs()))
    u_off = beta * part * dot((k * e).abs(), s.abs()) + 4 * 2.0 ** -24 * u_mag
    qk, qk_mag = (q * k).sum(-1, keepdim=True), (q * k).abs().sum(-1, keepdim=True)
    want = dot(q * e, s) + qk * u
    mag = dot((q * e).abs(), s.abs()) + qk_mag * u_mag
    tol = part * dot((q * e).abs(), s.abs()) + qk.abs() * u_off + (130 * 2.0 ** -24 + 2 * row) * qk_mag * (u.abs() + u_off) + 8 * 2.0 ** -24 * mag
    assert bool(((f32.double() - want * 128 ** -0.5).abs() <= tol * 128 ** -0.5).all())


def test_what_is_not_on_a_nodes_path_has_no_effect_on_it():
    gen, heads, tree = gen_of(12), 3, tree_of("binary15")
    x = kda_inputs(gen, 15, heads, 1)

    def call():
        f32 = torch.empty(15, heads, 128, device="cuda")
        hk.kda_tree_decode(x["qkv"], x["g"], x["beta"], x["state"], ints(tree), torch.empty(15, heads, 128, dtype=torch.bfloat16, device="cuda"), 15, heads,
                           out_f32=f32)
        finish()
        return f32

    good = call()
    x["qkv"][4], x["g"][6], x["beta"][9] = NAN, INF, INF
    out = call()
    for j in range(15):
        if not {4, 6, 9} & set(path(tree, j)):
            assert torch.equal(out[j], good[j]), j


@pytest.mark.parametrize("heads", [5, 230])
def test_raw_gates_give_what_prepared_gates_give(heads):
    gen = gen_of(13)
    trees = [tree_of((20, 1)), tree_of("chain5")]
    starts, parent, tree_start = layout(trees)
    m = starts[-1]
    x = kda_inputs(gen, m, heads, 2)
    f, b, dt, a_log = randn(gen, m, heads, 128), randn(gen, m, heads), 0.5 * randn(gen, heads, 128), randn(gen, heads)
    g, beta = torch.empty(m, heads, 128, device="cuda"), torch.empty(m, heads, dtype=torch.bfloat16, device="cuda")
    hk.kda_gate(b, f, dt, a_log, -5.0, beta, g, m, heads, 128)
    outs, states = [], []
    for args, more in (((g, beta), {}), ((f, b), dict(dt_bias=dt, a_log=a_log, lower_bound=-5.0))):
        out, st = torch.empty(m, heads, 128, device="cuda"), x["state"].clone()
        hk.kda_tree_decode(x["qkv"], *args, st, parent, torch.empty(m, heads, 128, dtype=torch.bfloat16, device="cuda"), m, heads, n_seqs=2, tree_start=tree_start,
                           out_f32=out, **more)
        hk.kda_tree_accept(None, None, x["qkv"], *args, st, parent, ints([19, 3]), m, heads, n_seqs=2, tree_start=tree_start, **more)
        outs.append(out)
        states.append(st)
    finish()
    assert torch.equal(*outs) and torch.equal(*states)


@pytest.mark.parametrize("heads,n", [(2, 1), (16, 5), (40, 3), (96, 5)])
def test_accepted_states_are_those_of_token_by_token_decoding(heads, n):
    """bit for bit: the states of the recurrence over the path's tokens, the windows of the convolution over them"""
    trees = [tree_of(t) for t in ("binary15", "chain64", (17, 4), "one", "star7")[:n]]
    leaves = [14, 63, 16, -1, 7][:n]                          # the last two: none
    gen, dim = gen_of(heads), 3 * heads * 128
    starts, parent, tree_start = layout(trees)
    m = starts[-1]
    slots = [n - s for s in range(n)]
    x = kda_inputs(gen, m, heads, n + 1)
    x32, window = randn(gen, m, dim), randn(gen, n + 1, dim, 4).bfloat16()
    state, win = x["state"].clone(), window.clone()
    hk.kda_tree_accept(x32, win, x["qkv"], x["g"], x["beta"], state, parent, ints(leaves), m, heads, n_seqs=n, tree_start=tree_start, slots=ints(slots))
    finish()
    for s in range(n):
        steps = path(trees[s], leaves[s]) if 0 <= leaves[s] < len(trees[s]) else []
        rows, k = [starts[s] + j for j in steps], len(steps)
        if k:
            one = x["state"][slots[s]:slots[s] + 1].clone()
            out = torch.empty(1, k, heads, 128, dtype=torch.bfloat16, device="cuda")
            hk.cuda_recurrent_gated_delta_rule(x["qkv"][rows].contiguous(), x["g"][rows].contiguous(), x["beta"][rows].contiguous(), one, out, 1, k, heads, heads, 128, 128, 1,
                                               None, True, False, force_recurrent=True)
            w = window[slots[s]:slots[s] + 1].clone()
            hk.kda_cast_conv(x32[rows].contiguous(), w, None, torch.zeros(dim, 4, dtype=torch.bfloat16, device="cuda"), None, torch.empty(1, k, dim, dtype=torch.bfloat16, device="cuda"),
                             1, dim, k, True)
            finish()
            assert torch.equal(state[slots[s]], one[0]) and torch.equal(win[slots[s]], w[0]), s
            exact = x["state"][slots[s]].double()
            for r in rows:
                q, kk, v = x["qkv"][r].double().view(3, heads, 128)
                exact, _ = kda_token(exact, q, kk, v, x["g"][r].double(), x["beta"][r].double())
            assert float((state[slots[s]].double() - exact).norm() / exact.norm()) < 1e-5
        else:
            assert torch.equal(state[slots[s]], x["state"][slots[s]]) and torch.equal(win[slots[s]], window[slots[s]]), s
    assert torch.equal(state[0], x["state"][0]) and torch.equal(win[0], window[0]), "a slot of nobody"


@pytest.mark.parametrize("raw", [False, True])
def test_accepted_states_that_stream_through_shared_memory(raw):
    """four accepted heads a CTA and more, so that every buffer is used again: paths of one to eight batches of tokens, sequences without an accepted node in between;
    bit for bit what decoding token by token gives"""
    heads, lengths = 64, [1, 8, 9, 16, 64, 2, 7, 17, 3, 24, 5]
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    n = (8 * sms // heads + 1) * 4 // 3 + 2
    gen, dim = gen_of(77), 3 * heads * 128
    trees = [list(range(-1, lengths[s % len(lengths)] - 1)) if s % 3 else tree_of((20 + s, s)) for s in range(n)]
    leaves = [(-1, 64)[s % 8 == 3] if s % 4 == 3 else len(t) - 1 for s, t in enumerate(trees)]
    assert heads * sum(s % 4 != 3 for s in range(n)) >= 4 * 2 * sms
    starts, parent, tree_start = layout(trees)
    m, slots = starts[-1], [(5 * s + 2) % n for s in range(n)]
    if math.gcd(5, n) > 1:
        slots = list(range(n))[::-1]
    x = kda_inputs(gen, m, heads, n)
    x32, window = randn(gen, m, dim), randn(gen, n, dim, 4).bfloat16()
    gates, more = (x["g"], x["beta"]), {}
    if raw:
        f, b, dt, a_log = randn(gen, m, heads, 128), randn(gen, m, heads), 0.5 * randn(gen, heads, 128), randn(gen, heads)
        hk.kda_gate(b, f, dt, a_log, -5.0, x["beta"], x["g"], m, heads, 128)
        gates, more = (f, b), dict(dt_bias=dt, a_log=a_log, lower_bound=-5.0)
    state, win = x["state"].clone(), window.clone()
    hk.kda_tree_accept(x32, win, x["qkv"], *gates, state, parent, ints(leaves), m, heads, n_seqs=n, tree_start=tree_start, slots=ints(slots), **more)
    alone = x["state"].clone()                               # the states without windows
    hk.kda_tree_accept(None, None, x["qkv"], *gates, alone, parent, ints(leaves), m, heads, n_seqs=n, tree_start=tree_start, slots=ints(slots), **more)
    finish()
    assert torch.equal(alone, state)
    taps = torch.zeros(dim, 4, dtype=torch.bfloat16, device="cuda")
    for s in range(n):
        at = slice(slots[s], slots[s] + 1)
        one, w = x["state"][at].clone(), window[at].clone()
        rows = [starts[s] + j for j in path(trees[s], leaves[s])] if 0 <= leaves[s] < len(trees[s]) else []
        if rows:
            k = len(rows)
            hk.cuda_recurrent_gated_delta_rule(x["qkv"][rows].contiguous(), x["g"][rows].contiguous(), x["beta"][rows].contiguous(), one,
                                               torch.empty(1, k, heads, 128, dtype=torch.bfloat16, device="cuda"), 1, k, heads, heads, 128, 128, 1, None, True, False, force_recurrent=True)
            hk.kda_cast_conv(x32[rows].contiguous(), w, None, taps, None, torch.empty(1, k, dim, dtype=torch.bfloat16, device="cuda"), 1, dim, k, True)
        assert torch.equal(state[at], one) and torch.equal(win[at], w), s


@pytest.mark.parametrize("dim", [4, 384, 2060])
@pytest.mark.parametrize("bias,activation", [(True, True), (False, False)])
def test_convolution_of_nodes(dim, bias, activation):
    """bit for bit what the convolution of a node's path gives for its last token; the windows stay as they are"""
    trees = [tree_of(t) for t in ("binary15", "chain5", "two_roots")]
    gen = gen_of(dim)
    starts, parent, tree_start = layout(trees, front=1)
    m, slots = starts[-1], [2, 0, 3]
    x, window, w = randn(gen, m, dim), randn(gen, 4, dim, 4).bfloat16(), (0.3 * randn(gen, dim, 4)).bfloat16()
    b = randn(gen, dim).bfloat16() if bias else None
    held = window.clone()
    out = torch.full((m, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    hk.kda_tree_conv(x, window, w, b, parent, out, m, dim, n_seqs=3, tree_start=tree_start, slots=ints(slots), activation=activation)
    finish()
    assert torch.equal(window, held) and bool((out[0] == 7).all())
    for s, tree in enumerate(trees):
        for j in range(len(tree)):
            rows = [starts[s] + i for i in path(tree, j)]
            one = torch.empty(1, len(rows), dim, dtype=torch.bfloat16, device="cuda")
            hk.kda_cast_conv(x[rows].contiguous(), window[slots[s]:slots[s] + 1].clone(), None, w, b, one, 1, dim, len(rows), activation)
            assert torch.equal(out[starts[s] + j], one[0, -1]), (s, j)
            # and by the formula: three additions in fp32, the exponential, the rounding to bf16
            back = torch.cat((window[slots[s]].double(), x[rows].bfloat16().double().T), 1)[:, -4:]
            y = (back * w.double()).sum(1) + (b.double() if bias else 0)
            mag = (back * w.double()).abs().sum(1) + (b.double().abs() if bias else 0)
            y = y * torch.sigmoid(y) if activation else y
            assert bool(((out[starts[s] + j].double() - y).abs() <= 2.0 ** -8 * y.abs() + 2.0 ** -19 * mag + 2.0 ** -30).all())


# ---------------------------------------------------------------------------------------------
# as they are used
# ---------------------------------------------------------------------------------------------
def test_a_drafted_step_and_the_tokens_decoded_one_by_one():
    """verify a tree in a KDA and an MLA layer, accept a node, go on: the same states, windows and cache as decoding the accepted tokens alone"""
    gen, heads, n = gen_of(20), 4, 137
    tree = tree_of((24, 9))
    leaf = max(range(24), key=lambda j: len(path(tree, j)))
    m, dim, steps = len(tree), 3 * heads * 128, path(tree, leaf)
    x32, f, b = randn(gen, m, dim), randn(gen, m, heads, 128), randn(gen, m, heads)
    dt, a_log, w = 0.5 * randn(gen, heads, 128), randn(gen, heads), (0.3 * randn(gen, dim, 4)).bfloat16()
    state, window = 0.3 * randn(gen, 1, heads, 128, 128), randn(gen, 1, dim, 4).bfloat16()
    ckv = torch.zeros(n + 64, 512, dtype=torch.float16, device="cuda")
    ckv[:n] = randn(gen, n, 512).half()
    kv_pre, ln_w = randn(gen, m, 512), (1 + 0.1 * randn(gen, 512)).half()
    q = (randn(gen, m, 64, 512) * 0.7).half()
    parent = ints(tree)
    # one by one: what decoding does with the accepted tokens
    st1, w1, c1, outs1, lat1 = state.clone(), window.clone(), ckv.clone(), [], []
    norm_w, gate = torch.ones(128, dtype=torch.bfloat16, device="cuda"), randn(gen, heads, 128)
    for i, j in enumerate(steps):
        out = torch.empty(1, heads, 128, dtype=torch.bfloat16, device="cuda")
        hk.kda_decode_layer(x32[j].contiguous(), w1, w, None, f[j].contiguous(), b[j].contiguous(), dt, a_log, -5.0, st1, out, norm_w, gate, torch.empty(heads, 128, dtype=torch.float16, device="cuda"), 1, heads)
        hk.mla_cache_append(kv_pre[j:j + 1].contiguous(), ln_w, c1, n + i, 1, 1e-6)
        lat = torch.empty(1, 64, 512, dtype=torch.float16, device="cuda")
        hk.mla_dense_prefill(q[j:j + 1].contiguous(), c1, lat, 1, n + i)
        outs1.append(out)
        lat1.append(lat)
    # the tree
    qkv, out, lat = (torch.empty(m, dim, dtype=torch.bfloat16, device="cuda"), torch.empty(m, heads, 128, dtype=torch.bfloat16, device="cuda"),
                     torch.empty(m, 64, 512, dtype=torch.float16, device="cuda"))
    raw = dict(dt_bias=dt, a_log=a_log, lower_bound=-5.0)
    rows = torch.empty(m, 512, dtype=torch.float16, device="cuda")
    hk.kda_tree_conv(x32, window, w, None, parent, qkv, m, dim)
    hk.kda_tree_decode(qkv, f, b, state, parent, out, m, heads, **raw)
    hk.mla_cache_append(kv_pre, ln_w, rows, 0, m, 1e-6)          # the nodes' latents, normalised into a buffer of their own
    hk.mla_tree_decode(q, ckv, rows, parent, lat, m, n)
    hk.kda_tree_accept(x32, window, qkv, f, b, state, parent, ints([leaf]), m, heads, **raw)
    length = torch.zeros(1, dtype=torch.int32, device="cuda")
    hk.mla_tree_accept(rows, ckv, parent, ints([leaf]), m, n, len_out=length)
    finish()
    assert torch.equal(state, st1) and torch.equal(window, w1) and torch.equal(ckv, c1) and int(length) == n + len(steps)
    for i, j in enumerate(steps):
        # fp32 sums in two orders, rounded to bf16 toward zero: a step of bf16 and 1e-5 of the largest
        a, c = out[j].double(), outs1[i][0].double()
        assert bool(((a - c).abs() <= 2.0 ** -7 * c.abs() + 1e-5 * c.abs().max()).all()), i
        o, tol = attend(q[j].double(), c1[:n + i + 1].double(), 0.0625)
        assert bool(((lat[j].double() - o).abs() <= tol).all()) and bool(((lat1[i][0].double() - o).abs() <= tol).all()), i


@pytest.mark.parametrize("kind", ["tree", "tree8", "kda"])
def test_captured_and_replayed_and_on_a_stream_of_its_own(kind):
    """trees, lengths and accepted nodes are the device's: a captured call follows them"""
    gen, heads = gen_of(30), 64
    trees = [tree_of((10, 1)), tree_of("chain5")]
    starts, parent, tree_start = layout(trees)
    m, lens = starts[-1], ints([300, 90])
    q, rows = (randn(gen, m, heads, 512) * 0.7).half(), randn(gen, m, 512).half()
    ckv8, scales = cache(gen, "e4m3", 12, 64)
    table, ckv = table_for(gen, 2, 6, 12), randn(gen, 800, 512).half()
    base = torch.tensor([0, 400], device="cuda")
    x = kda_inputs(gen, m, 6, 2)

    def call(out, stream=None):
        at = dict(n_seqs=2, tree_start=tree_start, stream=stream)
        if kind == "tree":
            hk.mla_tree_decode(q, ckv, rows, parent, out, m, kv_base=base, kv_len=lens, n_keys_hint=384, **at)
        elif kind == "tree8":
            hk.mla8_tree_decode(q, ckv8, scales, rows, parent, out, m, block_table=table, kv_len=lens, n_keys_hint=384, **at)
        else:
            hk.kda_tree_decode(x["qkv"], x["g"], x["beta"], x["state"], parent, out, m, 6, **at)

    fresh = lambda: torch.zeros(m, 6, 128, dtype=torch.bfloat16, device="cuda") if kind == "kda" else torch.zeros(m, heads, 512, dtype=torch.float16, device="cuda")  # noqa: E731
    first = fresh()
    call(first)
    side, there = torch.cuda.Stream(), fresh()
    side.wait_stream(torch.cuda.current_stream())
    call(there, side)
    finish()
    assert torch.equal(first, there)
    out = fresh()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    graph.replay()
    finish()
    assert torch.equal(out, first)
    # other trees, lengths and inputs under the same graph
    parent.copy_(ints(tree_of((m, 8))))
    tree_start.copy_(ints([0, 3, m]))
    lens.copy_(ints([17, 380]))
    q.copy_(q.flip(0))
    x["g"].mul_(0.5)
    graph.replay()
    again = fresh()
    call(again)
    finish()
    assert torch.equal(out, again) and not torch.equal(out, first)


def test_two_calls_at_once():
    """calls on two streams, each with scratch of its own, give what each gives alone"""
    gen, tree = gen_of(31), tree_of((40, 3))
    parent, lens = ints(tree), ints([1500])
    q, kv, ckv = (randn(gen, 40, 64, 512) * 0.7).half(), randn(gen, 40, 512).half(), randn(gen, 1500, 512).half()
    ckv8, scales = cache(gen, "e4m3", 24, 64)
    x = kda_inputs(gen, 40, 50, 1)
    calls = (lambda o, st: hk.mla_tree_decode(q, ckv, kv, parent, o, 40, kv_len=lens, n_keys_hint=1500, stream=st),
             lambda o, st: hk.mla8_tree_decode(q, ckv8, scales, kv, parent, o, 40, kv_len=lens, n_keys_hint=1500, stream=st),
             lambda o, st: hk.kda_tree_decode(x["qkv"], x["g"], x["beta"], x["state"], parent, o, 40, 50, stream=st))
    fresh = lambda i: torch.empty(40, 50, 128, dtype=torch.bfloat16, device="cuda") if i == 2 else torch.empty(40, 64, 512, dtype=torch.float16, device="cuda")  # noqa: E731
    alone = [fresh(i) for i in range(3)]
    for i, call in enumerate(calls):
        call(alone[i], None)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[fresh(i) for i in range(3)] for _ in range(8)]
    finish()
    for k, out in enumerate(outs):
        for i in range(3):
            calls[(i + k) % 3](out[(i + k) % 3], streams[k % 2])
    finish()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, alone))


def test_the_same_call_gives_the_same_bits():
    """a CTA a node with splits, pairs of CTAs, several nodes a CTA; the 8-bit cache converted and read first; every form of the recurrence and of the accepted step"""
    gen = gen_of(41)
    ckv = randn(gen, 9000, 512).half()
    ckv8, scales = cache(gen, "e4m3", 150, 64, spread=0.7)
    calls, keep = [], []
    for nodes, heads, n in ((8, 64, 5001), (64, 64, 4000), (40, 16, 2000), (1, 64, 9000), (3, 20, 700)):
        tree, q, rows = ints(tree_of((nodes, 1))), (randn(gen, nodes, heads, 512) * 0.7).half(), randn(gen, nodes, 512).half()
        calls.append((lambda o, a=(tree, q, rows, nodes, heads, n): hk.mla_tree_decode(a[1], ckv, a[2], a[0], o, a[3], a[5], n_heads=a[4]), (nodes, heads, 512), torch.float16))
        calls.append((lambda o, a=(tree, q, rows, nodes, heads, n): hk.mla8_tree_decode(a[1], ckv8, scales, a[2], a[0], o, a[3], a[5], n_heads=a[4]), (nodes, heads, 512), torch.float16))
    for nodes, heads in ((8, 2), (30, 60), (61, 200), (13, 400)):
        x, tree = kda_inputs(gen, nodes, heads, 1), ints(tree_of((nodes, 2)))
        keep.append(x)
        calls.append((lambda o, a=(x, tree, nodes, heads): hk.kda_tree_decode(a[0]["qkv"], a[0]["g"], a[0]["beta"], a[0]["state"], a[1], o, a[2], a[3]), (nodes, heads, 128), torch.bfloat16))

        def accept(o, a=(x, tree, nodes, heads)):
            o.copy_(a[0]["state"])
            hk.kda_tree_accept(None, None, a[0]["qkv"], a[0]["g"], a[0]["beta"], o, a[1], ints([a[2] - 1]), a[2], a[3])

        calls.append((accept, (1, heads, 128, 128), torch.float32))
    for call, shape, dtype in calls:
        outs = [torch.empty(shape, dtype=dtype, device="cuda") for _ in range(4)]
        for o in outs:
            call(o)
        finish()
        assert all(torch.equal(o, outs[0]) for o in outs), shape


def test_calls_without_rows_do_nothing():
    e = lambda *s: torch.empty(*s, dtype=torch.float16, device="cuda")  # noqa: E731
    none = ints([0])
    hk.mla_tree_decode(e(0, 64, 512), e(4, 512), e(0, 512), none, e(0, 64, 512), 0, 4)
    hk.kda_tree_decode(torch.empty(0, 384, dtype=torch.bfloat16, device="cuda"), torch.empty(0, 1, 128, device="cuda"), torch.empty(0, 1, dtype=torch.bfloat16, device="cuda"),
                       torch.zeros(1, 1, 128, 128, device="cuda"), none, torch.empty(0, 1, 128, dtype=torch.bfloat16, device="cuda"), 0, 1)
    length = ints([0])
    hk.mla_tree_accept(e(0, 512), e(4, 512), none, ints([3]), 0, 2, len_out=length)
    finish()
    assert int(length) == 2


def test_tensors_that_are_not_the_calls_are_refused():
    m = 3
    q, kv, out, c = (torch.zeros(s, dtype=torch.float16, device="cuda") for s in ((m, 64, 512), (m, 512), (m, 64, 512), (8, 512)))
    p = ints([-1, 0, 1])
    good = dict(q_lat=q, ckv=c, tree_kv=kv, parent=p, lat_out=out, m=m, pos_start=8)
    hk.mla_tree_decode(**good)
    for name, bad in (("q_lat", q.float()), ("tree_kv", kv[:2]), ("parent", p.long()), ("parent", p[:2]), ("ckv", c.t()), ("lat_out", out.cpu())):
        with pytest.raises(ValueError):
            hk.mla_tree_decode(**{**good, name: bad})
    for more in (dict(tree_start=ints([0])), dict(kv_len=ints([])), dict(kv_base=ints([0]))):
        with pytest.raises(ValueError):
            hk.mla_tree_decode(**good, **more)
    for more in (dict(pos_start=9), dict(n_seqs=2), dict(n_seqs=0), dict(n_heads=6), dict(pos_start=-1)):
        with pytest.raises((hk.HeliosB200Error, ValueError)):
            hk.mla_tree_decode(**{**good, **more})
    s, b = torch.zeros(1, 1, 128, 128, device="cuda"), torch.bfloat16
    kda = dict(mixed_qkv=torch.zeros(m, 384, dtype=b, device="cuda"), g=torch.zeros(m, 1, 128, device="cuda"), beta=torch.zeros(m, 1, dtype=b, device="cuda"), rec_state=s, parent=p,
               out=torch.zeros(m, 1, 128, dtype=b, device="cuda"), m=m, num_heads=1)
    hk.kda_tree_decode(**kda)
    for more in (dict(max_nodes=65), dict(max_nodes=-1), dict(rec_state=s[:, :, :64]), dict(beta=kda["beta"].float()), dict(dt_bias=torch.zeros(1, 128, device="cuda")), dict(n_seqs=2),
                 dict(out=kda["out"].float())):
        with pytest.raises((hk.HeliosB200Error, ValueError)):
            hk.kda_tree_decode(**{**kda, **more})
    finish()
