"""What the header promises of the 8-bit cache and of windows where ordinary inputs do not go."""
import math
import os
import subprocess
import sys

import pytest
import torch

import helios_glm53flash_b200 as hk
from latent8_ref import STORE, TOP, attend, cache, rows_of, table_for, visible
from test_gpu_mla8 import close, finish, gen_of, ints, queries

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------
# blocks of very unequal scales
# ---------------------------------------------------------------------------------------------
def attend_by_weight(q, keys, key_scale, top, scale):
    """q [heads][512], keys [n][512] in 64 bits, key_scale [n]: their blocks' scales -> (output, what it may be off by), by the keys that weigh.

    A score is an fp32 sum of 512 products, scaled twice: 520 roundings at most of relative 2^-24 of its own key's sum of magnitudes, and 2^-20 of
    itself and of 1 for the exponential; that moves its weight relatively by as much.  A weight times its key's scale is rounded to fp16: half a
    step, 2^-11, relative, or 2^-25 of the reference where that leaves fp16's normal range; the reference is at most 2^4 of the largest product of
    the two.  The sum of n weights in fp32 adds n 2^-24, the output's own rounding 2^-11 or half of fp16's smallest step, 2^-25."""
    s = q @ keys.T * scale
    p = torch.exp(s - s.amax(1, keepdim=True))
    tot = p.sum(1, keepdim=True)
    o = p @ keys / tot
    eta = torch.expm1((2.0 ** -24 * 520 * (q.abs() @ keys.abs().T) * scale + 2.0 ** -20 * (1 + s.abs())).clamp(max=500.0))
    moved = p * torch.where(p > 0, eta, torch.zeros_like(eta))
    mag = p @ keys.abs() / tot
    tol = (moved @ keys.abs() + moved.sum(1, keepdim=True) * o.abs()) / tot + keys.shape[0] * 2.0 ** -24 * o.abs()
    least = keys.shape[0] * 2.0 ** -21 * (p * key_scale).amax(1, keepdim=True) * top / tot
    return o, (tol + 2.0 ** -11 * (mag + o.abs()) + least) * 1.01 + 2.0 ** -25


def unequal(gen, kind, block, blocks, heads, m, big, small, low):
    """a sequence of `blocks` blocks, every third of the scale `big`, the others of `small`; queries that score the big blocks' keys lower by about
    `low` by one channel, in which all heads are 2; a big block's other values are in channels where the queries are 0"""
    top = TOP[kind]
    v = torch.randn(blocks, block, 512, device="cuda", generator=gen).clamp(-3, 3) * (top / 3)
    heavy = torch.arange(blocks, device="cuda") % 3 == 1
    v[heavy, :, :256] = 0.0
    v[heavy, :, 7] = -round(low / (0.0625 * 2 * big)) if kind == "i8" else -low / (0.0625 * 2 * big)
    ckv8 = (v.round() if kind == "i8" else v).to(STORE[kind])
    scales = torch.where(heavy, big, small).float()
    q = torch.randn(m, heads, 512, device="cuda", generator=gen) * 0.7
    q[:, :, 7] = 2.0
    q[:, :, 256:] = 0.0
    return ckv8, scales, q.half()


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("block", [16, 32, 64, 128])                # several blocks a tile of 64 keys, one, half of one
@pytest.mark.parametrize("big,small,low", [(100.0, 1e-3, 12.5), (100.0, 1e-4, 37.5), (100.0, 1e-5, 400), (100.0, 1e-5, 25), (1e4, 1e-3, 1250), (2e4, 3e-4, 2500)])
def test_blocks_that_weigh_keep_their_bits_beside_blocks_of_large_scale(kind, block, big, small, low):
    """large-scale blocks far below in score, or so that both weigh; decode, one CTA and several, fewer heads, gathered positions, a short chunk"""
    gen = gen_of(block + int(low))
    n, m = 700, 3
    blocks = (n + block - 1) // block
    ckv8, scales, q = unequal(gen, kind, block, blocks, 64, m, big, small, low)
    where = torch.randperm(blocks, device="cuda", generator=gen)
    pool, pool_s = torch.empty_like(ckv8.view(torch.uint8)), torch.empty_like(scales)
    pool[where], pool_s[where] = ckv8.view(torch.uint8), scales
    pool, table = pool.view(STORE[kind]), where.to(torch.int32)[None].contiguous()
    out = torch.empty(m, 64, 512, dtype=torch.float16, device="cuda")
    lens = [n, n - 1, block + 1]

    def check(got, row, p, heads):
        keys, ks = rows_of(pool, pool_s, table[0], p), pool_s[table[0][p // block].long()].double()
        close(got[row:row + 1], [attend_by_weight(q[row, :heads].double(), keys, ks, TOP[kind], 0.0625)])

    for heads, n_split in ((64, 0), (64, 1), (64, 4), (16, 0)):
        qh, oh = q[:, :heads].contiguous(), out[:, :heads].contiguous()
        hk.mla8_dense_prefill(qh, pool, pool_s, oh, m, 0, n_heads=heads, block_table=table, kv_len=ints(lens), n_keys_hint=n, n_split=n_split)
        finish()
        for r in range(m):
            check(oh, r, visible(lens[r], 0, 0), heads)
    hk.mla8_dense_prefill(q, pool, pool_s, out, m, 0, block_table=table, kv_len=ints(lens), n_keys_hint=1 << 20)         # shared out by length
    finish()
    for r in range(m):
        check(out, r, visible(lens[r], 0, 0), 64)
    hk.mla8_dense_prefill(q, pool, pool_s, out, m, n - m, block_table=table, window=300, sinks=3)
    finish()
    for r in range(m):
        check(out, r, visible(n - m + r + 1, 300, 3), 64)
    idx = torch.randint(0, n, (m, 333), device="cuda", generator=gen, dtype=torch.int32)
    for n_split in (0, 1):
        hk.mla8_sparse_decode(q, pool, pool_s, idx, 333, out, m, block_table=table, n_split=n_split)
        finish()
        for r in range(m):
            check(out, r, idx[r].long(), 64)


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("big,low", [(0.5, 6.0), (10.0, 12.5)])
def test_keys_of_zeros_that_score_highest(kind, big, low):
    """blocks of scale 0 have the score 0, the only keys with values score far below: those weigh little, and what they weigh is right"""
    gen, block, n = gen_of(61), 16, 600
    blocks = (n + block - 1) // block
    ckv8, scales, q = unequal(gen, kind, block, blocks, 64, 2, big, 0.0, low)
    out = torch.empty(2, 64, 512, dtype=torch.float16, device="cuda")
    for n_split in (0, 1, 3):
        hk.mla8_dense_prefill(q, ckv8, scales, out, 2, n - 2, n_split=n_split)
        finish()
        want = []
        for r in range(2):
            p = visible(n - 1 + r, 0, 0)
            want.append(attend_by_weight(q[r].double(), rows_of(ckv8, scales, torch.arange(blocks, device="cuda"), p), scales[p // block].double(), TOP[kind], 0.0625))
        close(out, want)


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("small", [1e-39, 3e-38, 1e-31, 1e-29])
def test_blocks_of_zeros_before_blocks_of_the_smallest_scales(kind, small):
    gen = gen_of(62)
    ckv8, _ = cache(gen, kind, 4, 64)
    q, out = queries(gen, 1, 64), torch.empty(1, 64, 512, dtype=torch.float16, device="cuda")
    for s in ([0.0, small, small, 0.0], [0.0, small, 1.0, small], [small, small, 0.0, 1.0], [0.0, 0.0, 0.0, small]):
        scales = torch.tensor(s, device="cuda")
        for n_split in (1, 2, 4):
            hk.mla8_dense_prefill(q, ckv8, scales, out, 1, 255, n_split=n_split)
            finish()
            p = torch.arange(256, device="cuda")
            close(out, [attend_by_weight(q[0].double(), rows_of(ckv8, scales, torch.arange(4, device="cuda"), p), scales[p // 64].double(), TOP[kind], 0.0625)])


# ---------------------------------------------------------------------------------------------
# keys that are not finite under a window
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("heads,rows,window,n_split,pos", [
    (64, 1, 100, 0, 800), (64, 1, 1000, 0, 1700), (64, 1, 3000, 0, 4000), (64, 1, 9000, 0, 9500), (64, 1, 1000, 1, 1700), (64, 1, 1000, 3, 1700), (64, 5, 700, 0, 1100),
    (64, 30, 300, 0, 600), (64, 200, 300, 0, 600), (64, 7, 2500, 1, 3000), (64, 40, 2500, 0, 3000), (16, 1, 100, 0, 800), (16, 3, 1000, 1, 1500), (16, 3, 1000, 4, 1500)])
def test_window_rows_that_see_a_key_that_is_not_finite(heads, rows, window, n_split, pos):
    """one CTA a row, a grid that walks rows, splits of every kind, clusters, pairs, the CUDA cores: a key with a NaN makes every channel of the rows
    that see it NaN, one with an infinity its own channels; other rows are as they would be without it.  At the window's first key, whose score can
    be the only one of a split, in its middle and at the row's own"""
    gen, sinks = gen_of(rows + window), 3
    clean = torch.randn(pos + rows, 512, device="cuda", generator=gen).half()
    q = queries(gen, rows, heads)
    q[:, :, 9] = 0.5                                           # the infinite channel: every head scores it the same way
    out = torch.empty(rows, heads, 512, dtype=torch.float16, device="cuda")
    lo, last = pos + rows - window, pos + rows - 1             # the last row's first and own key
    sees = lambda p: torch.tensor([p < sinks or pos + r + 1 - window <= p <= pos + r for r in range(rows)], device="cuda")
    for p in (1, lo, lo + window // 2, last):
        for bad, whole in ((math.nan, True), (math.nan, False), (math.inf, False), (-math.inf, False), (math.inf, True)):
            ckv = clean.clone()
            ckv[p, slice(None) if whole else 9] = bad
            hk.mla_window_prefill(q, ckv, out.zero_(), rows, pos, window, sinks=sinks, n_heads=heads, n_split=n_split)
            finish()
            hit = sees(p)
            if math.isnan(bad) or whole:
                assert torch.isnan(out[hit]).all(), (p, bad)
            else:
                assert not torch.isfinite(out[hit][:, :, 9]).any(), (p, bad)
            for r in torch.nonzero(~hit)[:, 0].tolist()[::7]:
                o, tol = attend(q[r].double(), ckv[:pos + r + 1][visible(pos + r + 1, window, sinks)].double(), 0.0625)
                assert bool(((out[r].double() - o).abs() <= tol).all()), (p, bad, r)


def test_window_rows_of_one_key_that_is_not_finite():
    """nothing else to see: an infinity that scores plus or minus infinity, a NaN; as a row's only split and as one of several"""
    gen = gen_of(71)
    ckv = torch.randn(400, 512, device="cuda", generator=gen).half()
    q = queries(gen, 1, 64)
    q[:, :, 9] = 0.5
    out = torch.empty(1, 64, 512, dtype=torch.float16, device="cuda")
    for bad in (math.inf, -math.inf, math.nan):
        ckv[399, 9] = bad
        for n_split in (0, 1, 2):
            hk.mla_window_prefill(q, ckv, out.zero_(), 1, 399, 1, n_split=n_split)
            finish()
            assert not torch.isfinite(out[:, :, 9]).any(), (bad, n_split)
        ckv[399 - 15:399, 9] = bad                             # sixteen such keys alone in the last tile, and finite ones before them
        for n_split in (0, 1, 7):
            hk.mla_window_prefill(q, ckv, out.zero_(), 1, 399, 400, n_split=n_split)
            finish()
            assert not torch.isfinite(out[:, :, 9]).any(), (bad, n_split)


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
def test_blocks_whose_scale_is_infinite(kind):
    """every key's score is infinite or NaN, whichever split has it"""
    gen = gen_of(72)
    ckv8, scales = cache(gen, kind, 3, 64)
    q, out = queries(gen, 1, 64), torch.empty(1, 64, 512, dtype=torch.float16, device="cuda")
    for bad in ([0, 1, 2], [1], [2]):
        s = scales.clone()
        s[bad] = math.inf
        for n_split in (1, 2, 3):
            hk.mla8_dense_prefill(q, ckv8, s, out.zero_(), 1, 128, n_split=n_split)
            finish()
            assert torch.isnan(out).all(), (bad, n_split)


# ---------------------------------------------------------------------------------------------
# the CUDA-core kernel, streams, the same call again
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("switch", ["HK_MLA_FORCE_SIMT", "HK_MLA_NO_TMA"])
def test_the_cuda_core_kernel_over_the_8_bit_cache(switch):
    """the form for machines without an encoder of tensor maps, in a process of its own: holes, sequence numbers out of range, NaN scales, windows, splits;
    asked for, and where the encoder is missing, when long chunks are read as fp16 rows first all the same"""
    names = ("test_dense8_rows", "test_dense8_chunk", "test_dense8_rows_and_blocks_that_do_not_count", "test_a_row_that_is_not_finite_is_seen_in_the_output",
             "test_splits_that_see_nothing", "test_sparse8", "test_window_rows", "test_dense8_without_a_table", "test_blocks_that_weigh", "test_keys_of_zeros")
    here = os.path.dirname(os.path.abspath(__file__))
    files = [os.path.join(here, f) for f in ("test_gpu_mla8.py", "test_gpu_mla8_contracts.py")]
    run = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-m", "gpu", "-p", "no:cacheprovider", "-k", " or ".join(names)] + files,
                         env={**os.environ, switch: "1"}, capture_output=True, text=True, timeout=600)
    assert run.returncode == 0, run.stdout[-3000:] + run.stderr[-2000:]


def test_windowed_calls_on_two_streams_at_once():
    gen = gen_of(32)
    sides = [torch.cuda.Stream() for _ in range(2)]
    states = [(torch.randn(3000, 512, device="cuda", generator=gen).half(), queries(gen, 2, 64), torch.empty(2, 64, 512, dtype=torch.float16, device="cuda")) for _ in sides]
    torch.cuda.synchronize()
    for _ in range(20):
        for stream, (ckv, q, out) in zip(sides, states):
            with torch.cuda.stream(stream):
                hk.mla_window_prefill(q, ckv, out, 2, 2998, 1000, sinks=3)
    finish()
    for ckv, q, out in states:
        close(out, [attend(q[r].double(), ckv[:2999 + r][visible(2999 + r, 1000, 3)].double(), 0.0625) for r in range(2)])


def test_the_same_call_gives_the_same_bits():
    gen, block = gen_of(33), 32
    ckv8, scales = cache(gen, "e4m3", 300, block, spread=1.0)
    q, ckv = queries(gen, 40, 64), torch.randn(5000, 512, device="cuda", generator=gen).half()
    table, lens = table_for(gen, 1, 300, 300), ints([9000 - 31 * i for i in range(40)])
    idx = torch.randint(0, 9000, (40, 700), device="cuda", generator=gen, dtype=torch.int32)
    got = []
    for _ in range(3):
        outs = [torch.empty(40, 64, 512, dtype=torch.float16, device="cuda") for _ in range(5)]
        hk.mla8_dense_prefill(q, ckv8, scales, outs[0], 40, 0, block_table=table, kv_len=lens, n_keys_hint=9000)
        hk.mla8_dense_prefill(q[:5], ckv8, scales, outs[1][:5], 5, 0, block_table=table, kv_len=lens[:5], n_keys_hint=9000)
        hk.mla8_dense_prefill(q, ckv8, scales, outs[2], 40, 9000, block_table=table, window=500, sinks=9)
        hk.mla8_sparse_decode(q, ckv8, scales, idx, 700, outs[3], 40, block_table=table)
        hk.mla_window_prefill(q, ckv, outs[4], 40, 4900, 900, sinks=9)
        outs[1][5:] = 0
        finish()
        got.append(outs)
    for outs in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs, got[0]))


@pytest.mark.parametrize("heads", [64, 16])
@pytest.mark.parametrize("window,sinks", [(1, 2 ** 31 - 1), (2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 30, 2 ** 30), (300, 7)])
def test_windows_and_lengths_of_all_31_bits(heads, window, sinks):
    """garbage in a padding row's length: the window stands where the length says, the cache's end cuts what is seen; times go by the cache"""
    gen, held = gen_of(91), 700
    ckv, q = torch.randn(held, 512, device="cuda", generator=gen).half(), queries(gen, 3, heads)
    out = torch.empty(3, heads, 512, dtype=torch.float16, device="cuda")
    lens = [2 ** 31 - 1, 500, 2 ** 31 - 40]
    want = []
    for r, n in enumerate(lens):
        p = torch.arange(min(n, held), device="cuda")
        want.append(attend(q[r].double(), ckv[p[(p >= n - window) | (p < sinks)]].double(), 0.0625))
    for n_split in (0, 1, 2, 5):
        hk.mla_window_prefill(q, ckv, out, 3, 0, window, sinks=sinks, n_heads=heads, kv_len=ints(lens), n_split=n_split, n_keys_hint=held)
        finish()
        close(out, want)


@pytest.mark.parametrize("heads,rows,pos,window,sinks", [(64, 1, 4999, 128, 0), (64, 1, 4999, 1016, 4), (64, 24, 3000, 1024, 64), (64, 4, 5000, 4096, 0), (16, 3, 2000, 512, 0),
                                                         (32, 24, 3000, 1024, 64), (64, 200, 500, 300, 5)])
def test_windows_in_the_workspace_that_is_said(heads, rows, pos, window, sinks):
    """the size functions' bytes are enough, for the library's own choice and the wrapper's, and nothing behind them is written"""
    gen = gen_of(rows + pos)
    ckv, q = torch.randn(pos + rows, 512, device="cuda", generator=gen).half(), queries(gen, rows, heads)
    out = torch.empty(rows, heads, 512, dtype=torch.float16, device="cuda")
    want = [attend(q[r].double(), ckv[:pos + r + 1][visible(pos + r + 1, window, sinks)].double(), 0.0625) for r in range(rows)]
    for wrapped in (False, True):
        need = (hk.mla_window_workspace_bytes if wrapped else hk.load_library().hk_mla_window_workspace_bytes)(rows, heads, pos + rows, window, sinks)
        ws = torch.full((need + 4096,), 0x5a, dtype=torch.uint8, device="cuda")
        if wrapped:
            hk.mla_window_prefill(q, ckv, out.zero_(), rows, pos, window, sinks=sinks, n_heads=heads, workspace=ws[:need] if need else None)
        else:
            hk._run("hk_mla_window", q, ckv, ckv, None, None, pos, window, sinks, out.zero_(), rows, heads, 0.0625, 0, ws[:need] if need else None, need, None)
        finish()
        close(out, want)
        assert (ws[need:] == 0x5a).all()


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("q7,scale,small", [(60000.0, 0.0625, 0.01), (60000.0, 1.0, 0.01), (-60000.0, 20.0, 0.01), (60000.0, 1e9, 1e-6), (-60000.0, 1e10, 1e-5)])
def test_scores_so_large_that_a_scale_is_lost_beside_them(kind, block, q7, scale, small):
    """one channel makes the scores, 0 for all keys but one, which has 37 at least: a row's output is that key's latent (its weight is rounded to
    fp16, and the output), whatever its block's scale, the largest or the smallest"""
    gen, n = gen_of(95), 320
    blocks, top = n // block, TOP[kind]
    v = torch.randn(blocks, block, 512, device="cuda", generator=gen).clamp(-3, 3) * (top / 4)
    ckv8 = (v.round() if kind == "i8" else v).to(STORE[kind])
    ckv8.view(torch.uint8)[:, :, 7] = 0                         # +0 in both types: the score 0
    scales = torch.where(torch.arange(blocks, device="cuda") % 2 == 0, 60000.0 / top, small).float()
    q = torch.zeros(2, 64, 512, dtype=torch.float16, device="cuda")
    q[:, :, 7] = q7
    out = torch.empty(2, 64, 512, dtype=torch.float16, device="cuda")
    for best in (3, n // 2 + 1, block + 5, n - block + 1, n - 1):
        c = ckv8.clone()
        c.view(torch.int8 if kind == "i8" else torch.uint8)[best // block, best % block, 7] = {"i8": 1, "e4m3": 0x38}[kind] if q7 > 0 else {"i8": -1, "e4m3": 0xb8}[kind]
        want = rows_of(c, scales, torch.arange(blocks, device="cuda"), torch.tensor([best], device="cuda"))
        for n_split in (0, 1, 2):
            hk.mla8_dense_prefill(q, c, scales, out, 2, 0, kv_len=ints([n, n]), scale=scale, n_split=n_split, n_keys_hint=n)
            finish()
            off = (out.double() - want).abs()
            assert bool((off <= want.abs() * 2.0 ** -10 * 1.01 + 2.0 ** -25).all()), (best, n_split, float(off.max()))
