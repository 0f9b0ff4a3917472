"""The 8-bit paged latent cache (append, read, dense and sparse attention) and attention with a window and sinks, against 64 bits."""
import math

import pytest
import torch

import helios_glm53flash_b200 as hk
import latent8_ref as ref
from latent8_ref import STORE, attend, cache, check_append, rows_of, table_for, visible

pytestmark = pytest.mark.gpu


def gen_of(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def queries(gen, m, heads):
    return (torch.randn(m, heads, 512, device="cuda", generator=gen) * 0.7).half()


def close(out, want):
    """want: a list of (output, bound) per row"""
    for r, (o, tol) in enumerate(want):
        off = (out[r].double() - o).abs()
        assert bool((off <= tol).all()), "row %d: off %.3e of %.3e" % (r, float((off - tol).max()), float(tol.max()))


def finish():
    torch.cuda.synchronize()
    assert hk.read_device_status() == 0


def inputs(gen, n, dtype=torch.float32):
    x = torch.randn(n, 512, device="cuda", generator=gen) * torch.exp(torch.randn(n, 1, device="cuda", generator=gen))
    return x, (1.0 + 0.1 * torch.randn(512, device="cuda", generator=gen)).half()


# ---------------------------------------------------------------------------------------------
# append, read
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("pos,rows", [([0], [1]), ([0], [16]), ([7], [1]), ([13], [200]), ([128], [128]), ([127], [2]),
                                      ([0, 5, 130, 63], [1, 1, 1, 1]), ([3, 0, 40], [0, 300, 17])])
def test_append(kind, block, pos, rows):
    gen = gen_of(block + len(pos))
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    blocks = max((p + r - 1) // block + 1 for p, r in zip(pos, rows))
    n_blocks = blocks * len(pos) + 2
    ckv8, scales = cache(gen, kind, n_blocks, block)
    scales *= torch.exp(0.5 * torch.randn(n_blocks, device="cuda", generator=gen))       # some grow, some stay
    scales *= 0.02
    table = table_for(gen, len(pos), blocks, n_blocks)
    x, w = inputs(gen, starts[-1])
    old, old_s = ckv8.clone(), scales.clone()
    new = torch.full((starts[-1], 512), 7.0, dtype=torch.float16, device="cuda")
    kw = dict(seq_start=ints(starts)) if len(set(rows)) > 1 else {}
    hk.mla8_cache_append(x, w, ckv8, scales, ints(pos), starts[-1], ref.EPS, block_table=table, n_seqs=len(pos), ckv_new=new, **kw)
    finish()
    check_append(old, old_s, ckv8, scales, x, w, table.cpu(), pos, starts, kind, ckv_new=new)
    again, again_s = ckv8.clone(), scales.clone()
    hk.mla8_cache_append(x, w, ckv8, scales, ints(pos), starts[-1], ref.EPS, block_table=table, n_seqs=len(pos), **kw)
    finish()
    assert torch.equal(ckv8.view(torch.uint8), again.view(torch.uint8)) and torch.equal(scales, again_s), "the same rows again change nothing"


@pytest.mark.parametrize("kind,block,pos,rows", [("i8", 64, [37], [1000]), ("e4m3", 64, [50], [6000]), ("i8", 128, [100], [1500]), ("e4m3", 128, [77], [5000]),
                                                 ("i8", 128, [1], [19200]), ("i8", 128, [70, 0, 9], [30, 900, 0]), ("e4m3", 128, [33], [8000]), ("i8", 64, [5], [9000]), ("i8", 128, [17], [64]), ("e4m3", 64, [63, 33, 9], [2, 0, 700])])
def test_append_of_blocks_shared_out_over_ctas(kind, block, pos, rows):
    """blocks of 64 and 128 tokens by one CTA, two, four and eight; a row that is not finite makes its whole block NaN, whichever CTA has it"""
    gen = gen_of(sum(rows))
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    blocks = max((p + r - 1) // block + 1 for p, r in zip(pos, rows))
    n_blocks = blocks * len(pos)
    ckv8, scales = cache(gen, kind, n_blocks, block)
    scales *= 0.02 * torch.exp(0.5 * torch.randn(n_blocks, device="cuda", generator=gen))
    table = table_for(gen, len(pos), blocks, n_blocks)
    x, w = inputs(gen, starts[-1])
    x[starts[-1] - 3, 5] = math.inf
    old, old_s = ckv8.clone(), scales.clone()
    hk.mla8_cache_append(x, w, ckv8, scales, ints(pos), starts[-1], ref.EPS, block_table=table, n_seqs=len(pos), seq_start=ints(starts))
    finish()
    assert bool(scales.isnan().any())
    check_append(old, old_s, ckv8, scales, x, w, table.cpu(), pos, starts, kind)


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
def test_append_one_token_after_another_and_read(kind):
    """a block fills token by token: each step against the definition from the state before it; then everything read back"""
    gen, block, n = gen_of(5), 32, 75
    ckv8, scales = torch.zeros(4, block, 512, dtype=torch.int8, device="cuda").view(STORE[kind]), torch.full((4,), math.nan, device="cuda")
    scales[3] = 0.5
    table = ints([[2, 0, 1]])
    x, w = inputs(gen, n)
    roundings = torch.zeros(n, dtype=torch.float64, device="cuda")     # of each row so far
    for p in range(n):
        old, old_s = ckv8.clone(), scales.clone()
        hk.mla8_cache_append(x[p:p + 1], w, ckv8, scales, ints([p]), 1, ref.EPS, block_table=table)
        finish()
        if p % block == 0:
            old_s[table[0, p // block].item()] = 0.0             # a new block's old scale says nothing
        check_append(old, old_s, ckv8, scales, x[p:p + 1], w, table.cpu(), [p], [0, 1], kind)
        b = table[0, p // block].item()
        roundings[p // block * block:p] += float(scales[b] != old_s[b])
        roundings[p] = 1
    out = torch.full((n + 30, 512), 3.0, dtype=torch.float16, device="cuda")
    hk.mla8_cache_read(ckv8, scales, out, 0, n, block_table=table)
    finish()
    assert torch.equal(out[:n], rows_of(ckv8, scales, table[0], torch.arange(n, device="cuda")).half())
    assert (out[n:] == 3.0).all()
    # k roundings of a value: int8, half a step of a scale that only grows each time; e4m3, relative 2^-4 each time, or half the smallest step
    y, s, k = ref.normed(x, w), scales[table[0].long()].double().repeat_interleave(block)[:n, None], roundings[:, None]
    tol = k * s / 2 if kind == "i8" else y.abs() * ((1 + 2.0 ** -4) ** k - 1) + k * s * 2.0 ** -10
    assert bool(((out[:n].double() - y).abs() <= tol * (1 + 2.0 ** -10) + y.abs() * 2.0 ** -10).all())


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
def test_append_edges(kind):
    """sequences without a place: a negative position, positions behind the table, entries that name no block; rows of zeros; rows
    that are not finite"""
    gen, block = gen_of(9), 16
    ckv8, scales = cache(gen, kind, 8, block)
    old, old_s = ckv8.clone(), scales.clone()
    table = ints([[0, 1], [-1, 2], [3, 99], [4, 5]])
    x, w = inputs(gen, 4 * 20)
    x[60:80] = 0.0
    pos, starts = [-1, 10, 14, 3], [0, 20, 40, 60, 80]
    new = torch.full((80, 512), 7.0, dtype=torch.float16, device="cuda")
    hk.mla8_cache_append(x, w, ckv8, scales, ints(pos), 80, ref.EPS, block_table=table, n_seqs=4, ckv_new=new)
    finish()
    check_append(old, old_s, ckv8, scales, x, w, table.cpu(), pos, starts, kind)
    assert (new[:20] == 7).all() and (new[20:26] == 7).all() and (new[26:40] != 7).any() and (new[42:60] == 7).all()
    assert (ckv8[5].view(torch.uint8)[:7] == 0).all() and scales[5] == 0, "a new block of zero rows"
    assert torch.equal(ckv8[4].view(torch.uint8)[:3], old[4].view(torch.uint8)[:3]) and scales[4] == old_s[4]
    for bad in (math.nan, math.inf, -math.inf):
        x, w = inputs(gen, 3)
        x[1, 77] = bad
        hk.mla8_cache_append(x, w, ckv8, scales, ints([0]), 3, ref.EPS, block_table=table[:1].contiguous())
        finish()
        assert math.isnan(float(scales[0])) and torch.isfinite(scales[1:]).all()
        hk.mla8_cache_append(x[:1], w, ckv8, scales, ints([5]), 1, ref.EPS, block_table=table[:1].contiguous())
        finish()
        assert math.isnan(float(scales[0])), "stays one until the block is begun anew"
        hk.mla8_cache_append(x[:1], w, ckv8, scales, ints([0]), 1, ref.EPS, block_table=table[:1].contiguous())
        finish()
        assert math.isfinite(float(scales[0]))


def test_append_of_no_rows_touches_nothing():
    """a sequence of the batch without new rows, in the middle of a block"""
    gen = gen_of(21)
    ckv8, scales = cache(gen, "i8", 4, 16)
    old, old_s = ckv8.clone(), scales.clone()
    scales[1] = old_s[1] = math.nan
    x, w = inputs(gen, 5)
    hk.mla8_cache_append(x, w, ckv8, scales, ints([5, 3, 20]), 5, ref.EPS, block_table=ints([[0, 1], [2, 2], [3, 1]]), n_seqs=3, seq_start=ints([0, 0, 5, 5]))
    finish()
    keep = torch.tensor([0, 1, 3], device="cuda")
    assert torch.equal(ckv8[keep], old[keep]) and torch.equal(scales[0], old_s[0]) and torch.equal(scales[3], old_s[3]) and math.isnan(float(scales[1]))
    assert not torch.equal(ckv8[2], old[2])


def test_tensors_that_are_not_on_the_device_are_refused():
    ckv8, scales = cache(gen_of(1), "i8", 2, 16)
    out = torch.zeros(1, 64, 512, dtype=torch.float16, device="cuda")
    for c, s, t in ((ckv8.cpu(), scales, None), (ckv8, scales.cpu(), None), (ckv8, scales, torch.zeros(1, 2, dtype=torch.int32))):
        with pytest.raises(ValueError):
            hk.mla8_dense_prefill(out, c, s, out, 1, 0, block_table=t)


def test_tensors_of_another_type_layout_or_size_are_refused():
    """what the addresses that the library gets cannot tell: the wrappers look at the tensors"""
    gen = gen_of(12)
    ckv8, scales = cache(gen, "i8", 8, 16)
    table = ints([[0, 1, 2, 3], [4, 5, 6, 7]])
    x, w = inputs(gen, 2)
    q, out = queries(gen, 2, 64), torch.empty(2, 64, 512, dtype=torch.float16, device="cuda")
    ckv = torch.randn(64, 512, device="cuda", generator=gen).half()
    append = (hk.mla8_cache_append, dict(kv_pre=x, ln_w=w, ckv8=ckv8, scales=scales, pos=ints([3, 7]), n=2, eps=ref.EPS, block_table=table, n_seqs=2,
                                         seq_start=ints([0, 1, 2]), ckv_new=torch.empty(2, 512, dtype=torch.float16, device="cuda")))
    read = (hk.mla8_cache_read, dict(ckv8=ckv8, scales=scales, out=torch.empty(20, 512, dtype=torch.float16, device="cuda"), pos=3, n=20, block_table=table[0]))
    dense = (hk.mla8_dense_prefill, dict(q_lat=q, ckv8=ckv8, scales=scales, lat_out=out, qlen=2, pos_start=0, block_table=table, row_seq=ints([0, 1]), kv_len=ints([40, 50])))
    sparse = (hk.mla8_sparse_decode, dict(q_lat=q, ckv8=ckv8, scales=scales, raw_idx=ints([[1, 2, 3], [4, 5, 6]]), kidx=3, lat_out=out, m=2, block_table=table, row_seq=ints([0, 1])))
    window = (hk.mla_window_prefill, dict(q_lat=q, ckv=ckv, lat_out=out, qlen=2, pos_start=0, window=9, kv_base=torch.tensor([0, 5], device="cuda"), kv_len=ints([40, 50])))
    wide = lambda t: torch.stack((t, t), -1)[..., 0]           # every second element
    for fn, args in (append, read, dense, sparse, window):
        fn(**args)
        for name, t in args.items():
            if not torch.is_tensor(t):
                continue
            other = {torch.float32: torch.float16, torch.float16: torch.bfloat16, torch.int32: torch.int64, torch.int64: torch.int32}.get(t.dtype, torch.uint8)
            small = t if name in ("ckv", "block_table") else t.reshape(-1)[:-1]   # (a shorter table is a table, of fewer positions)
            for bad in (t.to(other), wide(t), t.cpu(), small):
                if bad is not t:
                    with pytest.raises(ValueError):
                        fn(**{**args, name: bad})
    finish()


def test_lengths_that_are_far_too_long_end_with_the_table():
    """garbage in a padding row's length: as many keys as the table has places, a window behind them sees the sinks alone"""
    gen = gen_of(22)
    ckv8, scales = cache(gen, "i8", 6, 32)
    table = table_for(gen, 2, 3, 6)
    q = queries(gen, 3, 64)
    out = torch.empty(3, 64, 512, dtype=torch.float16, device="cuda")
    lens = [2 ** 31 - 1, 50, 2 ** 30]
    for window, sinks, hint in ((0, 0, 100), (64, 7, 100), (64, 0, 1 << 20), (2 ** 31 - 1, 2 ** 31 - 1, 1 << 20)):
        hk.mla8_dense_prefill(q, ckv8, scales, out, 3, 0, block_table=table, row_seq=ints([0, 1, 0]), kv_len=ints(lens), window=window, sinks=sinks, n_keys_hint=hint)
        finish()
        want = []
        for r, n in enumerate(lens):
            p = torch.arange(min(n, 96), device="cuda")
            p = p[(p >= n - window) | (p < sinks)] if window else p
            want.append(attend(q[r].double(), rows_of(ckv8, scales, table[[0, 1, 0][r]], p), 0.0625))
        close(out, want)


def test_read_of_holes_and_without_a_table():
    gen = gen_of(3)
    ckv8, scales = cache(gen, "i8", 4, 16)
    out = torch.full((70, 512), 3.0, dtype=torch.float16, device="cuda")
    hk.mla8_cache_read(ckv8, scales, out, 10, 60, block_table=ints([2, -1, 7, 0]))
    finish()
    want = torch.zeros(60, 512, dtype=torch.float16, device="cuda")
    v = (ref.as_f64(ckv8) * scales.double()[:, None, None]).half()
    want[:6], want[38:54] = v[2, 10:], v[0]
    assert torch.equal(out[:60], want) and (out[60:] == 3).all()
    hk.mla8_cache_read(ckv8, scales, out, 0, 64)
    finish()
    assert torch.equal(out[:64], v.view(64, 512))


# ---------------------------------------------------------------------------------------------
# attention over the 8-bit cache
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind,block,heads,lens,window,sinks,n_split", [
    ("i8", 64, 64, [1], 0, 0, 0), ("i8", 16, 64, [63, 64, 65], 0, 0, 1), ("e4m3", 32, 64, [1000], 0, 0, 0), ("i8", 128, 64, [129, 1, 517], 0, 0, 3),
    ("e4m3", 16, 16, [300, 17, 0, 450], 0, 0, 0), ("i8", 64, 4, [700], 0, 0, 0), ("i8", 32, 128, [333, 90], 0, 0, 0), ("e4m3", 64, 100, [200], 0, 0, 2),
    ("i8", 16, 64, [900, 100, 64, 5], 100, 4, 0), ("e4m3", 64, 64, [2000], 1, 0, 0), ("i8", 64, 32, [2000, 130], 64, 64, 2),
    ("i8", 16, 64, [777], 129, 200, 1), ("e4m3", 128, 64, [1500, 1501], 1499, 1, 0), ("i8", 64, 64, [6000], 0, 0, 0)])
def test_dense8_rows(kind, block, heads, lens, window, sinks, n_split):
    """one query row a sequence, lengths on the device, pages anywhere"""
    gen = gen_of(sum(lens) + block)
    blocks = max(1, (max(lens) + block - 1) // block)
    ckv8, scales = cache(gen, kind, blocks * len(lens) + 3, block, spread=1.0)
    table = table_for(gen, len(lens), blocks, blocks * len(lens) + 3)
    m = len(lens)
    q = queries(gen, m, heads)
    out = torch.full((m + 1, heads, 512), 5.0, dtype=torch.float16, device="cuda")
    hk.mla8_dense_prefill(q, ckv8, scales, out, m, 0, n_heads=heads, block_table=table, row_seq=torch.arange(m, device="cuda", dtype=torch.int32),
                          kv_len=ints(lens), window=window, sinks=sinks, n_split=n_split, n_keys_hint=max(lens))
    finish()
    close(out, [attend(q[r].double(), rows_of(ckv8, scales, table[r], visible(n, window, sinks)), 0.0625) for r, n in enumerate(lens)])
    assert (out[m:] == 5.0).all()


def read_first(pos, rows, heads, window, sinks):
    """whether a chunk reads its positions as fp16 rows first"""
    keys = pos + rows
    if window:
        keys = 64 * min(-(-sinks // 64) + (window + 62) // 64 + 1, -(-keys // 64))
    return heads == 64 and rows >= 8 and rows * keys >= 65536


@pytest.mark.parametrize("kind,block,heads,pos,rows,window,sinks", [
    ("i8", 32, 64, 0, 300, 0, 0), ("e4m3", 64, 64, 9000, 9, 0, 0), ("i8", 16, 64, 2000, 200, 400, 70), ("e4m3", 128, 64, 3000, 150, 500, 0),
    ("i8", 64, 64, 1000, 300, 100, 700), ("i8", 64, 64, 4000, 40, 2500, 3),
    ("i8", 64, 64, 0, 2, 0, 0), ("i8", 64, 64, 0, 70, 0, 0), ("e4m3", 32, 64, 333, 40, 0, 0), ("i8", 16, 16, 100, 9, 0, 0), ("i8", 64, 64, 1000, 130, 0, 0),
    ("i8", 64, 64, 700, 90, 200, 4), ("e4m3", 128, 64, 10, 150, 64, 0), ("e4m3", 16, 64, 500, 80, 33, 130), ("i8", 32, 32, 50, 200, 1000, 7)])
def test_dense8_chunk(kind, block, heads, pos, rows, window, sinks):
    """a causal chunk of one sequence; blocks behind the sequence and spare blocks are NaN in scale"""
    gen = gen_of(pos + rows)
    blocks = (pos + rows + block - 1) // block
    ckv8, scales = cache(gen, kind, blocks + 4, block, spread=0.5)
    table = table_for(gen, 1, blocks + 1, blocks + 4)
    spare = torch.ones(blocks + 4, dtype=torch.bool, device="cuda")
    spare[table[0, :blocks].long()] = False
    scales[spare] = math.nan
    q = queries(gen, rows, heads)
    out = torch.full((rows + 1, heads, 512), 5.0, dtype=torch.float16, device="cuda")
    hk.mla8_dense_prefill(q, ckv8, scales, out, rows, pos, n_heads=heads, block_table=table, window=window, sinks=sinks)
    finish()
    rows16 = read_first(pos, rows, heads, window, sinks)
    close(out, [attend(q[r].double(), rows_of(ckv8, scales, table[0], visible(pos + r + 1, window, sinks)), 0.0625, rows16) for r in range(rows)])
    assert (out[rows:] == 5.0).all()


@pytest.mark.parametrize("rows", [10, 300])
def test_dense8_chunk_with_a_position_without_a_block_and_a_row_that_is_not_finite(rows):
    """short chunks read the cache as they go, long ones as fp16 rows first: an entry that names no block is 16 latents of zeros in both, and a
    scale that is NaN makes the outputs of the rows that see it NaN, under a window only of those that see it"""
    gen, pos = gen_of(rows), 100
    ckv8, scales = cache(gen, "i8", 30, 16)
    table = table_for(gen, 1, 26, 30)
    table[0, 2] = -1
    q = queries(gen, rows, 64)
    out = torch.empty(rows, 64, 512, dtype=torch.float16, device="cuda")
    hk.mla8_dense_prefill(q, ckv8, scales, out, rows, pos, block_table=table)
    finish()
    zero = torch.zeros(16, 512, dtype=torch.float64, device="cuda")
    want = []
    for r in range(rows):
        p = visible(pos + r + 1, 0, 0)
        keys = torch.cat((rows_of(ckv8, scales, table[0], p[:32]), zero, rows_of(ckv8, scales, table[0], p[48:])))
        want.append(attend(q[r].double(), keys, 0.0625, read_first(pos, rows, 64, 0, 0)))
    close(out, want)
    scales[table[0, 6]] = math.nan                            # positions 96 .. 111
    hk.mla8_dense_prefill(q, ckv8, scales, out, rows, pos, block_table=table)
    finish()
    assert torch.isnan(out).all()
    hk.mla8_dense_prefill(q, ckv8, scales, out, rows, pos, block_table=table, window=5, sinks=17 if rows < 300 else 90)
    finish()
    bad = torch.tensor([pos + r + 1 - 5 <= 111 for r in range(rows)], device="cuda")
    assert torch.isnan(out[bad]).all() and torch.isfinite(out[~bad]).all()


def test_dense8_without_a_table_and_another_scale():
    gen = gen_of(2)
    ckv8, scales = cache(gen, "i8", 9, 32)
    q = queries(gen, 3, 64)
    out = torch.empty(3, 64, 512, dtype=torch.float16, device="cuda")
    hk.mla8_dense_prefill(q, ckv8, scales, out, 3, 280, scale=512 ** -0.5)
    finish()
    ident = torch.arange(9, device="cuda", dtype=torch.int32)
    close(out, [attend(q[r].double(), rows_of(ckv8, scales, ident, visible(281 + r, 0, 0)), 512 ** -0.5) for r in range(3)])


def test_dense8_rows_and_blocks_that_do_not_count():
    """padding rows (a sequence number outside, a length of 0 or below), lengths behind the table, entries that name no block, blocks of
    zeros, and blocks that no row sees which are NaN"""
    gen, block = gen_of(4), 16
    ckv8, scales = cache(gen, "e4m3", 12, block, spread=2.0)
    ckv8[3] = 0.0
    scales[3] = 0.0
    ckv8[11] = math.nan
    scales[11] = math.nan
    table = ints([[0, 1, 2, 3], [4, -1, 12, 5], [11, 6, 7, 11]])
    seqs, lens = [0, -1, 1, 3, 2, 0, 1, 0], [64, 64, 64, 64, 48, 0, 500, -5]
    q = queries(gen, 8, 64)
    out = torch.full((8, 64, 512), 5.0, dtype=torch.float16, device="cuda")
    for splits in (0, 1, 4):
        hk.mla8_dense_prefill(q, ckv8, scales, out, 8, 0, block_table=table, row_seq=ints(seqs), kv_len=ints(lens), window=32, sinks=0, n_split=splits,
                              n_keys_hint=64)
        finish()
        want = []
        for r, (s, n) in enumerate(zip(seqs, lens)):
            p = visible(n, 32, 0) if 0 <= s < 3 else visible(0, 0, 0)
            want.append(attend(q[r].double(), rows_of(ckv8, scales, table[max(s, 0) % 3], p), 0.0625))
        close(out, want)
        assert (out[[1, 3, 5, 6, 7]] == 0).all()


@pytest.mark.parametrize("kind,heads,lens,window,sinks", [
    ("i8", 64, [3000, 700], 0, 0), ("e4m3", 64, [64, 5000, 1, 0, 2500, 129, 640], 0, 0), ("i8", 16, [100] * 40, 0, 0), ("i8", 100, [2000, 90, 1500], 0, 0),
    ("e4m3", 64, [4000, 4000, 100], 700, 65), ("i8", 64, [(37 * i) % 300 for i in range(148)], 0, 0), ("i8", 64, [9000] + [3] * 100, 0, 0),
    ("e4m3", 64, [0, 0, -4], 0, 0)])
def test_dense8_splits_shared_out_by_length(kind, heads, lens, window, sinks):
    """a hint of long rows: the splits are shared out on the device; one long row among short ones, empty ones, a row a CTA, sequences out of range"""
    gen, block, m = gen_of(len(lens) + heads), 64, len(lens)
    blocks = max(1, (max(lens) + block - 1) // block)
    ckv8, scales = cache(gen, kind, min(4000, blocks * m + 2), block, spread=1.0)
    table = torch.randint(0, ckv8.shape[0], (m, blocks), device="cuda", generator=gen, dtype=torch.int32)
    seqs = list(range(m))
    if m > 100:
        seqs[7], seqs[m - 1] = -1, m
    q = queries(gen, m, heads)
    for _ in range(2):                                         # the second time the workspace holds other partials
        out = torch.full((m + 1, heads, 512), 5.0, dtype=torch.float16, device="cuda")
        hk.mla8_dense_prefill(q, ckv8, scales, out, m, 0, n_heads=heads, block_table=table, row_seq=ints(seqs), kv_len=ints(lens), window=window,
                              sinks=sinks, n_keys_hint=1 << 20)
        finish()
        want = []
        for r, n in enumerate(lens):
            s = seqs[r]
            p = visible(n if 0 <= s < m else 0, window, sinks)
            want.append(attend(q[r].double(), rows_of(ckv8, scales, table[max(0, min(s, m - 1))], p), 0.0625))
        close(out, want)
        assert (out[m:] == 5.0).all()


def test_a_row_that_is_not_finite_is_seen_in_the_output():
    gen = gen_of(6)
    ckv8, scales = cache(gen, "i8", 4, 64)
    scales[2] = math.nan
    q = queries(gen, 1, 64)
    out = torch.zeros(1, 64, 512, dtype=torch.float16, device="cuda")
    for splits in (1, 2):
        hk.mla8_dense_prefill(q, ckv8, scales, out, 1, 255, n_split=splits)
        finish()
        assert torch.isnan(out).all()
        hk.mla8_dense_prefill(q, ckv8, scales, out, 1, 255, window=64, sinks=128, n_split=splits)
        finish()
        assert torch.isfinite(out).all()


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("m,n", [(1, 65), (1, 129), (1, 2049), (1, 5001), (1, 12033), (3, 2113), (4, 8193), (8, 9025), (40, 577), (200, 193)])
def test_splits_that_see_nothing_but_rows_that_are_not_finite(kind, m, n):
    """the last block, or two, of a row, which are the keys of a whole split for some of these lengths; and all blocks"""
    gen, block = gen_of(n), 64
    blocks = (n + block - 1) // block
    ckv8, scales = cache(gen, kind, blocks, block)
    table = table_for(gen, 1, blocks, blocks)
    q = queries(gen, m, 64)
    out = torch.zeros(m, 64, 512, dtype=torch.float16, device="cuda")
    gather = torch.arange(n, device="cuda", dtype=torch.int32).repeat(m, 1)
    for bad in (1, 2, blocks):
        scales[table[0, blocks - bad:].long()] = math.nan
        for n_split in (0, 2, 7):
            hk.mla8_dense_prefill(q, ckv8, scales, out.zero_(), m, 0, block_table=table, kv_len=ints([n] * m), n_keys_hint=n, n_split=n_split)
            finish()
            assert torch.isnan(out).all(), (bad, n_split)
            hk.mla8_sparse_decode(q, ckv8, scales, gather, n, out.zero_(), m, block_table=table, n_split=n_split)
            finish()
            assert torch.isnan(out).all(), (bad, n_split)
    hk.mla8_dense_prefill(q, ckv8, scales, out.zero_(), m, n, block_table=torch.cat((table, table, table, table, table), 1).contiguous())
    finish()
    assert torch.isnan(out).all()


@pytest.mark.parametrize("kind,block,heads,m,kidx,n_split", [("i8", 64, 64, 1, 2052, 0), ("e4m3", 16, 64, 3, 130, 0), ("i8", 128, 16, 2, 1, 1), ("i8", 32, 64, 5, 64, 2),
                                                             ("e4m3", 64, 64, 2, 700, 5), ("i8", 64, 64, 200, 70, 0)])
def test_sparse8(kind, block, heads, m, kidx, n_split):
    gen, n = gen_of(m + kidx), 3000
    blocks = (n + block - 1) // block
    ckv8, scales = cache(gen, kind, 2 * blocks + 1, block, spread=1.0)
    table = table_for(gen, 2, blocks, 2 * blocks + 1)
    seqs = [(i * 7) % 2 for i in range(m)]
    idx = torch.randint(0, n, (m, kidx), device="cuda", generator=gen, dtype=torch.int32)
    if kidx > 20:
        idx[:, 3::7] = -1
        idx[:, 4::50] = blocks * block + 5                      # behind the table
        idx[0, 10:20] = idx[0, 0]                               # the same position again counts again
        idx[m - 1, 64:] = -1
    q = queries(gen, m, heads)
    out = torch.full((m + 1, heads, 512), 5.0, dtype=torch.float16, device="cuda")
    hk.mla8_sparse_decode(q, ckv8, scales, idx, kidx, out, m, n_heads=heads, block_table=table, row_seq=ints(seqs), n_split=n_split)
    finish()
    close(out, [attend(q[r].double(), rows_of(ckv8, scales, table[seqs[r]], idx[r][idx[r] >= 0].long()), 0.0625) for r in range(m)])
    assert (out[m:] == 5.0).all()


@pytest.mark.parametrize("kind,block,m,kidx,blocks", [("i8", 32, 100, 480, 90), ("e4m3", 16, 300, 65, 25), ("i8", 128, 200, 513, 16), ("e4m3", 64, 130, 2052, 30)])
def test_sparse8_of_many_rows(kind, block, m, kidx, blocks):
    """rows that gather many keys of few positions: read as fp16 rows first; a block that is none, positions behind the table, a scale that is NaN"""
    gen, n = gen_of(m + kidx), blocks * block
    ckv8, scales = cache(gen, kind, blocks + 3, block, spread=0.5)
    table = table_for(gen, 1, blocks, blocks + 3)
    table[0, 3], table[0, 5] = -1, blocks + 3
    idx = torch.randint(0, n, (m, kidx), device="cuda", generator=gen, dtype=torch.int32)
    idx[:, 3::7] = -1
    idx[:, 4::50] = n + 5
    idx[1] = 3 * block + 1                                    # nothing but a block that is none
    q = queries(gen, m, 64)
    out = torch.full((m + 1, 64, 512), 5.0, dtype=torch.float16, device="cuda")
    hk.mla8_sparse_decode(q, ckv8, scales, idx, kidx, out, m, block_table=table)
    finish()
    close(out, [attend(q[r].double(), rows_of(ckv8, scales, table[0], idx[r][idx[r] >= 0].long()), 0.0625, rows16=True) for r in range(m)])
    assert (out[m:] == 5.0).all() and (out[1] == 0).all()
    scales[table[0, 0]] = math.nan
    hk.mla8_sparse_decode(q, ckv8, scales, idx, kidx, out, m, block_table=table)
    finish()
    hit = ((idx >= 0) & (idx < block)).any(1)
    assert torch.isnan(out[:m][hit]).all() and torch.isfinite(out[:m][~hit]).all()


# ---------------------------------------------------------------------------------------------
# window and sinks over the fp16 cache
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("heads,lens,window,sinks,n_split", [
    (64, [1], 1, 0, 0), (64, [64, 65, 200], 64, 0, 1), (64, [1000], 100, 4, 0), (64, [5000], 2000, 64, 0), (64, [900, 3, 0, 129], 128, 65, 0),
    (64, [700, 701], 1, 0, 3), (16, [500, 40], 33, 2, 0), (64, [3000], 10000, 10000, 0), (64, [257], 64, 1, 2), (64, [4000], 63, 3999, 0),
    (64, [5000, 4100, 300, 4999], 4090, 5, 0), (64, [3000, 2999, 2200, 40, 0, 2049, 2600, 2500], 2040, 3, 0)])
def test_window_rows(heads, lens, window, sinks, n_split):
    gen = gen_of(sum(lens) + window)
    base = [sum(lens[:i]) for i in range(len(lens))]
    ckv = torch.randn(sum(lens) + 1, 512, device="cuda", generator=gen).half()
    for b, n in zip(base, lens):                               # what no row sees
        hidden = torch.ones(n, dtype=torch.bool, device="cuda")
        hidden[visible(n, window, sinks)] = False
        ckv[b:b + n][hidden] = math.nan if n % 2 else math.inf
    m = len(lens)
    q = queries(gen, m, heads)
    out = torch.full((m + 1, heads, 512), 5.0, dtype=torch.float16, device="cuda")
    hk.mla_window_prefill(q, ckv, out, m, 0, window, sinks=sinks, n_heads=heads, kv_base=torch.tensor(base, device="cuda"), kv_len=ints(lens),
                          n_split=n_split, n_keys_hint=max(lens))
    finish()
    close(out, [attend(q[r].double(), ckv[base[r]:base[r] + n][visible(n, window, sinks)].double(), 0.0625) for r, n in enumerate(lens)])
    assert (out[m:] == 5.0).all()


@pytest.mark.parametrize("pos,rows,window,sinks", [(0, 1, 1, 0), (0, 130, 64, 0), (500, 65, 100, 3), (1000, 37, 1000, 64), (200, 300, 1, 1), (3000, 21, 900, 130),
                                                   (2000, 64, 1024, 4), (1500, 33, 1500, 0), (900, 150, 129, 0), (5000, 2, 4000, 10), (2047, 6, 1, 900), (3000, 7, 2, 701), (1000, 9, 64, 640),
                                                   (0, 1500, 800, 3), (2000, 301, 700, 0), (3000, 21, 2400, 130), (2500, 300, 2310, 70), (3000, 6, 1, 2500), (6000, 64, 4000, 0),
                                                   (2350, 150, 2333, 1)])
def test_window_chunk(pos, rows, window, sinks):
    """a causal chunk; each row's first hidden key and everything before it is infinite or NaN for that row alone or for all"""
    gen = gen_of(pos + rows)
    ckv = torch.randn(pos + rows, 512, device="cuda", generator=gen).half()
    lo = pos + 1 - window                                      # the first row's first key; the keys before it nobody sees
    if lo > sinks:
        ckv[sinks:lo] = math.nan
    q = queries(gen, rows, 64)
    out = torch.full((rows + 1, 64, 512), 5.0, dtype=torch.float16, device="cuda")
    hk.mla_window_prefill(q, ckv, out, rows, pos, window, sinks=sinks)
    finish()
    close(out, [attend(q[r].double(), ckv[:pos + r + 1][visible(pos + r + 1, window, sinks)].double(), 0.0625) for r in range(rows)])
    assert (out[rows:] == 5.0).all()


@pytest.mark.parametrize("rows,window", [(7, 1000), (8, 1000), (200, 1000), (7, 2500), (40, 2500)])      # single CTAs, a grid that walks rows, pairs of CTAs
def test_window_rows_do_not_take_over_what_their_neighbours_see(rows, window):
    """keys that leave the window one by one are infinite: the rows that still see one are not finite, the others are what they are without"""
    gen, pos, sinks = gen_of(rows), window + 200, 5
    ckv = torch.randn(pos + rows, 512, device="cuda", generator=gen).half()
    hot = pos + 1 - window + 3                                 # seen by rows 0 .. 3
    ckv[hot] = math.inf
    ckv[pos + rows - 1] = math.nan                             # the last row's own
    q = queries(gen, rows, 64)
    out = torch.empty(rows, 64, 512, dtype=torch.float16, device="cuda")
    hk.mla_window_prefill(q, ckv, out, rows, pos, window, sinks=sinks)
    finish()
    clean = [r for r in range(rows - 1) if r > 3]
    for r in clean:
        o, tol = attend(q[r].double(), ckv[:pos + r + 1][visible(pos + r + 1, window, sinks)].double(), 0.0625)
        assert bool(((out[r].double() - o).abs() <= tol).all()), r
    ckv[hot] = 1.0
    ckv[pos + rows - 1] = 1.0
    hk.mla_window_prefill(q, ckv, out, rows, pos, window, sinks=sinks)
    finish()
    close(out, [attend(q[r].double(), ckv[:pos + r + 1][visible(pos + r + 1, window, sinks)].double(), 0.0625) for r in range(rows)])


def test_window_cut_by_the_end_of_the_cache():
    """a length behind the cache's end: the window stands where the length says, rows that are not there are skipped"""
    gen = gen_of(8)
    ckv = torch.randn(1000, 512, device="cuda", generator=gen).half()
    q = queries(gen, 3, 64)
    out = torch.empty(3, 64, 512, dtype=torch.float16, device="cuda")
    hk.mla_window_prefill(q, ckv, out, 3, 0, 300, sinks=10, kv_base=torch.tensor([0, 200, 0], device="cuda"), kv_len=ints([1100, 900, 5000]), n_keys_hint=1000)
    finish()
    want = []
    for base, n in ((0, 1100), (200, 900), (0, 5000)):
        p = visible(n, 300, 10)
        want.append(attend(q[len(want)].double(), ckv[base + p[base + p < 1000]].double(), 0.0625))
    close(out, want)


# ---------------------------------------------------------------------------------------------
# together, as a server uses them
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["i8", "e4m3"])
def test_prefill_then_decode_of_three_sequences(kind):
    """chunks of three sequences into one pool of pages, then decode steps of all three: append, dense, windowed and sparse attention"""
    gen, block, prompts, steps = gen_of(11), 16, [100, 37, 64], 5
    blocks = 8
    ckv8 = torch.zeros(3 * blocks, block, 512, dtype=torch.int8, device="cuda").view(STORE[kind])
    scales = torch.zeros(3 * blocks, device="cuda")
    table = table_for(gen, 3, blocks, 3 * blocks)
    x, w = inputs(gen, sum(prompts))
    starts = [0, 100, 137, 201]
    held = torch.empty(sum(prompts), 512, dtype=torch.float16, device="cuda")
    hk.mla8_cache_append(x, w, ckv8, scales, ints([0, 0, 0]), sum(prompts), ref.EPS, block_table=table, n_seqs=3, seq_start=ints(starts), ckv_new=held)
    finish()
    for s in range(3):
        assert torch.equal(held[starts[s]:starts[s + 1]], rows_of(ckv8, scales, table[s], torch.arange(prompts[s], device="cuda")).half())
    lens = ints(prompts)
    row_seq = ints([0, 1, 2])
    outs = torch.empty(3, 3, 64, 512, dtype=torch.float16, device="cuda")
    for step in range(steps):
        x, w2 = inputs(gen, 3)
        before, before_s = ckv8.clone(), scales.clone()
        hk.mla8_cache_append(x, w, ckv8, scales, lens, 3, ref.EPS, block_table=table, n_seqs=3)
        pos = lens.tolist()
        lens = lens + 1
        q = queries(gen, 3, 64)
        idx = torch.stack([torch.randint(0, n + 1, (40,), device="cuda", generator=gen) for n in pos]).int().contiguous()
        args = dict(block_table=table, row_seq=row_seq)
        hk.mla8_dense_prefill(q, ckv8, scales, outs[0], 3, 0, kv_len=lens, n_keys_hint=128, **args)
        hk.mla8_dense_prefill(q, ckv8, scales, outs[1], 3, 0, kv_len=lens, n_keys_hint=128, window=20, sinks=2, **args)
        hk.mla8_sparse_decode(q, ckv8, scales, idx, 40, outs[2], 3, **args)
        finish()
        check_append(before, before_s, ckv8, scales, x, w, table.cpu(), pos, [0, 1, 2, 3], kind)
        for s, n in enumerate(pos):
            for k, p in enumerate((visible(n + 1, 0, 0), visible(n + 1, 20, 2), idx[s].long())):
                o, tol = attend(q[s].double(), rows_of(ckv8, scales, table[s], p), 0.0625)
                assert bool(((outs[k, s].double() - o).abs() <= tol).all())


def test_two_streams_at_once():
    """two sequences' steps side by side, workspaces and caches of their own"""
    gen, block = gen_of(31), 64
    sides = [torch.cuda.Stream() for _ in range(2)]
    states = []
    for _ in sides:
        ckv8, scales = cache(gen, "i8", 40, block)
        states.append((ckv8, scales, queries(gen, 1, 64), torch.empty(1, 64, 512, dtype=torch.float16, device="cuda"), torch.randn(300, 512, device="cuda", generator=gen).half()))
    torch.cuda.synchronize()
    for _ in range(5):
        for stream, (ckv8, scales, q, out, ckv) in zip(sides, states):
            with torch.cuda.stream(stream):
                hk.mla8_dense_prefill(q, ckv8, scales, out, 1, 2499)
                hk.mla_window_prefill(q, ckv, out[:], 1, 299, 100, sinks=3)
                hk.mla8_dense_prefill(q, ckv8, scales, out, 1, 2499)
    finish()
    ident = torch.arange(40, device="cuda", dtype=torch.int32)
    for ckv8, scales, q, out, ckv in states:
        close(out, [attend(q[0].double(), rows_of(ckv8, scales, ident, visible(2500, 0, 0)), 0.0625)])


def test_captured_decode_step_replayed():
    """append and attention in one graph, positions and lengths on the device; the same bits as the calls, also on another stream"""
    gen, block = gen_of(13), 64
    ckv8, scales = cache(gen, "i8", 8, block)
    table = ints([[5, 1], [0, 7]])
    x, w = inputs(gen, 2)
    q = queries(gen, 2, 64)
    pos, lens, row_seq = ints([70, 13]), ints([71, 14]), ints([0, 1])
    ws = torch.empty(max(256, hk.mla8_dense_workspace_bytes(2, 64, 0, 128, per_row=True)), dtype=torch.uint8, device="cuda")

    def step(out, c, s, stream=None):
        hk.mla8_cache_append(x, w, c, s, pos, 2, ref.EPS, block_table=table, n_seqs=2, stream=stream)
        hk.mla8_dense_prefill(q, c, s, out, 2, 0, block_table=table, row_seq=row_seq, kv_len=lens, n_keys_hint=128, workspace=ws, stream=stream)

    c2, s2 = ckv8.clone(), scales.clone()
    out = torch.empty(2, 64, 512, dtype=torch.float16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(out, ckv8, scales)
    want = torch.empty_like(out)
    for k in range(3):
        x.copy_(inputs(gen, 2)[0])
        q.copy_(queries(gen, 2, 64))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        step(want, c2, s2, stream=side if k == 1 else None)
        finish()
        assert torch.equal(out, want) and torch.equal(ckv8, c2) and torch.equal(scales, s2)
        pos += 1
        lens += 1


def test_the_widest_window():
    """a window of all 31 bits with lengths on the device and none given to choose the splits by"""
    gen = gen_of(77)
    ckv, q = torch.randn(700, 512, device="cuda", generator=gen).half(), queries(gen, 3, 64)
    ckv8, scales = cache(gen, "i8", 11, 64)
    out = torch.empty(3, 64, 512, dtype=torch.float16, device="cuda")
    for sinks in (0, 5, 2 ** 31 - 1):
        hk.mla_window_prefill(q, ckv, out, 3, 0, 2 ** 31 - 1, sinks=sinks, kv_len=ints([700, 0, 65]))
        finish()
        close(out, [attend(q[r].double(), ckv[:n].double(), 0.0625) for r, n in enumerate([700, 0, 65])])
        hk.mla8_dense_prefill(q, ckv8, scales, out, 3, 0, window=2 ** 31 - 1, sinks=sinks, kv_len=ints([700, 0, 65]))
        finish()
        close(out, [attend(q[r].double(), rows_of(ckv8, scales, torch.arange(11), torch.arange(n)), 0.0625) for r, n in enumerate([700, 0, 65])])


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
def test_blocks_beyond_four_gigabytes(kind):
    """blocks at the end of a cache of 9.6 million latents, through a table and by their positions; an fp16 cache of 5 million likewise"""
    gen, block, n_blocks, n = gen_of(88), 64, 150000, 1000
    ckv8, scales = torch.empty(n_blocks, block, 512, dtype=torch.int8, device="cuda").view(STORE[kind]), torch.full((n_blocks,), math.nan, device="cuda")
    table = (n_blocks - 1 - torch.randperm(16, device="cuda", generator=gen)).to(torch.int32)[None].contiguous()
    x, w = inputs(gen, n)
    held, out = torch.empty(n, 512, dtype=torch.float16, device="cuda"), torch.empty(n, 512, dtype=torch.float16, device="cuda")
    hk.mla8_cache_append(x, w, ckv8, scales, ints([0]), n, ref.EPS, block_table=table, ckv_new=held)
    hk.mla8_cache_read(ckv8, scales, out, 0, n, block_table=table)
    finish()
    assert bool(torch.isfinite(held).all()) and torch.equal(held, out)
    q, o = queries(gen, 2, 64), torch.empty(2, 64, 512, dtype=torch.float16, device="cuda")
    keys = rows_of(ckv8, scales, table[0], torch.arange(n, device="cuda"))
    idx = torch.randint(0, n, (2, 300), device="cuda", generator=gen, dtype=torch.int32)
    hk.mla8_dense_prefill(q, ckv8, scales, o, 2, 0, block_table=table, kv_len=ints([n, n - 7]))
    finish()
    close(o, [attend(q[r].double(), keys[:n - 7 * r], 0.0625) for r in range(2)])
    hk.mla8_sparse_decode(q, ckv8, scales, idx, 300, o, 2, block_table=table)
    finish()
    close(o, [attend(q[r].double(), keys[idx[r].long()], 0.0625) for r in range(2)])
    # by position, without a table: the last 16 blocks in order
    far = (n_blocks - 16) * block
    order = torch.arange(n_blocks - 16, n_blocks, device="cuda", dtype=torch.int32)
    hk.mla8_cache_append(x, w, ckv8, scales, ints([far]), n, ref.EPS, ckv_new=held)
    hk.mla8_cache_read(ckv8, scales, out, far, n)
    finish()
    assert bool(torch.isfinite(held).all()) and torch.equal(held, out)
    keys = rows_of(ckv8, scales, order, torch.arange(n, device="cuda"))
    hk.mla8_dense_prefill(q, ckv8, scales, o, 2, 0, kv_len=ints([far + n, far + 900]), window=500, n_keys_hint=far + n)
    finish()
    close(o, [attend(q[0].double(), keys[n - 500:], 0.0625), attend(q[1].double(), keys[400:900], 0.0625)])
    hk.mla8_dense_prefill(q, ckv8, scales, o, 2, far + n - 2, window=500)
    finish()
    close(o, [attend(q[r].double(), keys[n - 501 + r:n - 1 + r], 0.0625) for r in range(2)])
    hk.mla8_sparse_decode(q, ckv8, scales, idx + far, 300, o, 2)
    finish()
    close(o, [attend(q[r].double(), keys[idx[r].long()], 0.0625) for r in range(2)])


def test_windows_beyond_four_gigabytes():
    gen, rows, n = gen_of(89), 5000000, 1000
    ckv, q, o = torch.empty(rows, 512, dtype=torch.float16, device="cuda"), queries(gen, 2, 64), torch.empty(2, 64, 512, dtype=torch.float16, device="cuda")
    ckv[rows - n:] = torch.randn(n, 512, device="cuda", generator=gen).half()
    ckv[:100] = torch.randn(100, 512, device="cuda", generator=gen).half()
    hk.mla_window_prefill(q, ckv, o, 2, 0, 300, sinks=70, kv_base=torch.tensor([rows - n, 0], device="cuda"), kv_len=ints([n, rows]), n_keys_hint=rows)
    finish()
    close(o, [attend(q[0].double(), torch.cat((ckv[rows - n:rows - n + 70], ckv[rows - 300:])).double(), 0.0625),
              attend(q[1].double(), torch.cat((ckv[:70], ckv[rows - 300:])).double(), 0.0625)])
    hk.mla_window_prefill(q, ckv, o, 2, rows - 2, 300, sinks=70)
    finish()
    close(o, [attend(q[r].double(), torch.cat((ckv[:70], ckv[rows - 301 + r:rows - 1 + r])).double(), 0.0625) for r in range(2)])


def test_scratch_follows_its_tensor_and_is_never_empty():
    t = torch.zeros(3, device="cuda")
    for asked in (0, 1, 1000):
        ws = hk._native.scratch(asked, t)
        assert ws.dtype == torch.uint8 and ws.device == t.device and ws.numel() == max(asked, 256)
    for bad in [(), (5,), (5, 7), ("5", t)]:
        with pytest.raises((TypeError, ValueError)):
            hk._native.scratch(*bad)
