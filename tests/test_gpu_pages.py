"""Pages of the 8-bit latent cache: fork, reserve, free, compact and copy against a model of them in whole numbers, block by block."""
import random

import pytest
import torch

import helios_glm53flash_b200 as hk
from latent8_ref import STORE

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def finish():
    torch.cuda.synchronize()
    assert hk.read_device_status() == 0


class Pool:
    """the device's pool and what it should be; every block has contents and a scale of its own"""

    def __init__(self, kind, n_blocks, block, n_seqs, stride):
        gen = torch.Generator(device="cuda").manual_seed(n_blocks)
        self.block, self.n = block, n_blocks
        self.ckv8 = torch.randint(0, 120, (n_blocks, block, 512), device="cuda", generator=gen, dtype=torch.uint8).view(STORE[kind])
        self.scales = torch.arange(n_blocks, device="cuda") + 0.5
        self.refs = torch.zeros(n_blocks, dtype=torch.int32, device="cuda")
        self.table = torch.full((n_seqs, stride), -1, dtype=torch.int32, device="cuda")
        self.first = self.ckv8.view(torch.uint8).clone()
        self.rows, self.count, self.holds = [[-1] * stride for _ in range(n_seqs)], [0] * n_blocks, list(range(n_blocks))
        self.told = ints([-5])
        self.tensors = (self.ckv8, self.scales, self.refs, self.table)

    def real(self, e):
        return 0 <= e < self.n

    def entries(self, length):
        return min((max(length, 0) + self.block - 1) // self.block, len(self.rows[0]))

    def release(self, s, first=0):
        for j in range(first, len(self.rows[s])):
            if self.rows[s][j] >= 0:
                if self.real(self.rows[s][j]):
                    self.count[self.rows[s][j]] -= 1
                self.rows[s][j] = -1

    def take(self):
        for b in range(self.n):
            if self.count[b] == 0:
                self.count[b] = 1
                return b
        return -1

    def ok(self, s):
        return 0 <= s < len(self.rows)

    def fork(self, pairs):
        hk.mla8_pages_fork(*self.tensors, ints([p for p, _, _ in pairs]), ints([c for _, c, _ in pairs]), ints([n for _, _, n in pairs]), len(pairs), missing=self.told)
        pairs = [x for x in pairs if self.ok(x[0]) and self.ok(x[1]) and x[0] != x[1]]
        missing = 0
        for _, c, _ in pairs:
            self.release(c)
        for p, c, n in pairs:
            for j in range(min(max(n, 0) // self.block, len(self.rows[0]))):
                if self.real(self.rows[p][j]):
                    self.rows[c][j] = self.rows[p][j]
                    self.count[self.rows[p][j]] += 1
        for p, c, n in pairs:
            j = max(n, 0) // self.block
            if n > 0 and n % self.block and j < len(self.rows[0]) and self.real(self.rows[p][j]):
                b = self.take()
                missing += b < 0
                if b >= 0:
                    self.rows[c][j] = b
                    self.holds[b] = self.holds[self.rows[p][j]]
        self.check(missing)

    def reserve(self, wants):
        hk.mla8_pages_reserve(*self.tensors, ints([s for s, _ in wants]), ints([n for _, n in wants]), len(wants), missing=self.told)
        missing = 0
        for s, n in wants:
            for j in range(self.entries(n) if self.ok(s) else 0):
                if not self.real(self.rows[s][j]):
                    b = self.take()
                    missing += b < 0
                    if b >= 0:
                        self.rows[s][j] = b
        self.check(missing)

    def free(self, keeps):
        hk.mla8_pages_free(*self.tensors, ints([s for s, _ in keeps]), ints([n for _, n in keeps]), len(keeps))
        for s, n in keeps:
            if self.ok(s):
                self.release(s, self.entries(n))
        self.check()

    def compact(self):
        hk.mla8_pages_compact(*self.tensors, n_live=self.told)
        live = sum(c != 0 for c in self.count)
        holes = [b for b in range(live) if self.count[b] == 0]
        goes = {}
        for src, dst in zip([b for b in range(live, self.n) if self.count[b]], holes):
            goes[src] = dst
            self.holds[dst] = self.holds[src]
            self.count[dst], self.count[src] = self.count[src], 0
        self.rows = [[goes.get(e, e) for e in row] for row in self.rows]
        self.check(live)

    def check(self, told=None):
        finish()
        assert self.table.tolist() == self.rows
        assert self.refs.tolist() == self.count
        at = torch.tensor(self.holds, device="cuda")
        assert torch.equal(self.ckv8.view(torch.uint8), self.first[at]) and torch.equal(self.scales, at + 0.5)
        if told is not None:
            assert int(self.told) == told


@pytest.mark.parametrize("n_blocks,block,n_seqs,stride", [(1, 16, 3, 2), (7, 128, 4, 3), (31, 16, 5, 9), (33, 64, 9, 40), (600, 32, 40, 33), (1024, 16, 20, 40), (300, 16, 60, 100), (1500, 128, 90, 70), (8192, 16, 60, 150), (9000, 16, 70, 150)])
def test_pages_come_and_go(n_blocks, block, n_seqs, stride):
    pool = Pool("i8" if block < 64 else "e4m3", n_blocks, block, n_seqs, stride)
    rng = random.Random(n_blocks)
    some = lambda: rng.sample(range(n_seqs), rng.randint(1, n_seqs))  # noqa: E731
    length = lambda: rng.choice([0, 1, block - 1, block, block + 1, rng.randint(0, block * stride), block * stride, block * stride + 5])  # noqa: E731
    pool.reserve([(s, length()) for s in some()])
    for turn in range(14):
        what = turn % 4
        if what == 0:
            seqs = rng.sample(range(n_seqs), n_seqs)
            parents, children = seqs[:max(1, n_seqs // 3)], seqs[max(1, n_seqs // 3):]
            pool.fork([(rng.choice(parents), c, length()) for c in children])
        elif what == 1:
            pool.free([(s, rng.choice([0, 0, length()])) for s in some()])
        elif what == 2:
            pool.compact()
        else:
            pool.reserve([(s, length()) for s in some()])


@pytest.mark.parametrize("n_blocks,block,n_seqs,stride", [(700, 16, 12, 4096), (90, 64, 4, 16384), (9000, 16, 10, 2049)])
def test_tables_that_are_wider_than_what_is_held(n_blocks, block, n_seqs, stride):
    """room for long contexts, of which the sequences use a part; once a sequence takes more than there is"""
    pool = Pool("i8", n_blocks, block, n_seqs, stride)
    rng = random.Random(stride)
    some = lambda: rng.sample(range(n_seqs), rng.randint(1, n_seqs))  # noqa: E731
    length = lambda: rng.choice([0, 1, block, block * 5 + 1, rng.randint(0, block * 40)])  # noqa: E731
    pool.reserve([(s, length()) for s in range(n_seqs)])
    for turn in range(2):
        pool.fork([(rng.choice([0, 1]), s, length()) for s in range(2, n_seqs)])
        pool.free([(s, rng.choice([0, length()])) for s in some()])
        pool.compact()
        pool.reserve([(s, length()) for s in some()])
    pool.free([(0, 0)])
    pool.reserve([(0, min(block * stride, block * (n_blocks + 3)))])
    pool.fork([(0, 1, block * stride - 1)])
    pool.compact()


def test_what_names_no_sequence_and_no_block_is_passed_over():
    pool = Pool("i8", 40, 16, 6, 8)
    pool.reserve([(0, 50), (-1, 100), (6, 100), (1, 100), (1 << 30, 7), (2, -3)])
    pool.fork([(0, 3, 50), (-1, 4, 20), (1, 9, 20), (1, 4, 100), (2, 2, 30), (2, 5, 30)])
    pool.table[1, 2] = pool.rows[1][2] = 1000                 # entries that name no block
    pool.table[1, 3] = pool.rows[1][3] = -9
    pool.count[pool.table[4, 2]] -= 1                         # whose references are the test's to keep
    pool.refs[pool.table[4, 2]] -= 1
    pool.count[pool.table[4, 3]] -= 1
    pool.refs[pool.table[4, 3]] -= 1
    pool.fork([(1, 5, 60), (1, 2, 40)])
    pool.free([(7, 0), (-2, 0)])
    pool.reserve([(1, 128)])
    pool.compact()


def test_a_full_pool_gives_what_it_has():
    pool = Pool("e4m3", 10, 32, 4, 8)
    pool.reserve([(0, 8 * 32), (1, 3 * 32), (2, 32)])         # 12 wanted, 10 there
    pool.fork([(0, 3, 100)])                                  # the last block of 4 tokens cannot be copied
    pool.free([(1, 0)])
    pool.fork([(0, 3, 100), (0, 2, 33), (0, 1, 31)])


def test_the_same_sequence_twice_is_given_back_once():
    pool = Pool("i8", 30, 16, 3, 6)
    pool.reserve([(0, 96), (1, 50)])
    hk.mla8_pages_free(*pool.tensors, ints([0, 0, 0]), None, 3)
    pool.release(0)
    pool.check()


def test_calls_without_sequences_tell_that_nothing_is_missing():
    pool = Pool("i8", 30, 16, 3, 6)
    pool.reserve([(0, 40)])
    none = ints([])
    hk.mla8_pages_fork(*pool.tensors, none, none, none, 0)
    hk.mla8_pages_free(*pool.tensors, none, None, 0)
    hk.mla8_pages_copy(*pool.tensors[:2], *pool.tensors[:2], none, none, 0)
    for call in (lambda told: hk.mla8_pages_fork(*pool.tensors, none, none, none, 0, missing=told),
                 lambda told: hk.mla8_pages_reserve(*pool.tensors, none, none, 0, missing=told)):
        told = ints([7])
        call(told)
        assert int(told) == 0
    pool.check()


def test_long_pools_and_offsets_beyond_four_gigabytes():
    """blocks beyond 2^32 bytes of the cache: fork copies one there, compaction brings it back"""
    n, block = (1 << 32) // (128 * 512) + 40, 128
    ckv8 = torch.empty(n, block, 512, dtype=torch.int8, device="cuda")
    scales, refs = torch.zeros(n, device="cuda"), torch.ones(n, dtype=torch.int32, device="cuda")
    table = ints([[n - 3, n - 20, -1], [-1, -1, -1], [0, 5, 9]])
    refs[n - 7], refs[3] = 0, 0
    refs[10:n - 21] = 0
    refs[10] = 0
    for b in (n - 3, n - 20, 0, 5, 9):
        ckv8[b].random_(-127, 127)
        scales[b] = b
    held = [ckv8[n - 3].clone(), ckv8[n - 20].clone()]
    refs[12:n - 25] = 1                                       # all but the last gap
    refs[n - 25:n - 21] = 0
    refs[3] = 1
    refs[10:12] = 1
    hk.mla8_pages_fork(ckv8, scales, refs, table, ints([0]), ints([1]), ints([200]), 1)
    finish()
    assert table[1].tolist() == [n - 3, n - 25, -1] and torch.equal(ckv8[n - 25], held[1]) and float(scales[n - 25]) == n - 20
    refs.zero_()
    refs[[n - 3, n - 20, n - 25, 0, 5, 9]] = ints([2, 1, 1, 1, 1, 1])
    live = ints([0])
    hk.mla8_pages_compact(ckv8, scales, refs, table, n_live=live)
    finish()
    assert int(live) == 6 and refs.nonzero().flatten().tolist() == [0, 1, 2, 3, 4, 5]
    assert table.tolist() == [[4, 3, -1], [4, 2, -1], [0, 5, 1]] and torch.equal(ckv8[4], held[0]) and torch.equal(ckv8[2], held[1]) and torch.equal(ckv8[3], held[1])


@pytest.mark.parametrize("kind,block", [("i8", 16), ("e4m3", 128)])
def test_copies_between_pools(kind, block):
    a, b = Pool(kind, 20, block, 1, 1), Pool(kind, 9, block, 1, 1)
    b.ckv8.view(torch.uint8).add_(1)
    want, want_s = b.ckv8.view(torch.uint8).clone(), b.scales.clone()
    src, dst = [3, 19, -1, 5, 20, 7, 0], [8, 0, 2, 9, 3, -4, 1]
    for x, y in zip(src, dst):
        if 0 <= x < 20 and 0 <= y < 9:
            want[y], want_s[y] = a.first[x], x + 0.5
    hk.mla8_pages_copy(a.ckv8, a.scales, b.ckv8, b.scales, ints(src), ints(dst), len(src))
    finish()
    assert torch.equal(b.ckv8.view(torch.uint8), want) and torch.equal(b.scales, want_s)
    with pytest.raises(ValueError):
        hk.mla8_pages_copy(a.ckv8, a.scales, Pool(kind, 9, 32, 1, 1).ckv8, b.scales, ints(src), ints(dst), len(src))


def test_a_captured_turn_of_calls_follows_the_device():
    """fork, free, compact and reserve under one graph, replayed on other sequences and lengths"""
    kinds = [Pool("i8", 60, 16, 6, 7) for _ in range(2)]
    pool = kinds[0]
    pool.reserve([(0, 100), (1, 60), (2, 33), (3, 112)])
    par, chi, lens, gone, want = ints([0, 1]), ints([4, 5]), ints([90, 50]), ints([2]), ints([40])
    ws = torch.empty(hk.mla8_pages_workspace_bytes(60, 2), dtype=torch.uint8, device="cuda")

    def turn():
        hk.mla8_pages_fork(*pool.tensors, par, chi, lens, 2, workspace=ws)
        hk.mla8_pages_free(*pool.tensors, gone, None, 1)
        hk.mla8_pages_compact(*pool.tensors, workspace=ws)
        hk.mla8_pages_reserve(*pool.tensors, gone, want, 1, workspace=ws)

    def model(pairs, s, n):
        tensors = [t.clone() for t in pool.tensors]
        graph.replay()
        finish()
        after = [t.clone() for t in pool.tensors]
        for t, x in zip(pool.tensors, tensors):
            t.copy_(x)
        pool.fork(pairs)
        pool.free([(s, 0)])
        pool.compact()
        pool.reserve([(s, n)])
        for t, x in zip(pool.tensors, after):
            assert torch.equal(t.view(torch.uint8) if t.element_size() == 1 else t, x.view(torch.uint8) if x.element_size() == 1 else x)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        turn()
    model([(0, 4, 90), (1, 5, 50)], 2, 40)
    par.copy_(ints([3, 3]))
    chi.copy_(ints([1, 0]))
    lens.copy_(ints([112, 7]))
    gone.copy_(ints([5]))
    want.copy_(ints([112]))
    model([(3, 1, 112), (3, 0, 7)], 5, 112)


def same(pool, other):
    return all(torch.equal(a.view(torch.uint8) if a.element_size() == 1 else a, b.view(torch.uint8) if b.element_size() == 1 else b) for a, b in zip(pool.tensors, other.tensors))


def test_a_captured_turn_with_scratch_of_its_own():
    """the calls take and give back their scratch inside the capture, where other tensors are made and let go too"""
    pool, other = Pool("e4m3", 60, 16, 6, 7), Pool("e4m3", 60, 16, 6, 7)
    for p in (pool, other):
        p.reserve([(0, 100), (1, 60), (2, 33), (3, 112)])
    par, chi, lens, gone, want = ints([0, 1]), ints([4, 5]), ints([90, 50]), ints([2]), ints([40])
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        hk.mla8_pages_fork(*pool.tensors, par, chi, lens, 2)
        kept = torch.full((5000,), 5, dtype=torch.int32, device="cuda")
        hk.mla8_pages_free(*pool.tensors, gone, None, 1)
        torch.full((300,), 9, dtype=torch.int32, device="cuda")
        hk.mla8_pages_compact(*pool.tensors)
        last = torch.full((300,), 7, dtype=torch.int32, device="cuda")
        hk.mla8_pages_reserve(*pool.tensors, gone, want, 1)
    for pairs, s, n in (([(0, 4, 90), (1, 5, 50)], 2, 40), ([(3, 1, 112), (3, 0, 7)], 5, 112), ([(1, 2, 17), (4, 3, 90)], 0, 1)):
        for t, v in ((par, [x[0] for x in pairs]), (chi, [x[1] for x in pairs]), (lens, [x[2] for x in pairs]), (gone, [s]), (want, [n])):
            t.copy_(ints(v))
        graph.replay()
        finish()
        other.fork(pairs)
        other.free([(s, 0)])
        other.compact()
        other.reserve([(s, n)])
        assert same(pool, other) and bool((kept == 5).all()) and bool((last == 7).all())


@pytest.mark.parametrize("given", [True, False])
def test_two_pools_on_two_streams_at_once(given):
    """given: the stream as an argument, else the current one; scratch of the calls is each stream's own"""
    pools = [Pool("i8", 3000, 16, 40, 60), Pool("e4m3", 900, 32, 30, 40)]
    others = [Pool("i8", 3000, 16, 40, 60), Pool("e4m3", 900, 32, 30, 40)]
    rng, turns = random.Random(5), []
    for p in others:
        turns.append([])
        n_seqs, room = len(p.rows), p.block * len(p.rows[0])
        lens = [rng.randint(0, room) for _ in range(n_seqs)]
        turns[-1].append(("reserve", [(s, n) for s, n in enumerate(lens)]))
        for _ in range(4):
            seqs = rng.sample(range(n_seqs), n_seqs)
            turns[-1].append(("fork", [(seqs[i % 5], c, rng.randint(0, room)) for i, c in enumerate(seqs[5:20])]))
            turns[-1].append(("free", [(s, rng.choice([0, rng.randint(0, room)])) for s in seqs[:12]]))
            turns[-1].append(("compact",))
            turns[-1].append(("reserve", [(s, rng.randint(0, room)) for s in seqs[::2]]))
    lists = [[[ints([x[i] for x in t[1]]) for i in range(len(t[1][0]))] if len(t) > 1 else None for t in ts] for ts in turns]
    sides = [torch.cuda.Stream() for _ in range(2)]
    finish()
    calls = dict(fork=hk.mla8_pages_fork, free=hk.mla8_pages_free, reserve=hk.mla8_pages_reserve, compact=hk.mla8_pages_compact)
    for step in range(len(turns[0])):
        for p, ts, ls, side in zip(pools, turns, lists, sides):
            args = p.tensors + ((*ls[step], len(ts[step][1])) if ls[step] else ())
            if given:
                calls[ts[step][0]](*args, stream=side)
            else:
                with torch.cuda.stream(side):
                    calls[ts[step][0]](*args)
    finish()
    for p, ts in zip(others, turns):
        for what, *rest in ts:
            getattr(p, what)(*rest)
    assert same(pools[0], others[0]) and same(pools[1], others[1])


def test_samples_of_one_prompt_append_and_attend_on_their_own():
    """reserve, append a prompt, fork it, append to each sample, attend: a sample sees the prompt and its own tokens, the prompt stays as it is"""
    gen = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    block, n, prompt = 16, 40, 37
    ckv8 = torch.zeros(n, block, 512, dtype=torch.int8, device="cuda")
    scales, refs = torch.zeros(n, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
    table = torch.full((4, 6), -1, dtype=torch.int32, device="cuda")
    pool, ln_w = (ckv8, scales, refs, table), torch.ones(512, dtype=torch.float16, device="cuda")
    hk.mla8_pages_reserve(*pool, ints([0]), ints([prompt]), 1)
    hk.mla8_cache_append(rand(prompt, 512), ln_w, ckv8, scales, ints([0, -1, -1, -1]), prompt, 1e-6, block_table=table, n_seqs=4, seq_start=ints([0, prompt, prompt, prompt, prompt]))
    read = lambda s, k: (hk.mla8_cache_read(ckv8, scales, o := torch.empty(k, 512, dtype=torch.float16, device="cuda"), 0, k, block_table=table[s:s + 1].contiguous()), o)[1]  # noqa: E731
    first = read(0, prompt)
    hk.mla8_pages_fork(*pool, ints([0, 0, 0]), ints([1, 2, 3]), ints([prompt] * 3), 3)
    lens = [prompt, prompt + 1, prompt + 11, prompt + 30]
    hk.mla8_pages_reserve(*pool, ints([1, 2, 3]), ints(lens[1:]), 3)
    hk.mla8_cache_append(rand(42, 512), ln_w, ckv8, scales, ints([-1, prompt, prompt, prompt]), 42, 1e-6, block_table=table, n_seqs=4, seq_start=ints([0, 0, 1, 12, 42]))
    finish()
    assert torch.equal(read(0, prompt), first)
    for s in (1, 2, 3):
        assert torch.equal(read(s, 32), first[:32])           # shared blocks; the copied one may have been rounded again for a larger row
        assert float((read(s, prompt)[32:].float() - first[32:].float()).abs().max()) <= 2 * float(scales[table[s, 2]])
    assert table[1:, :2].tolist() == [table[0, :2].tolist()] * 3 and refs[table[0, :2].long()].tolist() == [4, 4]
    assert len({int(x) for x in table[:, 2]}) == 4
    # a drafted tree on each sample, over the shared and the own pages
    q, rows, out = (rand(8, 64, 512) * 0.7).half(), rand(8, 512).half(), torch.empty(8, 64, 512, dtype=torch.float16, device="cuda")
    tree, starts = ints([-1, 0, -1, -1, 0, 0, -1, 0]), ints([0, 2, 3, 6, 8])
    hk.mla8_tree_decode(q, ckv8, scales, rows, tree, out, 8, n_seqs=4, tree_start=starts, block_table=table, kv_len=ints(lens), n_keys_hint=max(lens))
    finish()
    for s, r, mates in ((0, 1, [0, 1]), (1, 2, [2]), (2, 5, [3, 5]), (3, 7, [6, 7])):
        k = torch.cat((read(s, lens[s]).double(), rows[mates].double()))
        o = torch.softmax(q[r].double() @ k.T * 0.0625, 1) @ k
        # rows as read are fp16 roundings of the cache's: 2^-11 of scores of up to ~100 each way, and of the values
        assert float((out[r].double() - o).abs().max()) <= 2.0 ** -4
    hk.mla8_pages_free(*pool, ints([1, 2, 3]), None, 3)
    finish()
    assert int(refs.sum()) == 3 and table[1:].max() == -1
