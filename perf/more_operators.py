"""Trees of drafted tokens - attention over the latent caches, the KDA recurrence and its step to the accepted node - and the pages of the
8-bit cache: cases for measurement.

Kinds of case:

  tree      attention of drafted tokens: `seqs` sequences of about `ctx` cached keys, each with a tree of up to `nodes` tokens that hang on its
            last one.  A node attends to the sequence's cache and to its ancestors and itself.  Over the fp16 cache ("f16", sequences one after
            the other) or the paged 8-bit one ("i8", "e4m3" in blocks of `block` tokens); the nodes' own latents are fp16 rows beside it
  kda       the KDA recurrence of every node, each from its parent's state; the sequences' own states stay as they are
  accept    the states and convolution windows of a batch step to the node that was accepted of each tree (some trees have none)
  fork      sequences of a paged cache take over the pages of others: whole blocks shared, the last one copied (parallel samples, beams).
            Children are forked again by every pass, which gives back what they held
  turnover  half of the sequences end, the live pages move together, new sequences take pages; then the same with the other half

`run` computes the plain form (elementary operations in 32 bits) or, with `own`, makes the package's calls.
"""
import math

import torch

own = False

LAT, D, SCALE, MAX_NODES = 512, 128, 0.0625, 64
QMAX = {"i8": 127.0, "e4m3": 448.0}
STORE = {"i8": torch.int8, "e4m3": torch.float8_e4m3fn}


def listed():
    return [
        # one chat of a few thousand tokens, a small tree: the smallest call
        {"name": "tree_1x8_at_5001", "kind": "tree", "seqs": 1, "nodes": 8, "ctx": 5001, "cache": "f16", "block": 0, "heads": 64, "shape": "tree"},
        # a long document and a full tree
        {"name": "tree_1x64_at_32768", "kind": "tree", "seqs": 1, "nodes": 64, "ctx": 32768, "cache": "f16", "block": 0, "heads": 64, "shape": "tree"},
        # a batch on one of four GPUs that share the heads, chains of drafted tokens
        {"name": "tree_12x5_at_3000_of_16_heads", "kind": "tree", "seqs": 12, "nodes": 5, "ctx": 3000, "cache": "e4m3", "block": 16, "heads": 16,
         "shape": "chain"},
        # a batch of long ragged sequences
        {"name": "tree_6x16_at_10000", "kind": "tree", "seqs": 6, "nodes": 16, "ctx": 10000, "cache": "i8", "block": 64, "heads": 64, "shape": "tree"},
        # the recurrence beside the first of these cases, and beside a batch with full trees
        {"name": "kda_1x8", "kind": "kda", "seqs": 1, "nodes": 8, "heads": 32, "shape": "tree"},
        {"name": "kda_8x61", "kind": "kda", "seqs": 8, "nodes": 61, "heads": 32, "shape": "tree"},
        # their steps; the batch's states fill the GPU
        {"name": "accept_1x8", "kind": "accept", "seqs": 1, "nodes": 8, "heads": 32, "shape": "tree"},
        {"name": "accept_24x13", "kind": "accept", "seqs": 24, "nodes": 13, "heads": 64, "shape": "tree"},
        # four samples of one prompt, and 48 of twelve
        {"name": "fork_4_at_5001", "kind": "fork", "seqs": 4, "parents": 1, "ctx": 5001, "cache": "e4m3", "block": 64, "spare": 40},
        {"name": "fork_48_at_9000", "kind": "fork", "seqs": 48, "parents": 12, "ctx": 9000, "cache": "i8", "block": 128, "spare": 300},
        # a small pool, and one of 226 MB
        {"name": "turnover_10_at_1500", "kind": "turnover", "seqs": 10, "ctx": 1500, "cache": "e4m3", "block": 16, "spare": 111},
        {"name": "turnover_64_at_8191", "kind": "turnover", "seqs": 64, "ctx": 8191, "cache": "i8", "block": 64, "spare": 700},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "kda", "kda", "accept", "fork", "turnover"])
    shape = rng.choice(["tree", "tree", "chain"])
    paged = {"cache": rng.choice(["i8", "e4m3"]), "block": rng.choice([16, 32, 64, 128])}
    if kind == "tree":
        seqs, nodes = _log(rng, 1, 16), _log(rng, 1, 64)
        cache = paged if rng.random() < 0.5 else {"cache": "f16", "block": 0}
        return {"kind": kind, "seqs": seqs, "nodes": nodes, "ctx": _log(rng, 1, min(32768, 64 * 32768 // (seqs * nodes))), **cache,
                "heads": rng.choice([16, 32, 64]) if cache["block"] else 64, "shape": shape}
    if kind == "kda":
        heads = rng.choice([16, 32, 64])
        return {"kind": kind, "seqs": _log(rng, 1, 8 * 32 // heads), "nodes": _log(rng, 1, 61), "heads": heads, "shape": shape}
    if kind == "accept":
        return {"kind": kind, "seqs": _log(rng, 1, 24), "nodes": _log(rng, 1, 13), "heads": rng.choice([16, 32, 64]), "shape": shape}
    if kind == "fork":
        parents = _log(rng, 1, 12)
        return {"kind": kind, "seqs": parents * rng.randint(1, 4), "parents": parents, "ctx": _log(rng, 1, 9000), **paged, "spare": _log(rng, 100, 300)}
    return {"kind": kind, "seqs": _log(rng, 2, 64), "ctx": _log(rng, 16, 8191), **paged, "spare": _log(rng, 1, 700)}


def _lens(case):
    """keys of each sequence: from `ctx` down to about half of it"""
    n = case["seqs"]
    return [max(1, case["ctx"] - i * case["ctx"] // (2 * n)) for i in range(n)]


def _sizes(case):
    """nodes of each tree: up to `nodes`, a few less in some"""
    return [max(1, case["nodes"] - (i % 3) * case["nodes"] // 8) for i in range(case["seqs"])]


def _parents(case):
    """the trees, the same for every seed: a chain, or nodes that hang on one of the earlier ones"""
    trees, x = [], 12345
    for n in _sizes(case):
        tree = []
        for j in range(n):
            x = (x * 1103515245 + 12345) % (1 << 31)
            tree.append(j - 1 if case["shape"] == "chain" or j == 0 else (x >> 12) % (j + 1) - 1)
        trees.append(tree)
    return trees


def _paths(tree):
    """ancestors of each node, the node itself last"""
    paths = []
    for p in tree:
        paths.append((paths[p] if p >= 0 else []) + [len(paths)])
    return paths


def _leaves(case):
    """the accepted node of each tree: one of the deepest, of every seventh tree none"""
    out = []
    for i, tree in enumerate(_parents(case)):
        paths = _paths(tree)
        out.append(-1 if i % 7 == 3 else max(range(len(tree)), key=lambda j: (len(paths[j]), j)))
    return out


def _rows_like_a_layer(gen, n):
    """latent rows as they leave the RMS norm: channels of unequal size, a few large ones"""
    x = torch.randn(n, LAT, device="cuda", generator=gen)
    return x * (1.0 + 3.0 * (torch.arange(LAT, device="cuda") % 97 == 5))


def _pool(gen, case, n_blocks):
    """blocks of 8-bit values and their scales"""
    block, dtype = case["block"], case["cache"]
    q, s = [], []
    for b0 in range(0, n_blocks, 1 << 11):
        y = _rows_like_a_layer(gen, min(1 << 11, n_blocks - b0) * block).view(-1, block, LAT)
        scale = y.abs().amax((1, 2)) / QMAX[dtype]
        y = (y / scale[:, None, None]).clamp(-QMAX[dtype], QMAX[dtype])
        q.append((y.round() if dtype == "i8" else y).to(STORE[dtype]).view(torch.uint8))
        s.append(scale)
    return torch.cat(q).view(STORE[dtype]), torch.cat(s)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _blocks(n, block):
    return (n + block - 1) // block


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, seqs = case["kind"], case["seqs"]
    st = {"case": case}
    rand = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    if kind in ("fork", "turnover"):
        block = case["block"]
        if kind == "fork":
            # the parents hold `ctx` tokens and less; their children, the rows behind them, hold nothing yet
            n_par = case["parents"]
            lens = [max(1, case["ctx"] - i * case["ctx"] // (2 * n_par)) for i in range(n_par)]
            who = [i % n_par for i in range(seqs)]
            st["parents"], st["children"] = _ints(who), _ints([n_par + i for i in range(seqs)])
            st["lens"] = _ints([lens[p] for p in who])
            rows = n_par + seqs
            room = seqs + case["spare"]
        else:
            lens, rows, room = _lens(case), seqs, case["spare"]
            halves = [list(range(0, seqs, 2)), list(range(1, seqs, 2))]
            st["halves"] = [(_ints(h), _ints([0] * len(h)), _ints([lens[i] for i in h])) for h in halves]
        per = [_blocks(n, block) for n in lens]
        total = sum(per) + room
        st["ckv8"], st["scales"] = _pool(gen, case, total)
        where = torch.randperm(total, device="cuda", generator=gen).to(torch.int32)
        st["table"] = torch.full((rows, max(per)), -1, dtype=torch.int32, device="cuda")
        st["refs"] = torch.zeros(total, dtype=torch.int32, device="cuda")
        at = 0
        for i, k in enumerate(per):
            st["table"][i, :k] = where[at:at + k]
            at += k
        st["refs"][where[:at].long()] = 1
        st["max_entries"] = max(per)
        return st
    trees, sizes = _parents(case), _sizes(case)
    m = sum(sizes)
    starts = [sum(sizes[:i]) for i in range(seqs + 1)]
    st["trees"], st["starts"], st["m"] = trees, starts, m
    st["parent"], st["tree_start"] = _ints([p for t in trees for p in t]), _ints(starts)
    if kind == "tree":
        lens, heads, block = _lens(case), case["heads"], case["block"]
        st["max_len"], st["lens"] = max(lens), lens
        st["kv_len"] = _ints(lens)
        st["q"] = (rand(m, heads, LAT) * 0.7).half()
        st["tree_kv"] = _rows_like_a_layer(gen, m).mul_(0.7).half()
        st["out"] = torch.empty(m, heads, LAT, dtype=torch.float16, device="cuda")
        if case["cache"] == "f16":
            st["base"] = torch.tensor([sum(lens[:i]) for i in range(seqs)], dtype=torch.int64, device="cuda")
            st["ckv"] = _rows_like_a_layer(gen, sum(lens)).mul_(0.7).half()
        else:
            per = [_blocks(n, block) for n in lens]
            st["ckv8"], st["scales"] = _pool(gen, case, sum(per) + 3)
            where = torch.randperm(sum(per) + 3, device="cuda", generator=gen).to(torch.int32)
            st["table"] = torch.full((seqs, max(per)), -1, dtype=torch.int32, device="cuda")
            for i, k in enumerate(per):
                st["table"][i, :k] = where[sum(per[:i]):sum(per[:i]) + k]
        # ancestors and self of every node, for the plain form
        see = torch.zeros(m, MAX_NODES, dtype=torch.bool)
        for s, tree in enumerate(trees):
            for j, path in enumerate(_paths(tree)):
                see[starts[s] + j, path] = True
        st["see"] = see.cuda()
        return st
    heads = case["heads"]
    st["qkv"] = rand(m, 3 * heads * D).bfloat16()
    a_log = torch.rand(heads, 1, device="cuda", generator=gen) * math.log(8.0) + math.log(0.5)
    st["g"] = (-5.0 * torch.sigmoid(torch.exp(a_log) * (rand(m, heads, D) + 0.5 * rand(heads, D)))).contiguous()
    st["beta"] = torch.sigmoid(rand(m, heads)).bfloat16()
    st["state"] = 0.2 * rand(seqs, heads, D, D)
    if kind == "kda":
        st["out"] = torch.empty(m, heads, D, dtype=torch.bfloat16, device="cuda")
    else:
        st["x32"] = rand(m, 3 * heads * D)
        st["window"] = rand(seqs, 3 * heads * D, 4).bfloat16()
        st["leaves"] = _leaves(case)
        st["leaf"] = _ints(st["leaves"])
    return st


# ---- plain forms ----
def _values(st, blocks):
    """cache blocks as fp32 rows: [...][block][512]"""
    return st["ckv8"].view(torch.uint8)[blocks].view(STORE[st["case"]["cache"]]).float() * st["scales"][blocks][..., None, None]


def _plain_tree(st):
    heads = st["case"]["heads"]
    for s, n in enumerate(st["lens"]):
        t0, t1 = st["starts"][s], st["starts"][s + 1]
        if st["case"]["cache"] == "f16":
            first = sum(st["lens"][:s])
            past = st["ckv"][first:first + n].float()
        else:
            past = _values(st, st["table"][s, :_blocks(n, st["case"]["block"])].long()).reshape(-1, LAT)[:n]
        k = torch.cat((past, st["tree_kv"][t0:t1].float()))
        q = st["q"][t0:t1].float().reshape(-1, LAT)
        x = torch.mm(q, k.T).mul_(SCALE).view(t1 - t0, heads, -1)
        x[:, :, n:].masked_fill_(~st["see"][t0:t1, None, :t1 - t0], -math.inf)
        p = torch.exp(x - x.amax(-1, keepdim=True))
        out = torch.mm(p.view(q.shape[0], -1), k) / p.sum(-1).view(-1, 1)
        st["out"][t0:t1] = out.view(t1 - t0, heads, LAT)
    return st["out"]


def _normed(x):
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + 1e-6)


def _tokens(st, rows):
    """q, k, v, decay and beta of some nodes: [n][heads][...]"""
    heads = st["case"]["heads"]
    q, k, v = st["qkv"][rows].float().view(-1, 3, heads, D).unbind(1)
    return _normed(q), _normed(k), v, torch.exp(st["g"][rows]), st["beta"][rows].float()


def _step(s, k, v, d, b):
    """one token on states [n][heads][128][128]"""
    s = s * d[..., None]
    u = (v - (k[..., None] * s).sum(-2)) * b[..., None]
    return s + k[..., None] * u[..., None, :]


def _toward_zero(x):
    return (x.view(torch.int32) & -65536).view(torch.float32).bfloat16()


def _plain_kda(st):
    seqs = st["case"]["seqs"]
    most = max(len(t) for t in st["trees"])
    # every sequence's j-th node at once; where a tree has ended, its last node again
    states = torch.empty(most + 1, *st["state"].shape, device="cuda")
    states[0] = st["state"]
    every = torch.arange(seqs, device="cuda")
    for j in range(most):
        at = [min(j, len(t) - 1) for t in st["trees"]]
        rows = torch.tensor([st["starts"][s] + i for s, i in enumerate(at)], device="cuda")
        before = torch.tensor([t[i] + 1 for t, i in zip(st["trees"], at)], device="cuda")
        q, k, v, d, b = _tokens(st, rows)
        s = _step(states[before, every], k, v, d, b)
        states[j + 1] = s
        st["out"][rows] = _toward_zero((q[..., None] * s).sum(-2) * D ** -0.5)
    return st["out"]


def _plain_accept(st):
    for s, leaf in enumerate(st["leaves"]):
        if leaf < 0:
            continue
        rows = st["starts"][s] + torch.tensor(_paths(st["trees"][s])[leaf], device="cuda")
        _, k, v, d, b = _tokens(st, rows)
        x = st["state"][s]
        for i in range(len(rows)):
            x = _step(x, k[i], v[i], d[i], b[i])
        st["state"][s] = x
        st["window"][s] = torch.cat((st["window"][s], st["x32"][rows].bfloat16().T), 1)[:, -4:]
    return st["state"], st["window"]


def _drop(st, seqs):
    """the sequences' pages lose a reference each"""
    held = st["table"][seqs].flatten()
    held = held[held >= 0].long()
    st["refs"].scatter_add_(0, held, torch.full_like(held, -1, dtype=torch.int32))
    st["table"][seqs] = -1


def _plain_fork(st):
    block = st["case"]["block"]
    par, child, lens = st["parents"].long(), st["children"].long(), st["lens"].long()
    _drop(st, child)
    j = torch.arange(st["table"].shape[1], device="cuda")
    rows = torch.where(j < (lens // block)[:, None], st["table"][par], -1)
    shared = rows[rows >= 0].long()
    st["refs"].scatter_add_(0, shared, torch.ones_like(shared, dtype=torch.int32))
    part = (lens % block > 0).nonzero()[:, 0]
    fresh = (st["refs"] == 0).nonzero()[:len(part), 0]
    part = part[:len(fresh)]
    source = st["table"][par[part], lens[part] // block].long()
    rows[part, lens[part] // block] = fresh.int()
    st["refs"][fresh] = 1
    st["ckv8"].view(torch.uint8)[fresh] = st["ckv8"].view(torch.uint8)[source]
    st["scales"][fresh] = st["scales"][source]
    st["table"][child] = rows
    return _pool_outputs(st)


def _plain_turnover(st):
    for seqs, _, lens in st["halves"]:
        seqs, lens = seqs.long(), lens.long()
        _drop(st, seqs)
        live = st["refs"] > 0
        n_live = int(live.sum())
        source = live[n_live:].nonzero()[:, 0] + n_live
        target = (~live[:n_live]).nonzero()[:, 0]
        st["ckv8"].view(torch.uint8)[target] = st["ckv8"].view(torch.uint8)[source]
        st["scales"][target] = st["scales"][source]
        st["refs"][target] = st["refs"][source]
        st["refs"][source] = 0
        moved = torch.arange(len(st["refs"]), dtype=torch.int32, device="cuda")
        moved[source] = target.int()
        st["table"][:] = torch.where(st["table"] >= 0, moved[st["table"].clamp(min=0).long()], -1)
        need = (lens + st["case"]["block"] - 1) // st["case"]["block"]
        fresh = (st["refs"] == 0).nonzero()[:int(need.sum()), 0]
        st["refs"][fresh] = 1
        rows = torch.full((len(seqs), st["table"].shape[1]), -1, dtype=torch.int32, device="cuda")
        rows[torch.arange(st["table"].shape[1], device="cuda") < need[:, None]] = fresh.int()
        st["table"][seqs] = rows
    return _pool_outputs(st)


def _pool_outputs(st):
    return st["table"], st["refs"], st["scales"], st["ckv8"]


# ---- the package's calls ----
def _own(st):
    import helios_glm53flash_b200 as hk
    case, kind = st["case"], st["case"]["kind"]
    if kind == "tree":
        tree = dict(n_seqs=case["seqs"], tree_start=st["tree_start"], kv_len=st["kv_len"], n_keys_hint=st["max_len"], n_heads=case["heads"])
        if case["cache"] == "f16":
            hk.mla_tree_decode(st["q"], st["ckv"], st["tree_kv"], st["parent"], st["out"], st["m"], kv_base=st["base"], **tree)
        else:
            hk.mla8_tree_decode(st["q"], st["ckv8"], st["scales"], st["tree_kv"], st["parent"], st["out"], st["m"], block_table=st["table"], **tree)
        return st["out"]
    if kind == "kda":
        hk.kda_tree_decode(st["qkv"], st["g"], st["beta"], st["state"], st["parent"], st["out"], st["m"], case["heads"], n_seqs=case["seqs"],
                           tree_start=st["tree_start"], max_nodes=case["nodes"])
        return st["out"]
    if kind == "accept":
        hk.kda_tree_accept(st["x32"], st["window"], st["qkv"], st["g"], st["beta"], st["state"], st["parent"], st["leaf"], st["m"], case["heads"],
                           n_seqs=case["seqs"], tree_start=st["tree_start"])
        return st["state"], st["window"]
    pool = (st["ckv8"], st["scales"], st["refs"], st["table"])
    if kind == "fork":
        hk.mla8_pages_fork(*pool, st["parents"], st["children"], st["lens"], case["seqs"])
    else:
        for seqs, keep, lens in st["halves"]:
            hk.mla8_pages_free(*pool, seqs, keep, len(seqs))
            hk.mla8_pages_compact(*pool)
            hk.mla8_pages_reserve(*pool, seqs, lens, len(seqs))
    return _pool_outputs(st)


PLAIN = {"tree": _plain_tree, "kda": _plain_kda, "accept": _plain_accept, "fork": _plain_fork, "turnover": _plain_turnover}


def run(state):
    return _own(state) if own else PLAIN[state["case"]["kind"]](state)


def work(case):
    kind, seqs = case["kind"], case["seqs"]
    if kind in ("fork", "turnover"):
        page = case["block"] * LAT + 4
        if kind == "fork":
            n_par = case["parents"]
            lens = [max(1, case["ctx"] - i * case["ctx"] // (2 * n_par)) for i in range(n_par)]
            lens = [lens[i % n_par] for i in range(seqs)]
            entries = sum(_blocks(n, case["block"]) for n in lens)
            # entries of parent and child, their references twice; the last pages there and back; the count of references
            return {"bytes": entries * 4 * 4 + 2 * page * sum(n % case["block"] > 0 for n in lens) + 4 * seqs, "flops": entries}
        per = [_blocks(n, case["block"]) for n in _lens(case)]
        total = sum(per) + case["spare"]
        # from the second pass on each half lies behind the other, and moves as far as it is no longer than the gap or the gap itself
        a, b = sum(per[0::2]), sum(per[1::2])
        return {"bytes": 4 * page * min(a, b) + 2 * (2 * 4 * total + 3 * 4 * (a + b)), "flops": 2 * total}
    m = sum(_sizes(case))
    depths = [len(p) for t in _parents(case) for p in _paths(t)]
    if kind == "tree":
        lens, sizes, heads = _lens(case), _sizes(case), case["heads"]
        key = LAT * 2 if case["cache"] == "f16" else LAT + 4 / case["block"]
        pairs = sum(n * t for n, t in zip(lens, sizes)) + sum(depths)
        return {"bytes": int(sum(lens) * key) + m * (LAT * 2 + 4) + 2 * 2 * LAT * heads * m, "flops": 4 * LAT * heads * pairs}
    heads = case["heads"]
    token = 3 * heads * D * 2 + heads * D * 4 + heads * 2
    if kind == "kda":
        return {"bytes": seqs * heads * D * D * 4 + m * (token + heads * D * 2 + 4), "flops": heads * (4 * D * D * m + 8 * D * sum(depths))}
    steps = sum(len(_paths(t)[leaf]) for t, leaf in zip(_parents(case), _leaves(case)) if leaf >= 0)
    moved = sum(leaf >= 0 for leaf in _leaves(case))
    rows = sum(min(4, len(_paths(t)[leaf])) for t, leaf in zip(_parents(case), _leaves(case)) if leaf >= 0)
    return {"bytes": 2 * moved * heads * D * D * 4 + steps * token * 2 // 3 + 3 * heads * D * (rows * 4 + moved * 16),
            "flops": heads * 6 * D * D * steps}


# ---- the definition in 64 bits ----
def exact(case, seed):
    st = prepare(case, seed)
    kind, f64 = case["kind"], torch.float64
    if kind == "tree":
        heads, block = case["heads"], case["block"]
        out = torch.empty(st["m"], heads, LAT, dtype=f64, device="cuda")
        for s, (n, tree) in enumerate(zip(st["lens"], st["trees"])):
            if block:
                p = torch.arange(n, device="cuda")
                b = st["table"][s][p // block].long()
                past = st["ckv8"].view(torch.uint8)[b, p % block].view(STORE[case["cache"]]).to(f64) * st["scales"][b].to(f64)[:, None]
            else:
                past = st["ckv"][int(st["base"][s]):int(st["base"][s]) + n].to(f64)
            drafted = st["tree_kv"][st["starts"][s]:st["starts"][s + 1]].to(f64)
            for j in range(len(tree)):
                chain, i = [], j
                while i >= 0:
                    chain.append(i)
                    i = tree[i]
                k = torch.cat((past, drafted[chain]))
                r = st["starts"][s] + j
                out[r] = torch.softmax(st["q"][r].to(f64) @ k.T * SCALE, -1) @ k
        return out
    if kind in ("kda", "accept"):
        heads = case["heads"]
        out = torch.empty(st["m"], heads, D, dtype=f64, device="cuda")
        state = st["state"].to(f64)
        window = st["window"].to(f64) if kind == "accept" else None
        for s, tree in enumerate(st["trees"]):
            made = {-1: state[s].clone()}
            wanted = range(len(tree))
            if kind == "accept":
                wanted, i = [], st["leaves"][s]
                while i >= 0:
                    wanted.insert(0, i)
                    i = tree[i]
            for j in wanted:
                row = st["qkv"][st["starts"][s] + j].to(f64)
                q, k, v = (row[i * heads * D:(i + 1) * heads * D].view(heads, D) for i in range(3))
                q, k = (x / torch.sqrt(x.pow(2).sum(1, keepdim=True) + 1e-6) for x in (q, k))
                x = made[tree[j]] * torch.exp(st["g"][st["starts"][s] + j].to(f64)).unsqueeze(2)
                u = st["beta"][st["starts"][s] + j].to(f64)[:, None] * (v - torch.einsum("hk,hkv->hv", k, x))
                made[j] = x + torch.einsum("hk,hv->hkv", k, u)
                out[st["starts"][s] + j] = torch.einsum("hk,hkv->hv", q, made[j]) / math.sqrt(D)
                if kind == "accept":
                    new = st["x32"][st["starts"][s] + j].bfloat16().to(f64)
                    window[s] = torch.stack((window[s, :, 1], window[s, :, 2], window[s, :, 3], new), 1)
            if kind == "accept" and wanted:
                state[s] = made[wanted[-1]]
        return out if kind == "kda" else (state, window)
    # pages: whole numbers, block by block
    table, refs = st["table"].tolist(), st["refs"].tolist()
    order = list(range(len(refs)))                           # whose contents a block holds
    block = case["block"]

    def release(s):
        for j, b in enumerate(table[s]):
            if b >= 0:
                refs[b] -= 1
                table[s][j] = -1

    def take():
        b = refs.index(0)
        refs[b] = 1
        return b

    if kind == "fork":
        todo = list(zip(st["parents"].tolist(), st["children"].tolist(), st["lens"].tolist()))
        for _, c, _ in todo:
            release(c)
        for p, c, n in todo:
            for j in range(n // block):
                table[c][j] = table[p][j]
                refs[table[p][j]] += 1
        for p, c, n in todo:
            if n % block:
                b = take()
                table[c][n // block] = b
                order[b] = order[table[p][n // block]]
    else:
        for seqs, _, lens in st["halves"]:
            for s in seqs.tolist():
                release(s)
            n_live = sum(r > 0 for r in refs)
            holes = [b for b in range(n_live) if refs[b] == 0]
            goes = {}
            for src, dst in zip((b for b in range(n_live, len(refs)) if refs[b] > 0), holes):
                goes[src] = dst
                order[dst] = order[src]
                refs[dst], refs[src] = refs[src], 0
            table = [[goes.get(b, b) for b in row] for row in table]
            free = (b for b in range(len(refs)) if refs[b] == 0)
            for s, n in zip(seqs.tolist(), lens.tolist()):
                for j in range(_blocks(n, block)):
                    table[s][j] = next(free)
            for s in seqs.tolist():
                for b in table[s]:
                    if b >= 0:
                        refs[b] = 1
    at = torch.tensor(order, device="cuda")
    whole = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return whole(table), whole(refs), st["scales"][at], st["ckv8"].view(torch.uint8)[at].view(STORE[case["cache"]])
