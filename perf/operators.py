"""The 8-bit paged latent cache with the attention that reads it, and attention with a window and sinks: cases for measurement.

Kinds of case:

  append   RMS norm of new latent rows and their place in the paged 8-bit cache: one new token for each of `seqs` sequences, or a chunk of
           one sequence.  Blocks that hold rows already keep their scale or, where a new row needs a larger one, get it
  dense    attention over the paged 8-bit cache: one query row for each of `seqs` sequences of its own length each, or a causal chunk
           of `rows` rows of one sequence; `window` > 0: the last `window` keys of a row and the first `sinks`
  sparse   attention over `kidx` gathered positions a row (the model's selection) of the paged 8-bit cache
  window   attention with a window and sinks over the fp16 cache: rows of sequences that lie one after the other, or a causal chunk

The cache is int8 ("i8") or e4m3 ("e4m3") in blocks of `block` tokens with one fp32 scale each; a table says where a sequence's blocks
are.  `run` computes the plain form (elementary operations in 32 bits) or, with `own`, makes the package's calls.
"""
import math

import torch

own = False

LAT, SCALE, EPS, KIDX = 512, 0.0625, 1e-6, 2052
QMAX = {"i8": 127.0, "e4m3": 448.0}
STORE = {"i8": torch.int8, "e4m3": torch.float8_e4m3fn}


def listed():
    return [
        # the next token of one chat: the smallest call
        {"name": "append_1", "kind": "append", "seqs": 1, "rows": 1, "ctx": 4999, "dtype": "e4m3", "block": 64},
        # a decode step of a full batch, small blocks
        {"name": "append_64", "kind": "append", "seqs": 64, "rows": 1, "ctx": 2000, "dtype": "e4m3", "block": 16},
        # a prefill chunk that begins inside a block
        {"name": "append_chunk_4096", "kind": "append", "seqs": 1, "rows": 4096, "ctx": 8197, "dtype": "i8", "block": 64},
        # the next token of one chat of a few thousand tokens
        {"name": "dense_1_at_5001", "kind": "dense", "seqs": 1, "rows": 1, "ctx": 5001, "dtype": "i8", "block": 64, "heads": 64, "window": 0, "sinks": 0},
        # eight long sequences, each of its own length
        {"name": "dense_8_at_32768", "kind": "dense", "seqs": 8, "rows": 1, "ctx": 32768, "dtype": "i8", "block": 64, "heads": 64, "window": 0,
         "sinks": 0},
        # a batch on one of four GPUs that share the heads, small blocks, windows with sinks
        {"name": "dense_48x16_window_1000", "kind": "dense", "seqs": 48, "rows": 1, "ctx": 7000, "dtype": "e4m3", "block": 16, "heads": 16,
         "window": 1000, "sinks": 4},
        # a prefill chunk of no round length behind a cached prefix
        {"name": "dense_chunk_1000_at_8192", "kind": "dense", "seqs": 1, "rows": 1000, "ctx": 8192, "dtype": "i8", "block": 32, "heads": 64, "window": 0,
         "sinks": 0},
        # the sparse layer's attention of one decoded token
        {"name": "sparse_1_at_32768", "kind": "sparse", "rows": 1, "ctx": 32768, "kidx": KIDX, "dtype": "e4m3", "block": 64},
        # and of a prefill chunk
        {"name": "sparse_400_at_16384", "kind": "sparse", "rows": 400, "ctx": 16384, "kidx": KIDX, "dtype": "i8", "block": 128},
        # one long sequence that attends to its last 4,096 tokens and the first 4
        {"name": "window_1_at_100001", "kind": "window", "seqs": 1, "rows": 1, "ctx": 100001, "window": 4096, "sinks": 4},
        # a decode batch of short windows, lengths below the window among them
        {"name": "window_24_at_5000", "kind": "window", "seqs": 24, "rows": 1, "ctx": 5000, "window": 1024, "sinks": 64},
        # a prefill chunk
        {"name": "window_chunk_2048_at_20000", "kind": "window", "seqs": 1, "rows": 2048, "ctx": 20000, "window": 1023, "sinks": 16},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "dense", "dense", "sparse", "window", "window"])
    form = {"dtype": rng.choice(["i8", "e4m3"]), "block": rng.choice([16, 32, 64, 128])}
    chunk = rng.random() < 0.4
    if kind == "append":
        size = {"seqs": 1, "rows": _log(rng, 2, 4096)} if chunk else {"seqs": _log(rng, 1, 64), "rows": 1}
        return {"kind": kind, **size, "ctx": _log(rng, 1, 8192), **form}
    if kind == "sparse":
        return {"kind": kind, "rows": _log(rng, 1, 400), "ctx": _log(rng, 64, 32768), "kidx": rng.choice([KIDX, _log(rng, 1, KIDX)]), **form}
    band = {"window": _log(rng, 1, 4096), "sinks": rng.choice([0, 1, 4, 16, 64, 100])}
    if kind == "window":
        if chunk:
            return {"kind": kind, "seqs": 1, "rows": _log(rng, 2, 2048), "ctx": _log(rng, 1, 20000), **band, "window": _log(rng, 1, 1024)}
        seqs = _log(rng, 1, 24)
        return {"kind": kind, "seqs": seqs, "rows": 1, "ctx": _log(rng, 1, 100000 // seqs), **band}
    if rng.random() < 0.6:
        band = {"window": 0, "sinks": 0}
    if chunk:
        return {"kind": kind, "seqs": 1, "rows": _log(rng, 2, 1000), "ctx": _log(rng, 1, 8192), **form, "heads": 64, **band}
    seqs = _log(rng, 1, 48)
    return {"kind": kind, "seqs": seqs, "rows": 1, "ctx": _log(rng, 1, 8 * 32768 // seqs if seqs > 8 else 32768), **form,
            "heads": rng.choice([8, 16, 32, 64, 64]), **band}


def _lens(case):
    """keys of each sequence: from `ctx` down to about half of it; a chunk's sequence ends with the chunk"""
    if case["rows"] > 1 or case["kind"] == "sparse":
        return [case["ctx"] + case["rows"]]
    n = case["seqs"]
    return [max(1, case["ctx"] - i * case["ctx"] // (2 * n)) for i in range(n)]


def _seen(n, case):
    """keys that a row of length n attends to"""
    w = case.get("window", 0)
    return n if not w else min(n, w) + min(case["sinks"], max(0, n - w))


def _row_lens(case):
    lens = _lens(case)
    return [case["ctx"] + r + 1 for r in range(case["rows"])] if case["rows"] > 1 else lens


def _rows_like_a_layer(gen, n):
    """latent rows as they leave the RMS norm: channels of unequal size, a few large ones"""
    x = torch.randn(n, LAT, device="cuda", generator=gen)
    return x * (1.0 + 3.0 * (torch.arange(LAT, device="cuda") % 97 == 5))


def _stored(y, dtype):
    """[blocks][block][512] fp32 -> 8-bit values and a scale a block"""
    s = y.abs().amax((1, 2)) / QMAX[dtype]
    q = torch.where(s[:, None, None] > 0, y / s[:, None, None], torch.zeros((), device=y.device)).clamp(-QMAX[dtype], QMAX[dtype])
    return (q.round() if dtype == "i8" else q).to(STORE[dtype]), s


def _paged(gen, case, lens):
    """a pool of blocks with some to spare, the sequences' blocks anywhere in it"""
    block = case["block"]
    per = [(n + block - 1) // block for n in lens]
    total = sum(per) + 3
    where = torch.randperm(total, device="cuda", generator=gen).to(torch.int32)
    table = torch.full((len(lens), max(per)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, k in enumerate(per):
        table[i, :k] = where[at:at + k]
        at += k
    q, s = [], []
    for b0 in range(0, total, 1 << 12):
        nb = min(1 << 12, total - b0)
        qs = _stored(_rows_like_a_layer(gen, nb * block).view(nb, block, LAT), case["dtype"])
        q.append(qs[0])
        s.append(qs[1])
    return torch.cat([x.view(torch.uint8) for x in q]).view(STORE[case["dtype"]]), torch.cat(s), table


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, rows = case["kind"], case["rows"]
    lens = _lens(case)
    st = {"case": case, "max_len": max(lens)}
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if kind == "append":
        # the sequences hold `lens` tokens (a chunk's: ctx) before the call
        st["pos"] = ints([case["ctx"]] if rows > 1 else lens)
        st["ckv8"], st["scales"], st["table"] = _paged(gen, case, [n + (0 if rows > 1 else 1) for n in lens])
        n = case["seqs"] * rows
        st["kv_pre"] = _rows_like_a_layer(gen, n) * torch.exp(torch.randn(n, 1, device="cuda", generator=gen))
        st["ln_w"] = (1.0 + 0.1 * torch.randn(LAT, device="cuda", generator=gen)).half()
        st["new"] = torch.empty(n, LAT, dtype=torch.float16, device="cuda")
        return st
    m, heads = max(rows, case.get("seqs", 1)), case.get("heads", 64)
    st["q"] = (torch.randn(m, heads, LAT, device="cuda", generator=gen) * 0.7).half()
    st["out"] = torch.empty(m, heads, LAT, dtype=torch.float16, device="cuda")
    if rows == 1 and kind != "sparse":
        st["kv_len"] = ints(lens)
    if kind == "window":
        st["base"] = torch.tensor([sum(lens[:i]) for i in range(len(lens))], dtype=torch.int64, device="cuda")
        st["ckv"] = _rows_like_a_layer(gen, sum(lens)).mul_(0.7).half()
        return st
    st["ckv8"], st["scales"], st["table"] = _paged(gen, case, lens)
    if kind == "dense" and rows == 1:
        st["row_seq"] = torch.arange(m, dtype=torch.int32, device="cuda")
    if kind == "sparse":
        idx = torch.randint(0, max(lens), (m, case["kidx"]), device="cuda", generator=gen, dtype=torch.int32)
        idx[:, 5::41] = -1                                   # selections that are not full
        st["raw_idx"] = idx.contiguous()
    return st


# ---- plain forms ----
def _values(st, blocks):
    """cache blocks as fp32 rows: [...][block][512]"""
    return st["ckv8"].view(torch.uint8)[blocks].view(STORE[st["case"]["dtype"]]).float() * st["scales"][blocks][..., None, None]


def _attend(q, k, see):
    """q [b][r][512], k [b][n][512], see [b][r][n] -> [b][r][512]; rows that see nothing are zero"""
    s = torch.baddbmm(torch.zeros((), device=q.device), q, k.transpose(1, 2), beta=0, alpha=SCALE)
    s = torch.where(see, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isfinite(top), top, torch.zeros((), device=q.device)))
    tot = p.sum(-1, keepdim=True)
    return torch.bmm(p, k) / torch.where(tot > 0, tot, torch.ones((), device=q.device))


def _plain_append(st):
    case, block, top = st["case"], st["case"]["block"], QMAX[st["case"]["dtype"]]
    x = st["kv_pre"].double()                                # where a value falls between two steps of 8 bits
    y = x * st["ln_w"].double() / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    seqs, rows = case["seqs"], case["rows"]
    pos = st["pos"].long()[:, None] + torch.arange(rows, device="cuda")                    # [seqs][rows]
    first = st["pos"].long() // block
    touched = (rows - 1) // block + 2 if rows > 1 else 1
    number = first[:, None] + torch.arange(touched, device="cuda")                         # blocks that may get rows
    real = number <= pos[:, -1:] // block
    phys = torch.gather(st["table"].long(), 1, number.clamp(max=st["table"].shape[1] - 1))
    cell = ((pos // block - first[:, None]) * block + pos % block)                         # place within the touched blocks
    area = torch.zeros(seqs, touched * block, LAT, dtype=torch.float64, device="cuda")
    fresh = torch.zeros(seqs, touched * block, 1, dtype=torch.bool, device="cuda")
    area.scatter_(1, cell[..., None].expand(-1, -1, LAT), y.view(seqs, rows, LAT))
    fresh.scatter_(1, cell[..., None], True)
    area, fresh = area.view(seqs, touched, block, LAT), fresh.view(seqs, touched, block, 1)
    need = (area.abs().amax((2, 3)) / top).float()
    held = (number * block < st["pos"].long()[:, None])                                    # rows there before
    s0 = torch.where(held, st["scales"][phys], torch.zeros((), device="cuda"))
    s1 = torch.where(need > s0, need, s0)
    to8 = lambda v: (v.round() if case["dtype"] == "i8" else v).clamp(-top, top)  # noqa: E731
    old = st["ckv8"].view(torch.uint8)[phys].view(STORE[case["dtype"]]).double()
    place = number[..., None] * block + torch.arange(block, device="cuda")
    before = (place < st["pos"].long()[:, None, None]) & (need > s0)[..., None]           # rows behind the new ones stay as they are
    moved = torch.where(before[..., None], old * (s0.double() / s1.double())[..., None, None], old)
    q = torch.where(fresh, area / torch.where(s1 > 0, s1, torch.ones((), device="cuda")).double()[..., None, None], moved)
    q = to8(q).float().to(STORE[case["dtype"]])
    st["ckv8"].view(torch.uint8)[phys[real]] = q.view(torch.uint8)[real]
    st["scales"][phys[real]] = s1[real]
    kept = torch.gather((q.float() * s1[..., None, None]).view(seqs, touched * block, LAT), 1, cell[..., None].expand(-1, -1, LAT))
    st["new"].copy_(kept.view(seqs * rows, LAT))
    return _append_outputs(st)


def _append_outputs(st):
    """the new rows as the cache holds them, the scales, and a cache of floating values itself"""
    return (st["new"], st["scales"]) + ((st["ckv8"],) if st["case"]["dtype"] == "e4m3" else ())


def _plain_attention(st):
    case, kind, rows = st["case"], st["case"]["kind"], st["case"]["rows"]
    q = st["q"].float()
    m, heads, w, sinks = q.shape[0], q.shape[1], case.get("window", 0), case.get("sinks", 0)
    if kind == "sparse":
        block, idx = case["block"], st["raw_idx"].long()
        at = idx.clamp(min=0)
        phys = st["table"][0].long()[at // block]
        k = st["ckv8"].view(torch.uint8)[phys, at % block].view(STORE[case["dtype"]]).float() * st["scales"][phys][..., None]
        return _attend(q, k, (idx >= 0)[:, None, :]).half()
    if rows > 1:
        # one sequence: the keys that any row of the chunk sees
        lo = max(0, case["ctx"] + 1 - w) if w else 0
        p = torch.arange(st["max_len"], device="cuda")
        p = torch.cat((p[:min(sinks, lo)], p[lo:])) if w else p
        n = (case["ctx"] + 1 + torch.arange(rows, device="cuda"))[:, None]
        see = (p < n) & ((p >= n - w) | (p < sinks)) if w else p < n
        k = st["ckv"][p].float() if kind == "window" else _values(st, st["table"][0].long()).view(-1, LAT)[p]
        return _attend(q.view(1, m * heads, LAT), k[None], see[:, None, :].expand(m, heads, -1).reshape(1, m * heads, -1)).half().view(m, heads, LAT)
    n = st["kv_len"].long()[:, None]
    if w:                                                    # the sinks and the window, each row's own
        width, head = min(w, st["max_len"]), min(sinks, st["max_len"])
        p = torch.cat((torch.arange(head, device="cuda").expand(m, -1), n - width + torch.arange(width, device="cuda")), 1)
        see = torch.cat((p[:, :head] < torch.clamp(n - width, min=0), p[:, head:] >= 0), 1)
        p = p.clamp(min=0)
    else:
        p = torch.arange(st["max_len"], device="cuda").expand(m, -1)
        see = p < n
        p = torch.minimum(p, n - 1)
    if kind == "window":
        k = st["ckv"][st["base"][:, None] + torch.minimum(p, n - 1)].float()
    else:
        phys = torch.gather(st["table"].long(), 1, p // case["block"])
        k = st["ckv8"].view(torch.uint8)[phys, p % case["block"]].view(STORE[case["dtype"]]).float() * st["scales"][phys][..., None]
    return _attend(q, k, see[:, None, :]).half()


# ---- the package's calls ----
def _own(st):
    import helios_glm53flash_b200 as hk
    case, kind, rows = st["case"], st["case"]["kind"], st["case"]["rows"]
    if kind == "append":
        hk.mla8_cache_append(st["kv_pre"], st["ln_w"], st["ckv8"], st["scales"], st["pos"], case["seqs"] * rows, EPS, block_table=st["table"],
                             n_seqs=case["seqs"], ckv_new=st["new"])
        return _append_outputs(st)
    m, heads = st["q"].shape[:2]
    if kind == "sparse":
        hk.mla8_sparse_decode(st["q"], st["ckv8"], st["scales"], st["raw_idx"], case["kidx"], st["out"], m, block_table=st["table"])
    elif kind == "dense" and rows > 1:
        hk.mla8_dense_prefill(st["q"], st["ckv8"], st["scales"], st["out"], m, case["ctx"], block_table=st["table"], window=case["window"],
                              sinks=case["sinks"])
    elif kind == "dense":
        hk.mla8_dense_prefill(st["q"], st["ckv8"], st["scales"], st["out"], m, 0, n_heads=heads, block_table=st["table"], row_seq=st["row_seq"],
                              kv_len=st["kv_len"], n_keys_hint=st["max_len"], window=case["window"], sinks=case["sinks"])
    elif rows > 1:
        hk.mla_window_prefill(st["q"], st["ckv"], st["out"], m, case["ctx"], case["window"], sinks=case["sinks"])
    else:
        hk.mla_window_prefill(st["q"], st["ckv"], st["out"], m, 0, case["window"], sinks=case["sinks"], kv_base=st["base"], kv_len=st["kv_len"],
                              n_keys_hint=st["max_len"])
    return st["out"]


def run(state):
    if own:
        return _own(state)
    return _plain_append(state) if state["case"]["kind"] == "append" else _plain_attention(state)


def work(case):
    kind, rows = case["kind"], case["rows"]
    if kind == "append":
        n = case["seqs"] * rows
        blocks = case["seqs"] + n // case["block"]
        return {"bytes": n * LAT * (4 + 1 + 2) + blocks * 8 + LAT * 2, "flops": 8 * n * LAT}
    heads, key = case.get("heads", 64), LAT * 2 if kind == "window" else LAT + 4 / case["block"]
    if kind == "sparse":
        seen = [case["kidx"] - len(range(5, case["kidx"], 41))] * rows
        touched = min(sum(seen), case["ctx"] + rows)
        extra = 4 * case["kidx"] * rows
    else:
        seen = [_seen(n, case) for n in _row_lens(case)]
        if rows > 1:
            lo = max(0, case["ctx"] + 1 - case["window"]) if case.get("window") else 0
            touched = case["ctx"] + rows - lo + min(case.get("sinks", 0), lo)
        else:
            touched = sum(seen)
        extra = 0
    return {"bytes": int(touched * key) + 2 * 2 * LAT * heads * len(seen) + extra, "flops": 4 * LAT * heads * sum(seen)}


# ---- the definition in 64 bits ----
def exact(case, seed):
    st = prepare(case, seed)
    f64, dev = torch.float64, "cuda"
    if case["kind"] == "append":
        top, block, e4m3 = QMAX[case["dtype"]], case["block"], case["dtype"] == "e4m3"
        x, w = st["kv_pre"].to(f64), st["ln_w"].to(f64)
        y = (w * x * (EPS + x.pow(2).sum(1, keepdim=True) / LAT).rsqrt()).cpu()
        store, scales, table = st["ckv8"].to(f64).cpu(), st["scales"].to(f64).cpu(), st["table"].cpu()
        fit = lambda v: (v.float().to(torch.float8_e4m3fn).to(f64) if e4m3 else torch.round(v)).clamp(-top, top)  # noqa: E731
        rows, new = case["rows"], torch.empty_like(y)
        for s, p0 in enumerate(st["pos"].tolist()):
            p = p0
            while p < p0 + rows:                             # block by block
                b, end = int(table[s, p // block]), min(p0 + rows, (p // block + 1) * block)
                mine = slice(s * rows + p - p0, s * rows + end - p0)
                need = float(y[mine].abs().max()) / top
                before = float(scales[b]) if p % block else 0.0
                if need > before:
                    store[b, :p % block] = fit(store[b, :p % block] * (before / need))
                    scales[b] = need
                elif not p % block:
                    scales[b] = 0.0
                unit = float(scales[b])
                store[b, p % block:p % block + end - p] = fit(y[mine] / unit) if unit else 0.0
                new[mine] = store[b, p % block:p % block + end - p] * unit
                p = end
        return (new.to(dev), scales.to(dev)) + ((store.to(dev),) if e4m3 else ())
    q = st["q"].to(f64)
    m, heads, w, sinks = q.shape[0], q.shape[1], case.get("window", 0), case.get("sinks", 0)
    out = torch.zeros(m, heads, LAT, dtype=f64, device=dev)
    lens = _row_lens(case)

    def keys(r, p):
        if case["kind"] == "window":
            return st["ckv"][p + (int(st["base"][r]) if case["rows"] == 1 else 0)].to(f64)
        b = st["table"][r if case["kind"] == "dense" and case["rows"] == 1 else 0][p // case["block"]].long()
        return st["ckv8"].view(torch.uint8)[b, p % case["block"]].view(STORE[case["dtype"]]).to(f64) * st["scales"][b].to(f64)[:, None]

    everything = keys(0, torch.arange(_lens(case)[0], device=dev)) if case["rows"] > 1 and case["kind"] != "sparse" else None
    for r in range(m):
        if case["kind"] == "sparse":
            p = st["raw_idx"][r].long()
            p = p[p >= 0]
        else:
            n = lens[r]
            p = torch.arange(n, device=dev)
            if w:
                p = p[(p >= n - w) | (p < sinks)]
        if p.numel():
            k = keys(r, p) if everything is None else everything[p] if w else everything[:n]
            out[r] = torch.softmax(q[r] @ k.T * SCALE, 1) @ k
    return out
