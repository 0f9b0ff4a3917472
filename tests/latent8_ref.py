"""The 8-bit paged latent cache and windowed attention in 64 bits, and how far the kernels may be from it."""
import math

import torch

STORE = {"i8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"i8": 127.0, "e4m3": 448.0}
EPS = 1e-6


def as_f64(ckv8):
    return ckv8.double() if ckv8.dtype == torch.int8 else ckv8.float().double()


def normed(kv_pre, ln_w, eps=EPS):
    x = kv_pre.double()
    return x * ln_w.double() * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)


def half_step(x, kind):
    """half the distance between neighbouring 8-bit values at |x| (unscaled)"""
    if kind == "i8":
        return torch.full_like(x, 0.5)
    return 2.0 ** (torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 4)      # three bits behind the leading one, subnormals below 2^-6


def check_append(before, before_scales, after, after_scales, kv_pre, ln_w, table, pos, starts, kind, eps=EPS, ckv_new=None):
    """Block by block against the definition.  fp32 on the way to 8 bits: a sum of 512 squares (21 roundings along the longest path), the mean,
    the root and three products: relative 2^-19 covers them; what is rounded to 8 bits may then be half a step off and that."""
    rel = 2.0 ** -19
    y = normed(kv_pre, ln_w, eps)
    want = as_f64(before).clone()
    tol = torch.zeros_like(want)
    scales = before_scales.double().clone()
    for s, p0 in enumerate(pos):
        p, end = p0, p0 + starts[s + 1] - starts[s]
        block = before.shape[1]
        while p0 >= 0 and p < end:
            stop = min(end, (p // block + 1) * block)
            lb = p // block
            b = -1 if lb >= table.shape[1] else int(table[s, lb])
            if 0 <= b < before.shape[0]:
                mine = y[starts[s] + p - p0:starts[s] + stop - p0]
                c = p % block
                need = float(mine.abs().max()) / TOP[kind]
                s0 = float(scales[b]) if c else 0.0
                now = max(need, s0)
                got = float(after_scales[b])
                if math.isfinite(now):
                    assert abs(got - now) <= rel * now, (s, lb, got, now)
                    kept = got == s0 or now == 0
                    assert kept or got > s0
                    if not kept:                             # (a need within rounding of s0 may go either way: `got` says)
                        want[b, :c] = want[b, :c] * (s0 / got)
                        tol[b, :c] = half_step(want[b, :c], kind) * (1 + rel) + want[b, :c].abs() * rel
                    want[b, c:c + stop - p] = mine / got if got else 0.0
                    # the largest value may round up by the scale's own rounding: saturated
                    tol[b, c:c + stop - p] = half_step(want[b, c:c + stop - p], kind) * (1 + rel) + want[b, c:c + stop - p].abs() * rel
                else:
                    assert math.isnan(got)
                    tol[b] = math.inf
                scales[b] = got
                if ckv_new is not None:
                    held = (as_f64(after[b, c:c + stop - p]) * got).half()
                    assert torch.equal(held, ckv_new[starts[s] + p - p0:starts[s] + stop - p0]) or math.isnan(got)
            p = stop
    assert torch.equal(scales[torch.isfinite(scales)], after_scales.double()[torch.isfinite(scales)]), "scales of other blocks"
    off = (as_f64(after) - want).abs()
    assert bool((off <= tol).all()), float((off - tol).max())


def visible(n, window, sinks):
    """positions that a row of n keys attends to"""
    p = torch.arange(max(n, 0), device="cuda")
    return p[(p >= n - window) | (p < sinks)] if window else p


def attend(q, keys, scale, rows16=False):
    """q [heads][512], keys [n][512] in 64 bits -> (output, what it may be off by).

    P and the output are rounded to fp16 (half a step is 2^-11 relative), scores are fp32 sums of 512 products scaled twice: with S the sum of
    magnitudes, 520 roundings at most of relative 2^-24 of it, which move a weight by as much relatively, and the normaliser too.  Weights
    below 2^-10 of the largest may be subnormal in fp16: 2^-25 absolute, times 16 where a block's scale is that much below the largest.
    rows16: the keys have been rounded to fp16 first, 2^-11 relative of each product of a score and of each value that is weighed."""
    if not keys.shape[0]:
        z = torch.zeros(q.shape[0], 512, dtype=torch.float64, device=q.device)
        return z, z
    s = q @ keys.T * scale
    p = torch.exp(s - s.amax(1, keepdim=True))
    tot = p.sum(1, keepdim=True)
    o, mag = p @ keys / tot, p @ keys.abs() / tot
    eta = (2.0 ** -24 * 520 + (2.0 ** -11 if rows16 else 0.0)) * (q.abs() @ keys.abs().T).amax(1, keepdim=True) * scale + 2.0 ** -20 * (1 + s.abs().amax(1, keepdim=True)) + keys.shape[0] * 2.0 ** -24
    small = (p < 2.0 ** -10).sum(1, keepdim=True) * 2.0 ** -25 * 16 * keys.abs().max() / tot
    return o, 2.0 ** -11 * (mag * (2 if rows16 else 1) + o.abs()) * 1.01 + 2 * eta * mag + small + 2.0 ** -25


def cache(gen, kind, n_blocks, block, spread=0.0):
    """random blocks; spread > 0: scales that differ by e^(+- spread)"""
    y = torch.randn(n_blocks, block, 512, device="cuda", generator=gen)
    if spread:
        y = y * torch.exp(spread * torch.randn(n_blocks, 1, 1, device="cuda", generator=gen))
    s = y.abs().amax((1, 2)) / TOP[kind]
    q = (y / s[:, None, None]).clamp(-TOP[kind], TOP[kind])
    return (q.round() if kind == "i8" else q).to(STORE[kind]), s


def table_for(gen, n_seqs, blocks, n_blocks):
    """[n_seqs][blocks] different blocks out of n_blocks"""
    return torch.randperm(n_blocks, device="cuda", generator=gen)[:n_seqs * blocks].to(torch.int32).view(n_seqs, blocks).contiguous()


def rows_of(ckv8, scales, table_row, p):
    """fp64 rows at positions p of a sequence; positions without a block are left out"""
    block = ckv8.shape[1]
    lb = p // block
    p, lb = p[lb < table_row.numel()], lb[lb < table_row.numel()]
    b = table_row[lb].long()
    ok = (b >= 0) & (b < ckv8.shape[0])
    b, p = b[ok], p[ok]
    raw = ckv8.view(torch.uint8)[b, p % block].view(ckv8.dtype)
    return as_f64(raw) * scales[b].double()[:, None]
