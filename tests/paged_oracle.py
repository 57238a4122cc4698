"""64-bit definitions (CPU, plain loops) of the rotary positions and of the paged int8 cache, and the
rounding bounds that the kernels are held to."""

import math

import torch

F64 = torch.float64
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}     # half a step, relative
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133, torch.float32: 2.0 ** -149}  # half a subnormal step
FLOOR = 2.0 ** -40


def rotate(x, positions, inv_freq, freq_axis=None, interleaved=False, inverse=False):
    """x [B, H, S, D], positions [S] / [B, S] / [axes, B, S] -> (y, |a| + |b| of every element's pair), fp64."""
    B, H, S, D = x.shape
    p = positions.to(F64)
    if p.dim() < 3:
        p = p.reshape(1, *((1, S) if p.dim() == 1 else p.shape))
    p = p.expand(p.shape[0], B, S)
    half = inv_freq.numel()
    axis = torch.zeros(half, dtype=torch.long) if freq_axis is None else freq_axis.long().clamp(max=p.shape[0] - 1)
    ang = p[axis].permute(1, 2, 0) * inv_freq.to(F64)                      # [B, S, half]
    if inverse:
        ang = -ang
    c, s = ang.cos().unsqueeze(1), ang.sin().unsqueeze(1)
    x = x.to(F64)
    y, size = x.clone(), torch.zeros_like(x)
    ia = torch.arange(0, 2 * half, 2) if interleaved else torch.arange(half)
    ib = ia + 1 if interleaved else ia + half
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    size[..., ia] = size[..., ib] = a.abs() + b.abs()
    return y, size


# cos / sin: 2 ulp each of a value <= 1 (2^-22), the reduced angle rounded to fp32 (pi 2^-24), three fp32
# roundings of the two-term sum (3 * 2^-24), all relative to |a| + |b|
ROTATE_ERR = 2.0 ** -22 + math.pi * 2.0 ** -24 + 3 * 2.0 ** -24


def rounded(y, dtype):
    """Half a step of ``dtype`` at the values y."""
    return y.abs() * U[dtype] + TINY[dtype]


def place_of(table, page, token, num_pages):
    """Page number and slot of a token, None where the cache has no such page."""
    j = token // page
    if j >= len(table) or not 0 <= table[j] < num_pages:
        return None
    return table[j], token % page


def dequant(codes, scale, table, n, first=0):
    """Tokens first .. first + n - 1 as fp64 [H, n, D], and which of them a page holds."""
    P, H, page, D = codes.shape
    out, there = torch.zeros(H, n, D, dtype=F64), torch.zeros(n, dtype=torch.bool)
    for i in range(n):
        at = place_of(table, page, first + i, P)
        if at is not None:
            out[:, i] = codes[at[0], :, at[1]].to(F64) * scale[at[0]].to(F64).unsqueeze(1)
            there[i] = True
    return out, there


def attend(q, k_i8, k_scale, v_i8, v_scale, table, lens, scale=None, causal=True, window=-1, query_lens=None,
           limit=None):
    """(out, tolerance) fp64 [B, Hq, M, D]; the tolerance bounds a kernel that splits q into two int8 planes (or
    takes it as it is), rounds the weights to fp16 against their maximum, sums in fp32 and
    rounds once at the end.  Keys at or past ``limit`` are not seen."""
    q_dt = q.dtype
    B, Hq, M, D = q.shape
    P, H, page, _ = k_i8.shape
    G = Hq // H
    scale = D ** -0.5 if scale is None else scale
    weight_err = U[torch.float16]
    out, tol = torch.zeros(B, Hq, M, D, dtype=F64), torch.zeros(B, Hq, M, D, dtype=F64)
    for b in range(B):
        row = table[b].tolist()
        total = max(0, int(lens[b]))
        m = M if query_lens is None else min(M, max(0, int(query_lens[b])))
        n = min(total, len(row) * page, total if limit is None else limit)
        if n == 0 or m == 0:
            continue
        K, there = dequant(k_i8, k_scale, row, n)
        V, _ = dequant(v_i8, v_scale, row, n)
        vs = torch.zeros(H, n, dtype=F64)
        for i in range(n):
            at = place_of(row, page, i, P)
            if at is not None:
                vs[:, i] = v_scale[at[0]].to(F64)
        key = torch.arange(n)
        for h in range(H):
            for gi in range(G):
                x = q[b, h * G + gi, :m].to(F64)
                logit = x @ K[h].t() * scale
                pos = (total - m + torch.arange(m)).unsqueeze(1)
                seen = there & (vs[h] != 0) & torch.ones(m, 1, dtype=torch.bool)
                if causal:
                    seen = seen & (key <= pos)
                if window >= 0:
                    seen = seen & (key > pos - window)
                logit = logit.masked_fill(~seen, -math.inf)
                p = torch.softmax(logit, -1)
                p = torch.where(seen.any(1, keepdim=True), p, torch.zeros_like(p))
                o = p @ V[h]
                # q: half a step of amax / 16256 per channel, and fp32 roundings of scale and logit (2^-21)
                amax = x.abs().amax(1, keepdim=True)
                size = torch.where(seen, logit.abs(), torch.zeros_like(p)).amax(1, keepdim=True)
                ell = abs(scale) * amax / 32512 * K[h].abs().sum(1).max() + size * 2.0 ** -21 + 2.0 ** -20
                # weights: their 16-bit rounding, exponential and sums in fp32 (2^-18 covers a few thousand terms)
                rel = torch.expm1(2 * ell) + weight_err + 2.0 ** -18
                big = (p * vs[h]).amax(1, keepdim=True)
                code = torch.where(vs[h] > 0, 1 / vs[h], torch.zeros_like(vs[h])).unsqueeze(1) * V[h].abs()
                t = rel * (p @ V[h].abs()) + big * 2.0 ** -24 * code.sum(0)
                out[b, h * G + gi, :m] = o
                tol[b, h * G + gi, :m] = t + (o.abs() + t) * U[q_dt] + TINY[q_dt]
    return out, tol


def append(x, codes, scale, table, lens, new):
    """What an append of x fp64 [B, H, M, D] may leave: {(page, head): (exact codes fp64 of its slots [n, D],
    its scale, slots written)} from the pools before the call."""
    P, H, page, D = codes.shape
    got = {}
    for b in range(x.shape[0]):
        row = table[b].tolist()
        start = int(lens[b]) - int(new[b])
        tokens = [i for i in range(int(new[b])) if start + i >= 0 and place_of(row, page, start + i, P) is not None]
        for pg in sorted({place_of(row, page, start + i, P)[0] for i in tokens}):
            mine = [i for i in tokens if place_of(row, page, start + i, P)[0] == pg]
            slots = [(start + i) % page for i in mine]
            older = slots[0]
            for h in range(H):
                fresh = x[b, h, mine]
                was = float(scale[pg, h]) if older > 0 else 0.0
                now = max(was, float(fresh.abs().max()) / 127, FLOOR)
                keep = codes[pg, h, :older].to(F64) * (was / now)
                got[pg, h] = (torch.cat([keep, fresh / now]), now, older, slots)
    return got


def pages_for(lens, page, spare=2, seed=0, width=None):
    """A shuffled block table [B, width] int32 (unused entries -1) and the number of pages of its pool."""
    need = [max(0, -(-int(n) // page)) for n in lens]
    pool = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    width = (max(need) + 1) if width is None else width
    table = torch.full((len(need), width), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        n = min(n, width)
        table[b, :n] = torch.tensor([pool.pop() for _ in range(n)], dtype=torch.int32)
    return table, sum(need) + spare


def random_cache(pages, H, page, D, seed=0):
    g = torch.Generator().manual_seed(seed)
    codes = [(torch.randn(pages, H, page, D, generator=g) * 35).round().clamp(-127, 127).to(torch.int8) for _ in "kv"]
    scales = [(2 + 4 * torch.rand(pages, H, generator=g)) / 127 for _ in "kv"]
    return codes[0], scales[0], codes[1], scales[1]
