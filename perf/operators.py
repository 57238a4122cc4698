"""Measured cases of the paged 8-bit K/V cache and of the position rotation that feeds it.

Three operators, as a serving or training program calls them:

* ``rope``    rotary positions with one or several axes on q and k, forward and backward (``apply_rope``);
* ``append``  new keys and values go into the pages of an int8 cache with one scale per page and KV head,
              rotated on the way (``kv_append_paged``); what the call may have changed is read back as
              16-bit values (``kv_read_paged``), with the scales;
* ``attend``  attention of one or many query tokens per sequence over that cache (``attn_paged_cached``).

``own = False`` computes them from elementary torch operations, ``own = True`` through the package.

The cache: codes int8 [pages, KV heads, page_size, D] and scales fp32 [pages, KV heads] for K and for V;
``table`` int32 [B, pages per sequence]; ``lens`` int32 [B], the tokens of every sequence with the new ones.
A page of one head stands for code * scale.  An append gives a page the scale
max(old scale if it holds older tokens, max |new| / 127, 2^-40); new codes are round(x / scale), and the
codes of the older tokens of that page become round(code * old scale / new scale).
"""

import math

import torch

own = False

_DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_FLOOR = 2.0 ** -40


def listed():
    rope = dict(op="rope", base=10000.0, axes=1, mixed=False, pos0=0)
    append = dict(op="append", base=500000.0, axes=1, mixed=False, interleaved=False)
    attend = dict(op="attend", causal=True, window=-1)
    return [
        # one decode step's q and k of a batch of 16, far into their sequences: latency
        dict(rope, name="rope decode B16 bf16", B=16, Hq=32, Hkv=8, S=1, D=128, rot=128, dtype="bf16", interleaved=False,
             pos0=100000, backward=False),
        # a training step on a 4096-token sequence with image tokens: time, height and width axes
        dict(rope, name="rope train S4096 3 axes bf16", B=1, Hq=32, Hkv=8, S=4096, D=128, rot=128, dtype="bf16",
             interleaved=False, axes=3, backward=True),
        # a large prompt batch, neighbouring channels paired
        dict(rope, name="rope prompts B4 S8192 fp16", B=4, Hq=64, Hkv=8, S=8192, D=128, rot=128, dtype="fp16",
             interleaved=True, backward=False),
        # a single conversation's decode step: latency
        dict(append, name="append 1 token B1 fp16", B=1, Hq=8, Hkv=2, M=1, lo=1000, hi=1000, D=128, rot=128, page=16,
             dtype="fp16"),
        # a serving batch's decode step, every page at another fill
        dict(append, name="append 1 token B128 fp16", B=128, Hq=64, Hkv=8, M=1, lo=33, hi=512, D=128, rot=128, page=16,
             dtype="fp16"),
        # a prompt entering an empty cache
        dict(append, name="append prompt 4096 bf16", B=1, Hq=32, Hkv=8, M=4096, lo=4096, hi=4096, D=128, rot=128, page=64,
             dtype="bf16"),
        # ragged prompt pieces with image tokens behind earlier ones, half of the channels rotated
        dict(append, name="append ragged 777 3 axes bf16", B=8, Hq=16, Hkv=4, M=777, lo=100, hi=2048, D=64, rot=32, page=32,
             dtype="bf16", axes=3, mixed=True),
        # one short conversation: latency
        dict(attend, name="attend 1 token B1 N1024 fp16", B=1, Hq=8, Hkv=2, M=1, lo=1024, hi=1024, D=128, page=16,
             dtype="fp16"),
        # multi-query attention over ragged lengths, small heads
        dict(attend, name="attend 1 token B8 MQA D64 bf16", B=8, Hq=16, Hkv=1, M=1, lo=100, hi=2048, D=64, page=32,
             dtype="bf16"),
        # a serving batch of long ragged contexts
        dict(attend, name="attend 1 token B64 N32768 fp16", B=64, Hq=64, Hkv=8, M=1, lo=1024, hi=32768, D=128, page=64,
             dtype="fp16"),
        # up to five drafted tokens per sequence, checked in one call
        dict(attend, name="attend 5 tokens B16 N8192 bf16", B=16, Hq=32, Hkv=8, M=5, lo=700, hi=8192, D=128, page=16,
             dtype="bf16"),
        # a prompt's next 1024 tokens behind 8192 cached ones
        dict(attend, name="attend 1024 tokens N9216 fp16", B=2, Hq=32, Hkv=8, M=1024, lo=9001, hi=9216, D=128, page=128,
             dtype="fp16"),
    ]


def draw(rng):
    def span(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["rope", "append", "attend", "attend"])
    heads = rng.choice([(8, 2), (16, 1), (32, 8), (64, 8), (12, 4), (6, 6), (28, 4)])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "rope":
        D = rng.choice([32, 64, 72, 80, 128, 256])
        B = span(1, 8)
        S = span(1, max(1, min(8192, 200_000_000 // (B * sum(heads) * D))))
        return dict(op=op, B=B, Hq=heads[0], Hkv=heads[1], S=S, D=D, rot=rng.choice([D, D // 2]),
                    dtype=rng.choice([dtype, dtype, "fp32"]), interleaved=rng.random() < 0.5, axes=rng.choice([1, 2, 3]),
                    mixed=rng.random() < 0.5, base=rng.choice([10000.0, 1000000.0]), pos0=span(1, 1000000),
                    backward=rng.random() < 0.5)
    D, page = rng.choice([32, 64, 128, 128, 256]), rng.choice([16, 32, 64, 128, 256])
    if op == "append":
        M = rng.choice([1, 1, span(2, 9), span(10, 2048)])
        B = span(1, max(1, min(128, 4096 // M)))
        lo = span(1, 700)
        return dict(op=op, B=B, Hq=heads[0], Hkv=heads[1], M=M, lo=lo, hi=lo + span(1, 1400) + M, D=D,
                    rot=rng.choice([D, D // 2]), page=page, dtype=dtype, axes=rng.choice([1, 3]),
                    mixed=rng.random() < 0.5, interleaved=rng.random() < 0.5, base=rng.choice([10000.0, 500000.0]))
    M = rng.choice([1, 1, span(2, 9), span(10, 1000)])
    hi = span(1, 32768 if M < 10 else 8192)
    B = span(1, max(1, min(64, 2_000_000_000 // (hi * heads[1] * D * 2), 1_000_000_000 // (heads[0] * M * hi))))
    return dict(op=op, B=B, Hq=heads[0], Hkv=heads[1], M=M, lo=rng.randint(1, hi), hi=hi, D=D, page=page, dtype=dtype,
                causal=rng.random() < 0.8, window=rng.choice([-1, -1, span(1, 4096)]))


def _spread(lo, hi, n):
    """n whole numbers over [lo, hi], the first of them hi, in no order (golden-ratio steps)."""
    return [hi - int((hi - lo + 1) * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]


def _lens(case):
    """Per sequence: tokens in the cache with the new ones, and how many of them are new."""
    lens = _spread(case["lo"], case["hi"], case["B"])
    new = [min(m, n) for m, n in zip(_spread(max(1, case["M"] // 3), case["M"], case["B"]), lens)]
    return lens, new


def _window(case):
    """Tokens read back behind an append: the new ones and whatever shares a page with them."""
    return case["M"] + case["page"] - 1


def work(case):
    if case["op"] == "rope":
        e = 4 if case["dtype"] == "fp32" else 2
        n = case["B"] * (case["Hq"] + case["Hkv"]) * case["S"] * case["D"]
        passes = 2 if case["backward"] else 1
        return {"bytes": passes * (2 * n * e + 8 * case["axes"] * case["B"] * case["S"]), "flops": passes * 3 * n}
    lens, new = _lens(case)
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if case["op"] == "append":
        rows = sum(new)
        back = sum(min(n, _window(case)) for n in lens)
        rotate = rows * D * (2 * 2 * Hq + 2 * 2 * Hkv)          # q read and written, k and v read
        store = rows * D * 2 * Hkv                                 # the codes
        read = back * D * Hkv * 2 + case["B"] * Hkv * _window(case) * D * 2 * 2   # codes read, 16-bit rows written
        return {"bytes": rotate + store + read, "flops": rows * D * (3 * Hq + 8 * Hkv)}
    keys = sum(min(n, n if case["window"] < 0 else case["window"] + m) for n, m in zip(lens, new))
    pairs = 0
    for n, m in zip(lens, new):
        for i in range(m):
            top = n - m + i + 1 if case["causal"] else n
            low = max(0, n - m + i + 1 - case["window"]) if case["window"] >= 0 else 0
            pairs += max(0, top - low)
    rows = case["B"] * case["M"]
    return {"bytes": keys * Hkv * 2 * D + 8 * Hkv * keys // case["page"] + rows * Hq * D * 2 * 2, "flops": 4 * Hq * D * pairs}


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    B, Hq, Hkv, D, dt = case["B"], case["Hq"], case["Hkv"], case["D"], _DT[case["dtype"]]
    st = dict(case=case, dt=dt)

    def normal(*shape):
        return torch.randn(*shape, device=dev, dtype=torch.float32, generator=g).to(dt)

    if case["op"] != "attend":
        half = case["rot"] // 2
        st["inv_freq"] = (case["base"] ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)).float()
        i = torch.arange(half, device=dev)
        A = case["axes"]
        st["freq_axis"] = None if A == 1 else ((i % A) if case["mixed"] else (i * A // max(half, 1))).to(torch.uint8)
    if case["op"] == "rope":
        S, A = case["S"], case["axes"]
        jump = torch.randint(0, 50, (B, 1), device=dev, generator=g)
        i = torch.arange(S, device=dev).unsqueeze(0) + jump + case["pos0"]
        # several axes: frames of 16 x 24 patches (time, height, width)
        grid = [i, case["pos0"] + (i // 24) % 16, case["pos0"] + i % 24]
        st["positions"] = i if A == 1 else torch.stack(grid[:A])
        st["q"], st["k"] = normal(B, Hq, S, D), normal(B, Hkv, S, D)
        if case["backward"]:
            st["gq"], st["gk"] = normal(B, Hq, S, D), normal(B, Hkv, S, D)
            st["q"].requires_grad_(True)
            st["k"].requires_grad_(True)
        return st

    M, page = case["M"], case["page"]
    lens, new = _lens(case)
    per = -(-max(lens) // page) + 1
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, device=dev, generator=g).to(torch.int32)
    held = torch.zeros(B, per, dtype=torch.bool)
    for b, n in enumerate(need):
        held[b, :n] = True
    table = torch.zeros(B, per, dtype=torch.int32, device=dev)
    table[held.to(dev)] = order[:sum(need)]
    st["table"], st["lens"], st["max_len"] = table, torch.tensor(lens, dtype=torch.int32, device=dev), max(lens)
    st["new"] = torch.tensor(new, dtype=torch.int32, device=dev)
    for name in ("k", "v"):
        codes = torch.empty(pages, Hkv, page, D, dtype=torch.int8, device=dev)
        codes.view(-1).copy_((torch.randn(codes.numel(), device=dev, dtype=torch.float16, generator=g) * 35).round_().clamp_(-127, 127))
        st[name + "_i8"] = codes
        # scales of pages whose largest value lies between two and six of the values' own size
        st[name + "_scale"] = (2 + 4 * torch.rand(pages, Hkv, device=dev, generator=g)) / 127
    # the projections' outputs, token-major as a model's linear layers leave them
    st["q"] = normal(B, M, Hq, D).transpose(1, 2)
    if case["op"] == "attend":
        return st
    st["k"], st["v"] = normal(B, M, Hkv, D).transpose(1, 2), normal(B, M, Hkv, D).transpose(1, 2)
    at = st["lens"].long().unsqueeze(1) - st["new"].long().unsqueeze(1) + torch.arange(M, device=dev)
    st["positions"] = at if case["axes"] == 1 else torch.stack([at, 7 + (at // 24) % 16, 7 + at % 24])
    st["first"] = (st["lens"] - _window(case)).clamp_(min=0)
    return st


def _angles(positions, inv_freq, freq_axis):
    """cos and sin fp32 [B, S, rot / 2]; the angles themselves in 64 bits (far positions)."""
    p = positions.double()
    if freq_axis is None:
        turn = p.unsqueeze(-1) * inv_freq.double()
    else:
        turn = p.movedim(0, -1)[..., freq_axis.long()] * inv_freq.double()
    return turn.cos().float(), turn.sin().float()


def _rotate(x, cos, sin, interleaved):
    """fp32 rotation of x [B, H, S, D] by cos / sin [B, S, rot / 2]; channels from rot on stay."""
    x, cos, sin = x.float(), cos.unsqueeze(1), sin.unsqueeze(1)
    half = cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, x[..., 2 * half:]], -1)


def _rope(st):
    c = st["case"]
    if own:
        import superl8_b200 as s8
        q, k = s8.apply_rope(st["q"], st["k"], st["positions"], st["inv_freq"], freq_axis=st["freq_axis"],
                             interleaved=c["interleaved"])
        if not c["backward"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["gq"], st["gk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
    with torch.no_grad():
        cos, sin = _angles(st["positions"], st["inv_freq"], st["freq_axis"])
        got = {n: _rotate(st[n], cos, sin, c["interleaved"]).to(st["dt"]) for n in ("q", "k")}
        if c["backward"]:   # the rotation is orthogonal: its gradient is the rotation by the opposite angle
            got |= {"d" + n: _rotate(st["g" + n], cos, -sin, c["interleaved"]).to(st["dt"]) for n in ("q", "k")}
    return got


def _append_one(x, codes, scale, slots, new_at, is_new, is_old, touched):
    """Plain append of x fp32 [B, H, M, D] to one pool (codes and scale are updated in place)."""
    B, H, _, D = x.shape
    P = slots.shape[1]
    page = codes.shape[2]
    rows = torch.gather(x, 2, new_at[:, None, :, None].expand(B, H, P * page, D))
    rows = rows.view(B, H, P, page, D).transpose(1, 2)                      # [B, P, H, page, D]
    fresh, kept = is_new.view(B, P, 1, page, 1), is_old.view(B, P, 1, page, 1)
    top = torch.where(fresh, rows.abs(), torch.zeros_like(rows)).amax((-1, -2))     # [B, P, H]
    old = torch.where(kept.any(3).squeeze(-1), scale[slots], torch.zeros_like(top))
    now = torch.maximum(torch.maximum(old, top / 127), torch.full_like(top, _FLOOR))
    was = codes[slots]
    again = (was.float() * (old / now)[..., None, None]).round()
    put = torch.where(fresh, (rows / now[..., None, None]).round().clamp(-127, 127), torch.where(kept, again, was.float()))
    codes[slots[touched]] = put[touched].to(torch.int8)
    scale[slots[touched]] = now[touched]


def _read_one(codes, scale, table, lens, first, count, dt):
    """Rows first .. first + count - 1 of every sequence as 16-bit values [B, H, count, D], zero behind its end."""
    page = codes.shape[2]
    at = first.long().unsqueeze(1) + torch.arange(count, device=codes.device)
    there = at < lens.long().unsqueeze(1)
    slot = torch.gather(table.long(), 1, (at // page).clamp(max=table.shape[1] - 1))
    rows = codes[slot, :, at % page].float() * scale[slot].unsqueeze(-1)    # [B, count, H, D]
    return torch.where(there[..., None, None], rows, torch.zeros_like(rows)).transpose(1, 2).to(dt)


def _append(st):
    c = st["case"]
    cache = (st["k_i8"], st["k_scale"], st["v_i8"], st["v_scale"])
    count = _window(c)
    if own:
        import superl8_b200 as s8
        q = s8.kv_append_paged(st["k"], st["v"], *cache, st["table"], st["lens"], new_lens=st["new"], q=st["q"],
                               positions=st["positions"], inv_freq=st["inv_freq"], freq_axis=st["freq_axis"],
                               interleaved=c["interleaved"])
        k, v = s8.kv_read_paged(*cache, st["table"], st["lens"], count, first=st["first"], dtype=st["dt"])
    else:
        page, M = c["page"], c["M"]
        lens, new = st["lens"].long(), st["new"].long()
        cos, sin = _angles(st["positions"], st["inv_freq"], st["freq_axis"])
        real = (torch.arange(M, device=lens.device) < new.unsqueeze(1))[:, None, :, None]
        q = _rotate(st["q"], cos, sin, c["interleaved"])
        q = torch.where(real, q, torch.zeros_like(q)).to(st["dt"])
        P = (M + page - 2) // page + 1
        p0 = (lens - new) // page
        which = p0.unsqueeze(1) + torch.arange(P, device=lens.device)
        touched = which * page < lens.unsqueeze(1)
        slots = torch.gather(st["table"].long(), 1, which.clamp(max=st["table"].shape[1] - 1))
        at = (p0 * page).unsqueeze(1) + torch.arange(P * page, device=lens.device)
        i = at - (lens - new).unsqueeze(1)
        is_new, is_old = (i >= 0) & (i < new.unsqueeze(1)), i < 0
        i = i.clamp(0, M - 1)
        _append_one(_rotate(st["k"], cos, sin, c["interleaved"]), cache[0], cache[1], slots, i, is_new, is_old, touched)
        _append_one(st["v"].float(), cache[2], cache[3], slots, i, is_new, is_old, touched)
        k = _read_one(cache[0], cache[1], st["table"], st["lens"], st["first"], count, st["dt"])
        v = _read_one(cache[2], cache[3], st["table"], st["lens"], st["first"], count, st["dt"])
    return {"q": q, "k": k, "v": v, "k_scale": st["k_scale"], "v_scale": st["v_scale"]}


def _attend(st):
    c = st["case"]
    if own:
        import superl8_b200 as s8
        return s8.attn_paged_cached(st["q"], st["k_i8"], st["k_scale"], st["v_i8"], st["v_scale"], st["table"], st["lens"],
                                    causal=c["causal"], window_left=c["window"], query_lens=st["new"],
                                    max_context_len=st["max_len"])
    q, lens, new = st["q"].float(), st["lens"].long(), st["new"].long()
    B, Hq, M, D = q.shape
    H, page = st["k_i8"].shape[1:3]
    slots = st["table"].long()[:, :-(-st["max_len"] // page)]
    N = slots.shape[1] * page
    k = (st["k_i8"][slots].float() * st["k_scale"][slots][..., None, None]).transpose(1, 2).reshape(B, H, N, D)
    s = torch.matmul(q.reshape(B, H, Hq // H * M, D), k.transpose(2, 3)).view(B, Hq, M, N) / math.sqrt(D)
    del k
    row = torch.arange(M, device=q.device)
    pos = (lens - new).unsqueeze(1) + row                                  # [B, M]
    key = torch.arange(N, device=q.device)
    seen = (key < lens[:, None, None]) & (row < new.unsqueeze(1)).unsqueeze(2)
    if c["causal"]:
        seen = seen & (key <= pos.unsqueeze(2))
    if c["window"] >= 0:
        seen = seen & (key > pos.unsqueeze(2) - c["window"])
    s = torch.where(seen.unsqueeze(1), s, torch.full((), -math.inf, device=q.device))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    del s
    total = p.sum(-1, keepdim=True)
    v = (st["v_i8"][slots].float() * st["v_scale"][slots][..., None, None]).transpose(1, 2).reshape(B, H, N, D)
    o = torch.matmul(p.view(B, H, Hq // H * M, N), v).view(B, Hq, M, D)
    return (o / torch.where(total == 0, torch.ones_like(total), total)).to(st["dt"])


def run(state):
    return {"rope": _rope, "append": _append, "attend": _attend}[state["case"]["op"]](state)


def exact(case, seed):
    st = prepare(case, seed)
    f64 = torch.float64

    def turned(x, pos, back=False):
        """x [H, S, D] by complex multiplication, pos [axes, S]."""
        freq = st["inv_freq"].to(f64)
        axis = torch.zeros(freq.numel(), dtype=torch.long, device=freq.device) if st["freq_axis"] is None else st["freq_axis"].long()
        angle = pos.to(f64)[axis].t() * freq * (-1 if back else 1)
        unit = torch.polar(torch.ones_like(angle), angle)
        x = x.detach().to(f64)
        r = 2 * freq.numel()
        if case["interleaved"]:
            pair = torch.complex(x[..., 0:r:2], x[..., 1:r:2]) * unit
            y = torch.view_as_real(pair).reshape(*x.shape[:-1], r)
        else:
            pair = torch.complex(x[..., :r // 2], x[..., r // 2:r]) * unit
            y = torch.cat([pair.real, pair.imag], -1)
        return torch.cat([y, x[..., r:]], -1)

    def places(b):
        p = st["positions"]
        return p[:, b] if case["axes"] > 1 else p[b].unsqueeze(0)

    if case["op"] == "rope":
        got = {n: torch.stack([turned(st[n][b], places(b)) for b in range(case["B"])]) for n in ("q", "k")}
        if case["backward"]:
            got |= {"d" + n: torch.stack([turned(st["g" + n][b], places(b), True) for b in range(case["B"])]) for n in ("q", "k")}
        return got

    lens, new = _lens(case)
    page, D, B, M = case["page"], case["D"], case["B"], case["M"]
    table = st["table"].long().cpu().tolist()
    if case["op"] == "attend":
        out = torch.zeros(st["q"].shape, dtype=f64, device="cuda")
        share = case["Hq"] // case["Hkv"]
        for b in range(B):
            n, m = lens[b], new[b]
            ids = torch.tensor(table[b][:-(-n // page)], device="cuda")
            for h in range(case["Hkv"]):
                K = (st["k_i8"][ids, h].to(f64) * st["k_scale"][ids, h].to(f64)[:, None, None]).reshape(-1, D)[:n]
                V = (st["v_i8"][ids, h].to(f64) * st["v_scale"][ids, h].to(f64)[:, None, None]).reshape(-1, D)[:n]
                logit = st["q"][b, h * share:(h + 1) * share, :m].to(f64) @ K.t() * D ** -0.5
                here, there = torch.arange(n, device="cuda"), torch.arange(n - m, n, device="cuda").unsqueeze(1)
                hidden = torch.zeros(m, n, dtype=torch.bool, device="cuda")
                if case["causal"]:
                    hidden |= here > there
                if case["window"] >= 0:
                    hidden |= here <= there - case["window"]
                weight = torch.softmax(logit.masked_fill(hidden, -math.inf), -1).nan_to_num(0.0)
                out[b, h * share:(h + 1) * share, :m] = weight @ V
        return out

    count = _window(case)
    got = {"q": torch.zeros(st["q"].shape, dtype=f64, device="cuda")}
    for b in range(B):
        got["q"][b, :, :new[b]] = turned(st["q"][b], places(b))[:, :new[b]]
    first = st["first"].cpu().tolist()
    for name in ("k", "v"):
        scale = st[name + "_scale"].to(f64)
        back = torch.zeros(B, case["Hkv"], count, D, dtype=f64, device="cuda")
        for b in range(B):
            x = turned(st["k"][b], places(b)) if name == "k" else st["v"][b].to(f64)
            start = lens[b] - new[b]
            for j in range(-(-lens[b] // page)):
                lo, hi = j * page, min(lens[b], (j + 1) * page)
                if hi <= first[b]:
                    continue
                slot = table[b][j]
                held = st[name + "_i8"][slot, :, :hi - lo].to(f64)          # [H, tokens, D]
                s = scale[slot].clone()
                if hi > start:
                    cut = max(0, start - lo)
                    fresh = x[:, max(0, lo - start):hi - start]
                    was = s.clone() if cut else torch.zeros_like(s)
                    s = torch.maximum(was, fresh.abs().amax((1, 2)) / 127).clamp(min=_FLOOR)
                    held = torch.cat([(held[:, :cut] * (was / s)[:, None, None]).round(),
                                      (fresh / s[:, None, None]).round().clamp(-127, 127)], 1)
                    scale[slot] = s
                lo2 = max(lo, first[b])
                back[b, :, lo2 - first[b]:hi - first[b]] = held[:, lo2 - lo:] * s[:, None, None]
        got[name], got[name + "_scale"] = back, scale
    return got
