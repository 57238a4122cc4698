"""The paged int8 cache against its definition in 64 bits: append (scales, requantised codes, what must stay
untouched), read back, attention from one to many query tokens, and a serving loop of all of them."""

import math

import pytest
import torch

import paged_oracle as po
import superl8_b200 as s8
from superl8_b200 import _C, _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["compiled", "ctypes"])
def binding(request):
    if request.param == "compiled" and _C._ext is None:
        pytest.skip("the compiled extension is not built")
    prev = _C.use_binding(request.param)
    yield
    _C.use_binding(prev)


def on(device, *ts):
    return [t.to(device) for t in ts]


def freqs(rot, base=10000.0):
    return (base ** (-torch.arange(rot // 2, dtype=torch.float64) / (rot // 2))).float()


# ---- append ----

APPEND = [  # Hq, Hkv, M, D, rot, page, dtype, axes, interleaved, lens, new
    (8, 2, 1, 128, 128, 16, torch.float16, 1, False, [1, 16, 17, 40], [1, 1, 1, 1]),
    (4, 4, 1, 64, 32, 64, torch.bfloat16, 1, True, [65, 64, 1], [1, 1, 0]),
    (4, 1, 37, 32, 32, 16, torch.float16, 3, False, [37, 100, 20, 5], [37, 37, 11, 0]),
    (6, 3, 130, 128, 64, 64, torch.bfloat16, 3, True, [130, 300, 129], [130, 77, 128]),
    (2, 1, 300, 256, 256, 128, torch.float16, 1, False, [300, 429], [300, 300]),
    (2, 1, 260, 256, 256, 256, torch.bfloat16, 1, True, [270], [260]),
    (2, 2, 9, 64, 0, 32, torch.float16, 1, False, [9, 40], [9, 8]),
]


@pytest.mark.parametrize("case", APPEND)
def test_append_against_definition(device, binding, case):
    Hq, Hkv, M, D, rot, page, dtype, axes, interleaved, lens, new = case
    B = len(lens)
    g = torch.Generator().manual_seed(M + D)
    table, pages = po.pages_for(lens, page, seed=M)
    cache = po.random_cache(pages, Hkv, page, D, seed=D)
    # token-major projections, some large values so that some scales grow and some do not
    q, k, v = (torch.randn(B, M, H, D, generator=g).to(dtype).transpose(1, 2) for H in (Hq, Hkv, Hkv))
    k[0] *= 3
    lens_t, new_t = torch.tensor(lens, dtype=torch.int32), torch.tensor(new, dtype=torch.int32)
    place = (lens_t - new_t).long().unsqueeze(1) + torch.arange(M)
    pos, axis = place, None
    if axes == 3:
        pos = torch.stack([place, place // 7 % 11, place % 7])
        axis = s8.rope_freq_axis([rot // 2 // 4, rot // 2 // 4, rot // 2 - 2 * (rot // 2 // 4)])
    dev = on(device, *cache)
    args = dict(new_lens=new_t.to(device))
    if rot:
        inv = freqs(rot)
        args.update(q=q.to(device), inv_freq=inv.to(device), interleaved=interleaved)
        if axes == 3:
            args.update(positions=pos.to(device), freq_axis=axis.to(device))
        kr, size = po.rotate(k, pos, inv, axis, interleaved)
        qr, q_size = po.rotate(q, pos, inv, axis, interleaved)
    else:
        kr, size = k.double(), torch.zeros(k.shape, dtype=po.F64)
    out = s8.kv_append_paged(k.to(device), v.to(device), *dev, table.to(device), lens_t.to(device), **args)
    if rot:
        tol = q_size * po.ROTATE_ERR
        tol = tol + po.rounded(qr.abs() + tol, dtype)
        real = (torch.arange(M) < new_t.unsqueeze(1))[:, None, :, None]
        assert out.shape == q.shape and (out.cpu().double() - qr * real).abs().le(tol).all()
        assert (out.cpu()[~real.expand_as(q)] == 0).all()
    else:
        assert out is None
    for name, x, err, codes, scale, codes_dev, scale_dev in (("k", kr, size.max().item() * po.ROTATE_ERR, cache[0], cache[1], dev[0], dev[1]),
                                                             ("v", v.double(), 0.0, cache[2], cache[3], dev[2], dev[3])):
        want = po.append(x, codes, scale, table, lens, new)
        left_codes, left_scale = codes.clone(), scale.clone()
        got_codes, got_scale = codes_dev.cpu(), scale_dev.cpu()
        for (pg, h), (exact, now, older, slots) in want.items():
            s = float(got_scale[pg, h])
            assert abs(s - now) <= now * 2.0 ** -22 + err / 127, name
            # a code is its value over the scale, rounded: half a step, the fp32 of the quotient (127 * 2^-22),
            # and what the rotation and the scale are off by
            slack = 0.5 + 127 * 2.0 ** -21 + 2 * err / now
            assert (got_codes[pg, h, :slots[-1] + 1].double() - exact).abs().max() <= slack, name
            left_codes[pg, h, :slots[-1] + 1] = got_codes[pg, h, :slots[-1] + 1]
            left_scale[pg, h] = s
            if s == float(scale[pg, h]) and older:    # the scale did not grow: the older codes are the same bits
                assert torch.equal(got_codes[pg, h, :older], codes[pg, h, :older]), name
        assert torch.equal(got_codes, left_codes) and torch.equal(got_scale, left_scale), f"{name}: something else was written"


def test_append_places_and_pages_that_do_not_exist(device, binding):
    """Tokens before the sequence, past the table, on page -1 or past the pool: skipped, the rest is stored."""
    Hkv, D, page, pages = 2, 64, 16, 5
    table = torch.tensor([[0, 1, 2], [3, -1, 4], [7, 3, 2]], dtype=torch.int32)
    table[2, 0], table[2, 1], table[2, 2] = pages, -5, 2**31 - 1
    lens, new = torch.tensor([60, 40, 33], dtype=torch.int32), torch.tensor([20, 40, 33], dtype=torch.int32)
    k = torch.randn(3, Hkv, 40, D, generator=torch.Generator().manual_seed(1)).half()
    cache = po.random_cache(pages, Hkv, page, D)
    dev = on(device, *cache)
    s8.kv_append_paged(*on(device, k, k), *dev, table.to(device), lens.to(device), new_lens=new.to(device))
    want = po.append(k.double(), cache[0], cache[1], table, lens, new)
    assert {p for p, _ in want} == {2, 3, 4}
    got, scale = dev[0].cpu(), dev[1].cpu()
    for pg in range(pages):
        for h in range(Hkv):
            if (pg, h) not in want:
                assert torch.equal(got[pg, h], cache[0][pg, h]) and scale[pg, h] == cache[1][pg, h]
                continue
            exact, now, older, slots = want[pg, h]
            assert abs(float(scale[pg, h]) - now) <= now * 2.0 ** -22
            assert (got[pg, h, :slots[-1] + 1].double() - exact).abs().max() <= 0.5 + 127 * 2.0 ** -21
            assert torch.equal(got[pg, h, slots[-1] + 1:], cache[0][pg, h, slots[-1] + 1:])
    # more new tokens than the sequence has: the last ones are stored from place 0 on
    dev = on(device, *po.random_cache(pages, Hkv, page, D))
    s8.kv_append_paged(*on(device, k[:1], k[:1]), *dev, table[:1].to(device), torch.tensor([5], dtype=torch.int32, device=device))
    read, _ = s8.kv_read_paged(*dev, table[:1].to(device), torch.tensor([5], dtype=torch.int32, device=device), 5)
    assert (read.cpu().float() - k[:1, :, 35:40].float()).abs().max() <= 0.51 * k[0, :, 35:40].abs().max().item() / 127 + 2.0 ** -11 * 4


def test_append_zeros_and_what_is_not_finite(device):
    """A page of zeros gets the smallest scale and grows out of it; NaN and infinity poison their page only."""
    D, page = 64, 16
    dev = s8.empty_paged_cache(3, 1, page, D, device)
    table = torch.tensor([[2, 1]], dtype=torch.int32, device=device)
    z = torch.zeros(1, 1, 4, D, device=device, dtype=torch.float16)
    lens = torch.tensor([4], dtype=torch.int32, device=device)
    s8.kv_append_paged(z, z, *dev, table, lens)
    assert float(dev[1][2]) == 2.0 ** -40 and (dev[0] == 0).all()
    x = torch.full((1, 1, 1, D), 0.5, device=device, dtype=torch.float16)
    s8.kv_append_paged(x, x, *dev, table, lens + 1)
    assert abs(float(dev[1][2]) - 0.5 / 127) <= 2.0 ** -30 and (dev[0][2, 0, 4] == 127).all() and (dev[0][2, 0, :4] == 0).all()
    for poison in (float("nan"), float("inf"), -float("inf")):
        bad = x.clone()
        bad[..., 7] = poison
        pool = [t.clone() for t in dev]
        s8.kv_append_paged(bad, x, *pool, table, lens + 2)
        assert not math.isfinite(float(pool[1][2])) and math.isfinite(float(pool[3][2]))
        s8.kv_append_paged(x, x, *pool, table, lens + 3)       # what comes later does not hide it
        assert not math.isfinite(float(pool[1][2]))
        q = torch.ones(1, 1, 1, D, device=device, dtype=torch.float16)
        assert torch.isnan(s8.attn_paged_cached(q, *pool, table, lens + 3).float()).all()
        assert torch.isfinite(s8.attn_paged_cached(q, *dev, table, lens + 1).float()).all()


def test_append_infinity_alone_in_its_page(device):
    """What is not finite makes its page NaN whatever the signs: also as the page's only token, and read back."""
    D, page = 64, 16
    table = torch.tensor([[1]], dtype=torch.int32, device=device)
    lens = torch.tensor([1], dtype=torch.int32, device=device)
    x = torch.full((1, 1, 1, D), 0.5, device=device, dtype=torch.float16)
    q = torch.ones(1, 2, 1, D, device=device, dtype=torch.float16)
    q[0, 1] = -1
    for poison in (float("inf"), -float("inf"), float("nan")):
        bad = x.clone()
        bad[..., 7] = poison
        for pair in ((bad, x), (x, bad)):
            dev = s8.empty_paged_cache(2, 1, page, D, device)
            s8.kv_append_paged(*pair, *dev, table, lens)
            assert torch.isnan(s8.attn_paged_cached(q, *dev, table, lens).float()).all()
            read = s8.kv_read_paged(*dev, table, lens, 1)
            for got, given in zip(read, pair):
                assert torch.isnan(got.float()).all() if given is bad else torch.isfinite(got.float()).all()


def test_append_equals_rope_then_append_and_is_repeatable(device):
    """Rotation on the way = apply_rope first (up to the 16-bit rounding between the two); twice the same bits."""
    B, Hkv, M, D, page = 3, 4, 50, 128, 32
    g = torch.Generator(device=device).manual_seed(3)
    k, v = (torch.randn(B, Hkv, M, D, device=device, generator=g).half() for _ in "kv")
    lens = torch.tensor([50, 90, 61], dtype=torch.int32, device=device)
    table, pages = po.pages_for(lens.cpu(), page)
    inv = freqs(D).to(device)
    place = lens.long().unsqueeze(1) - M + torch.arange(M, device=device)
    pools = [on(device, *po.random_cache(pages, Hkv, page, D)) for _ in range(3)]
    for p in pools[:2]:
        s8.kv_append_paged(k, v, *p, table.to(device), lens, inv_freq=inv)
    _, kr = s8.apply_rope(k, k, place, inv)
    s8.kv_append_paged(kr, v, *pools[2], table.to(device), lens)
    assert all(torch.equal(a, b) for a, b in zip(pools[0], pools[1]))
    assert (pools[0][0].int() - pools[2][0].int()).abs().max() <= 1 and torch.equal(pools[0][2], pools[2][2])


# ---- read back ----

@pytest.mark.parametrize("page,D,dtype", [(16, 128, torch.float16), (64, 32, torch.bfloat16), (256, 256, torch.float16)])
def test_read_against_definition(device, binding, page, D, dtype):
    lens = [0, 1, 300, 77]
    table, pages = po.pages_for(lens, page, width=5 if page == 64 else None)
    table[3, 0] = -1 if page == 16 else table[3, 0]
    cache = po.random_cache(pages, 3, page, D)
    first = torch.tensor([0, -3, 290, 5], dtype=torch.int32)
    lens_t = torch.tensor(lens, dtype=torch.int32)
    k, v = s8.kv_read_paged(*on(device, *cache, table, lens_t), 33, first=first.to(device), dtype=dtype)
    for got, codes, scale in ((k, cache[0], cache[1]), (v, cache[2], cache[3])):
        assert got.shape == (4, 3, 33, D) and got.dtype == dtype
        for b in range(4):
            held = min(lens[b], table.shape[1] * page)
            for j in range(33):
                token = int(first[b]) + j
                at = po.place_of(table[b].tolist(), page, token, pages) if 0 <= token < held else None
                want = torch.zeros(3, D)
                if at is not None:
                    want = codes[at[0], :, at[1]].float() * scale[at[0]].unsqueeze(1)
                assert torch.equal(got[b, :, j].cpu(), want.to(dtype))
    whole, _ = s8.kv_read_paged(*on(device, *cache, table, lens_t), 0)
    assert whole.shape == (4, 3, 0, D)


# ---- attention ----

ATTEND = [  # B lens, Hq, Hkv, M, D, page, dtype, causal, window, query_lens
    ([1, 15, 16, 17], 8, 2, 1, 128, 16, torch.float16, True, -1, None),
    ([1000, 0, 333, 1], 8, 1, 1, 128, 64, torch.bfloat16, True, -1, None),
    ([257, 700], 16, 1, 1, 64, 32, torch.bfloat16, True, -1, None),
    ([500, 31], 6, 6, 1, 256, 128, torch.float16, True, -1, None),
    ([900], 32, 1, 1, 32, 256, torch.float16, True, -1, None),
    ([600, 45, 9], 28, 4, 1, 128, 16, torch.float16, True, 40, None),
    ([300, 7, 0, 64], 8, 2, 5, 128, 16, torch.bfloat16, True, -1, [5, 5, 0, 2]),
    ([123, 300], 12, 4, 9, 64, 64, torch.float16, True, 17, [9, 3]),
    ([90, 200], 16, 2, 8, 256, 16, torch.float16, True, -1, None),
    ([260], 8, 1, 33, 128, 32, torch.float16, True, -1, None),
    ([70, 130], 4, 2, 64, 32, 16, torch.bfloat16, False, -1, [64, 50]),
    ([3, 90], 4, 2, 20, 128, 64, torch.float16, True, -1, None),        # more queries than context: rows without keys
    ([500], 8, 2, 3, 64, 32, torch.float16, False, 100, None),
    ([40], 2, 1, 1, 64, 16, torch.float16, True, 0, None),              # a window of nothing
]


def held_to(out, q, cache, table, lens, **kw):
    ref, tol = po.attend(q, *cache, table, lens, **kw)
    off = (out.cpu().double() - ref).abs()
    assert torch.isfinite(out.float()).all() and (off <= tol).all(), float((off / tol.clamp(min=1e-30)).max())


def attend_case(device, case, backend=_lib.SL8_BACKEND_AUTO):
    lens, Hq, Hkv, M, D, page, dtype, causal, window, query_lens = case
    B = len(lens)
    table, pages = po.pages_for(lens, page, seed=sum(lens))
    cache = po.random_cache(pages, Hkv, page, D, seed=Hq)
    q = (torch.randn(B, M, Hq, D, generator=torch.Generator().manual_seed(M)) * 1.5).to(dtype).transpose(1, 2)
    lens_t = torch.tensor(lens, dtype=torch.int32)
    ql = None if query_lens is None else torch.tensor(query_lens, dtype=torch.int32)
    out = s8.attn_paged_cached(*on(device, q, *cache, table, lens_t), causal=causal, window_left=window,
                               query_lens=None if ql is None else ql.to(device), backend=backend)
    assert out.shape == q.shape and out.dtype == dtype
    held_to(out, q, cache, table, lens, causal=causal, window=window, query_lens=query_lens)


@pytest.mark.parametrize("case", ATTEND)
def test_attend_against_definition(device, binding, case):
    attend_case(device, case)


def test_attend_scales_of_very_different_pages(device):
    """Pages whose V scales lie a factor of 10^4 apart, a page of zeros, a negative and a given softmax scale."""
    lens, page, D = [100, 64], 16, 128
    table, pages = po.pages_for(lens, page)
    cache = list(po.random_cache(pages, 2, page, D, seed=9))
    cache[3] = cache[3] * torch.tensor([1e-2, 1.0, 1e2, 3.0, 0.1, 10.0] * 3)[:pages].unsqueeze(1)
    cache[2][table[0, 1]] = 0
    cache[3][table[0, 1]] = po.FLOOR
    q = torch.randn(2, 4, 1, D, generator=torch.Generator().manual_seed(2)).half()
    for scale in (None, 0.3, -0.05, 0.0):
        out = s8.attn_paged_cached(*on(device, q, *cache, table, torch.tensor(lens, dtype=torch.int32)), scale=scale)
        held_to(out, q, cache, table, lens, scale=scale)


def test_attend_large_and_tiny_queries(device):
    """bf16 rows far outside fp16's range, a row of zeros, and logits that saturate the softmax."""
    lens, page, D = [80], 16, 64
    table, pages = po.pages_for(lens, page)
    cache = po.random_cache(pages, 1, page, D, seed=4)
    q = torch.randn(1, 5, 1, D, generator=torch.Generator().manual_seed(5))
    q = (q * torch.tensor([1e-20, 1.0, 0.0, 60.0, 1e-6]).view(1, 5, 1, 1)).bfloat16()
    out = s8.attn_paged_cached(*on(device, q, *cache, table, torch.tensor(lens, dtype=torch.int32)))
    held_to(out, q, cache, table, lens)
    q[0, 1, 0, 3] = float("nan")
    out = s8.attn_paged_cached(*on(device, q, *cache, table, torch.tensor(lens, dtype=torch.int32)))
    assert torch.isnan(out[0, 1].float()).all() and torch.isfinite(out[0, [0, 2, 3, 4]].float()).all()


def test_attend_ignores_what_is_not_there(device):
    """Missing pages, pages never written, and garbage behind a sequence's end."""
    lens, page, D = [100, 50], 16, 128
    table, pages = po.pages_for(lens, page, spare=3)
    cache = list(po.random_cache(pages, 2, page, D, seed=6))
    table[0, 2], table[0, 4] = -1, pages + 7
    table[0, 7:] = 2**31 - 1
    empty = int(table[1, 1])
    cache[1][empty] = cache[3][empty] = 0
    q = torch.randn(2, 8, 1, D, generator=torch.Generator().manual_seed(7)).half()
    lens_t = torch.tensor(lens, dtype=torch.int32)
    out = s8.attn_paged_cached(*on(device, q, *cache, table, lens_t))
    held_to(out, q, cache, table, lens)
    # slots behind the end, and pages of nobody: any codes, any scales
    used = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for i in range(n):
            at = po.place_of(table[b].tolist(), page, i, pages)
            if at is not None:
                used[at] = True
    for i in (0, 2):
        cache[i] = torch.where(used[:, None, :, None], cache[i], torch.full_like(cache[i], 113))
    nobody = ~used.any(1)
    for i in (1, 3):
        cache[i][nobody] = float("nan")
    again = s8.attn_paged_cached(*on(device, q, *cache, table, lens_t))
    assert torch.equal(out, again)
    # no page at all
    none = s8.attn_paged_cached(q.to(device), *s8.empty_paged_cache(0, 2, page, D, device), torch.zeros(2, 0, dtype=torch.int32, device=device),
                                lens_t.to(device))
    assert (none == 0).all()


@pytest.mark.parametrize("M,backend", [(4, _lib.SL8_BACKEND_AUTO), (40, _lib.SL8_BACKEND_MMA), (40, _lib.SL8_BACKEND_TCGEN05)])
@pytest.mark.parametrize("side", [1, 3])
def test_attend_rows_that_do_not_see_a_bad_page(device, M, backend, side):
    """A page whose K or V scale is NaN makes the rows that see it NaN and leaves the others alone: the last
    page under the causal mask, an early one under a window."""
    n, page, D, Hkv, Hq, window = 98, 16, 64, 1, 4, 34
    table, pages = po.pages_for([n], page)
    cache = list(po.random_cache(pages, Hkv, page, D, seed=21))
    q = torch.randn(1, Hq, M, D, generator=torch.Generator().manual_seed(22)).half()
    lens = torch.tensor([n], dtype=torch.int32)
    place = torch.arange(n - M, n)
    first_seen = (place - window + 1).clamp(min=0)
    hits = 0
    for at, win in ((n - 1) // page, -1), (3, window):
        bad = [t.clone() for t in cache]
        bad[side][int(table[0, at])] = float("nan")
        out = s8.attn_paged_cached(*on(device, q, *bad, table, lens), window_left=win, backend=backend).cpu()
        ref, tol = po.attend(q, *cache, table, [n], window=win)
        sees = (place >= at * page) & ((first_seen < (at + 1) * page) if win >= 0 else torch.ones(M, dtype=torch.bool))
        hits += int(sees.any()) * int((~sees).any())
        assert torch.isnan(out[:, :, sees].float()).all()
        assert ((out.double() - ref).abs() <= tol)[:, :, ~sees].all()
    assert hits == 2


def test_attend_long_context_offsets(device):
    """A pool of more than 2^31 bytes, read at its end, and more contexts than the grid has blocks."""
    page, D, Hkv = 256, 256, 8
    pages = 2**31 // (page * D * Hkv) + 40
    codes = torch.randint(-127, 128, (pages, Hkv, page, D), dtype=torch.int8, device=device)
    scale = torch.rand(pages, Hkv, device=device) * 0.02 + 0.01
    ids = torch.tensor([pages - 1, 0, pages - 3, pages - 2], dtype=torch.int32)
    small = [codes[ids.long()].cpu(), scale[ids.long()].cpu()]
    q = torch.randn(1, 16, 1, D, generator=torch.Generator().manual_seed(8)).half()
    lens = torch.tensor([901], dtype=torch.int32)
    out = s8.attn_paged_cached(*on(device, q), codes, scale, codes, scale, *on(device, ids.unsqueeze(0), lens))
    held_to(out, q, small * 2, torch.arange(4, dtype=torch.int32).unsqueeze(0), [901])


def test_attend_strides_streams_and_repeats(device, binding):
    lens, page, D = [700, 90, 333, 5] * 20, 16, 128
    table, pages = po.pages_for(lens, page)
    cache = on(device, *po.random_cache(pages, 2, page, D))
    lens_t, table = on(device, torch.tensor(lens, dtype=torch.int32), table)
    wide = torch.randn(80, 1, 8, 2 * D + 3, device=device).half()
    a = wide[..., :D].transpose(1, 2)                       # rows that are not 16-byte aligned
    b = torch.randn(80, 3, 8, D, device=device).half()[:, 1:2].transpose(1, 2)
    for q in (a, b):
        ref = s8.attn_paged_cached(q.contiguous(), *cache, table, lens_t)
        assert torch.equal(s8.attn_paged_cached(q, *cache, table, lens_t), ref)
        assert torch.equal(s8.attn_paged_cached(q, *cache, table[:, : table.shape[1] - 1], lens_t, max_context_len=700), ref)
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        outs = [s8.attn_paged_cached(q, *cache, table, lens_t) for _ in range(5)]
    here = [s8.attn_paged_cached(q, *cache, table, lens_t) for _ in range(5)]     # beside the other stream's calls
    torch.cuda.current_stream(device).wait_stream(side)
    assert all(torch.equal(o, ref) for o in outs + here)
    # one sequence at a time gives the same rows up to the split's rounding: the split is not observable beyond it
    one = s8.attn_paged_cached(q[:1], *cache, table[:1], lens_t[:1])
    assert (one.float() - ref[:1].float()).abs().max() <= 4 * 2.0 ** -11 * ref.float().abs().max()


@pytest.mark.parametrize("M,backend", [(1, _lib.SL8_BACKEND_AUTO), (70, _lib.SL8_BACKEND_MMA), (70, _lib.SL8_BACKEND_TCGEN05)])
def test_attend_sees_no_key_past_the_stated_length(device, M, backend):
    lens, page, D = [500, 300, 100], 64, 64
    table, pages = po.pages_for(lens, page)
    cache = po.random_cache(pages, 2, page, D)
    q = torch.randn(3, 4, M, D, generator=torch.Generator().manual_seed(9)).half()
    args = on(device, q, *cache, table, torch.tensor(lens, dtype=torch.int32))
    for limit in (500, 333, 16, 1):
        held_to(s8.attn_paged_cached(*args, max_context_len=limit, backend=backend), q, cache, table, lens, limit=limit)


# More units than SMs, or more chunks than a cluster takes: the line of all units is cut into equal ranges
LINE = [
    ([7, 0, 33, 64, 100, 1] * 16, 4, 2, 1, 64, 16, torch.float16, True, -1, None),
    ([300, 5, 0, 170] * 10, 10, 5, 1, 128, 32, torch.bfloat16, True, 37, None),
    ([65, 130, 31] * 14, 20, 4, 4, 128, 16, torch.float16, True, -1, [4, 2, 0] * 14),
    ([90, 40] * 45, 6, 2, 9, 64, 64, torch.bfloat16, True, -1, None),
    ([20, 70] * 40, 4, 2, 20, 32, 16, torch.float16, False, -1, None),
    ([33, 48] * 45, 4, 2, 3, 256, 16, torch.float16, True, -1, None),
    ([129] * 80, 16, 2, 5, 256, 64, torch.float16, True, 60, None),
    ([21000], 4, 1, 1, 128, 64, torch.float16, True, -1, None),
    ([9000, 17], 8, 1, 6, 64, 128, torch.bfloat16, True, -1, [6, 6]),
    ([9000], 2, 1, 1, 32, 256, torch.float16, True, -1, None),
    # 9 ... 64 rows per KV head: keys on the rows of the MMA
    ([200, 128, 129, 1, 0] * 20, 16, 2, 2, 128, 16, torch.float16, True, -1, None),
    ([300, 77] * 40, 32, 2, 4, 64, 32, torch.bfloat16, True, 33, [4, 3] * 40),
    ([140, 260] * 40, 10, 2, 8, 128, 64, torch.float16, True, 5, None),
    ([90, 400, 30] * 26, 12, 2, 4, 128, 256, torch.bfloat16, False, 100, None),
    ([3000, 2900, 2999] * 4, 12, 6, 8, 64, 128, torch.float16, True, 2500, None),
    ([7000, 3, 0], 11, 1, 1, 128, 16, torch.float16, True, -1, None),
    ([20, 3] * 40, 4, 2, 30, 128, 16, torch.float16, True, -1, None),   # more queries than context
]


@pytest.mark.parametrize("case", LINE)
def test_many_units_against_definition(device, case):
    attend_case(device, case)


PREFILL = [  # lens, Hq, Hkv, M, D, page, dtype, causal, window, query_lens
    ([200], 4, 4, 200, 128, 16, torch.float16, True, -1, None),
    ([300, 77, 0, 129], 8, 2, 77, 128, 64, torch.bfloat16, True, -1, [77, 77, 0, 40]),
    ([700, 130], 4, 1, 65, 64, 32, torch.float16, True, -1, None),
    ([260, 64], 28, 4, 33, 128, 128, torch.float16, True, 50, [33, 20]),
    ([400], 6, 6, 150, 256, 16, torch.bfloat16, True, -1, None),
    ([190, 70], 4, 2, 128, 64, 256, torch.bfloat16, False, -1, [100, 70]),
    ([90], 2, 2, 130, 128, 16, torch.float16, True, -1, None),          # more queries than context
    ([333], 3, 1, 90, 64, 16, torch.float16, False, 100, None),
    ([150], 2, 1, 70, 128, 16, torch.float16, True, 0, None),
    ([129], 16, 1, 17, 32, 16, torch.float16, True, -1, None),          # D = 32: the split kernel, several row units
]


@pytest.mark.parametrize("case", PREFILL)
def test_many_rows_against_definition(device, binding, case):
    if case[4] != 32:
        attend_case(device, case, _lib.SL8_BACKEND_TCGEN05)
    attend_case(device, case, _lib.SL8_BACKEND_MMA)
    attend_case(device, case)
    assert _C.device_status() == 0


def test_many_rows_missing_pages_scales_and_groups(device):
    """Missing and empty pages, V scales far apart, a negative softmax scale (the split kernel serves it), rows in
    a strided layout; and a batch whose dense copies are made in several groups."""
    lens, page, D, M = [150, 90], 16, 128, 40
    table, pages = po.pages_for(lens, page, spare=3)
    cache = list(po.random_cache(pages, 2, page, D, seed=6))
    table[0, 2], table[0, 4] = -1, pages + 7
    empty = int(table[1, 1])
    cache[1][empty] = cache[3][empty] = 0
    cache[3] = cache[3] * torch.tensor([1e-2, 1.0, 1e2, 3.0, 0.1, 10.0] * 9)[:pages].unsqueeze(1)
    q = torch.randn(2, M, 8, 2 * D, generator=torch.Generator().manual_seed(7)).half()[..., :D].transpose(1, 2)
    lens_t = torch.tensor(lens, dtype=torch.int32)
    for scale in (None, 0.2, -0.05):
        out = s8.attn_paged_cached(*on(device, q, *cache, table, lens_t), scale=scale,
                                   backend=_lib.SL8_BACKEND_AUTO if scale == -0.05 else _lib.SL8_BACKEND_TCGEN05)
        held_to(out, q, cache, table, lens, scale=scale)
    with pytest.raises(RuntimeError, match="not supported"):
        s8.attn_paged_cached(*on(device, q, *cache, table, lens_t), scale=-0.05, backend=_lib.SL8_BACKEND_TCGEN05)
    bad = q.clone()
    bad[1, 3, 5, 2] = float("nan")
    out = s8.attn_paged_cached(*on(device, bad, *cache, table, lens_t), backend=_lib.SL8_BACKEND_TCGEN05)
    assert torch.isnan(out[1, 3, 5].float()).all()
    out[1, 3, 5] = 0
    assert torch.isfinite(out.float()).all()
    # 24 units of 200000 keys at D = 128 are 2.5 GB of dense copies: two groups; against one sequence at a time
    g = torch.Generator(device=device).manual_seed(11)
    lens = [200000, 29000, 257]
    table, pages = po.pages_for(lens, 128)
    big = [torch.randint(-127, 128, (pages, 8, 128, D), dtype=torch.int8, device=device, generator=g) for _ in "kv"]
    sc = [torch.rand(pages, 8, device=device, generator=g) * 0.02 + 0.01 for _ in "kv"]
    cache = (big[0], sc[0], big[1], sc[1])
    q = torch.randn(3, 16, 40, D, device=device, generator=g).half()
    args = on(device, table, torch.tensor(lens, dtype=torch.int32))
    out = s8.attn_paged_cached(q, *cache, *args, max_context_len=200000, backend=_lib.SL8_BACKEND_TCGEN05)
    for b in range(3):
        one = s8.attn_paged_cached(q[b:b + 1], *cache, args[0][b:b + 1], args[1][b:b + 1], max_context_len=lens[b],
                                   backend=_lib.SL8_BACKEND_TCGEN05)
        assert torch.equal(out[b:b + 1], one)
    # and the first rows against the split kernel (up to 64 rows: 20 tokens of 2 heads per KV head)
    few = s8.attn_paged_cached(q[:, :, 20:], *cache, *args, max_context_len=200000)
    assert (few.float() - out[:, :, 20:].float()).abs().max() <= 0.01 * out.float().abs().max()
    assert _C.device_status() == 0


@pytest.mark.parametrize("M,Hq,D", [(1, 16, 128), (3, 8, 64), (2, 16, 256), (9, 8, 32)])
@pytest.mark.parametrize("longest", [3, 40, 200])
def test_many_short_contexts(device, M, Hq, D, longest):
    """More (sequence, head) units than blocks, a chunk or less each, some empty, one far longer: the bound given and not."""
    B, Hkv, page = 90, 2, 16
    g = torch.Generator().manual_seed(longest + M)
    lens = torch.randint(0, longest + 1, (B,), generator=g).tolist()
    lens[37] = 3 * longest + 160
    table, pages = po.pages_for(lens, page, seed=longest)
    cache = po.random_cache(pages, Hkv, page, D, seed=M)
    q = torch.randn(B, Hq, M, D, generator=g).half()
    dev = on(device, q, *cache, table, torch.tensor(lens, dtype=torch.int32))
    out = s8.attn_paged_cached(*dev, max_context_len=max(lens))
    held_to(out, q, cache, table, lens)
    held_to(s8.attn_paged_cached(*dev), q, cache, table, lens)
    assert torch.equal(out, s8.attn_paged_cached(*dev, max_context_len=max(lens)))


def test_line_and_many_rows_in_graphs(device):
    """The two kernels with a second launch behind them (partials joined, dense copies), captured and replayed over
    new contents, two graphs side by side on two streams."""
    g = torch.Generator(device=device).manual_seed(12)
    lens = torch.tensor([40, 700, 333, 5] * 25, dtype=torch.int32)
    table, pages = po.pages_for(lens, 16)
    cache = on(device, *po.random_cache(pages, 2, 16, 64))
    table, lens = on(device, table, lens)
    q1 = torch.randn(100, 4, 1, 64, device=device, generator=g).half()
    q2 = torch.randn(100, 4, 70, 64, device=device, generator=g).half()
    calls = [lambda: s8.attn_paged_cached(q1, *cache, table, lens), lambda: s8.attn_paged_cached(q2, *cache, table, lens, max_context_len=700)]
    eager = [c().clone() for c in calls]
    graphs, outs = [], []
    for c in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(c())
        graphs.append(graph)
    lens.sub_(3)
    want = [c().clone() for c in calls]
    side = [torch.cuda.Stream(device) for _ in graphs]
    for _ in range(3):
        for s, graph in zip(side, graphs):
            s.wait_stream(torch.cuda.current_stream(device))
            with torch.cuda.stream(s):
                graph.replay()
        for s in side:
            torch.cuda.current_stream(device).wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(outs, want)) and not torch.equal(outs[0], eager[0])
    assert _C.device_status() == 0


def test_window_of_any_size(device):
    lens, page, D = [90, 3], 16, 64
    table, pages = po.pages_for(lens, page)
    cache = po.random_cache(pages, 1, page, D)
    q = torch.randn(2, 2, 9, D, generator=torch.Generator().manual_seed(13)).half()
    args = on(device, q, *cache, table, torch.tensor(lens, dtype=torch.int32))
    for window in (2**31 - 1, 2**40, 2**30, 2**30 - 1):
        held_to(s8.attn_paged_cached(*args, window_left=window), q, cache, table, lens)


def test_serving_loop_and_graphs(device):
    """A prompt, single tokens and a piece of several tokens through append and attention, against 16-bit
    attention over the values read back; then the decode step captured twice and replayed."""
    B, Hq, Hkv, D, page = 3, 8, 2, 128, 16
    g = torch.Generator(device=device).manual_seed(10)
    cache = s8.empty_paged_cache(40, Hkv, page, D, device)
    table = torch.randperm(36, device=device, generator=g).int().view(3, 12)
    inv = freqs(D, 500000.0).to(device)
    lens = torch.zeros(3, dtype=torch.int32, device=device)

    def piece(M):
        return (torch.randn(B, M, Hq if i == 0 else Hkv, D, device=device, generator=g).half().transpose(1, 2) for i in range(3))

    kept = [[] for _ in range(B)]
    for M, new in ((40, [40, 17, 1]), (1, [1, 1, 1]), (1, [1, 1, 1]), (5, [5, 0, 3]), (1, [1, 1, 1])):
        q, k, v = piece(M)
        n = torch.tensor(new, dtype=torch.int32, device=device)
        lens += n
        qr = s8.kv_append_paged(k, v, *cache, table, lens, new_lens=n, q=q, inv_freq=inv)
        out = s8.attn_paged_cached(qr, *cache, table, lens, query_lens=n, max_context_len=192)
        kf, vf = s8.kv_read_paged(*cache, table, lens, 192)
        for b in range(B):
            L, m = int(lens[b]), new[b]
            kept[b].append(v[b, :, :m])
            if m:
                ref = s8.attn_fp16_fwd(qr[b:b + 1, :, :m].contiguous(), kf[b:b + 1, :, :L].contiguous(), vf[b:b + 1, :, :L].contiguous(),
                                       causal=True)
                assert (out[b, :, :m].float() - ref[0].float()).abs().max() <= 0.01 * vf[b, :, :L].float().abs().max()
            assert (out[b, :, m:] == 0).all()
    for b in range(B):   # the cache holds what was appended: half a step of a page's scale per growth (at most six appends)
        truth = torch.cat(kept[b], 1).float()
        L = truth.shape[1]
        step = cache[3][table[b, torch.arange(L, device=device) // page].long()].t().unsqueeze(-1)
        assert ((vf[b, :, :L].float() - truth).abs() <= 3.01 * step + 2.0 ** -10 * truth.abs()).all()

    q, k, v = piece(1)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            lens.add_(1)
            qr = s8.kv_append_paged(k, v, *cache, table, lens, q=q, inv_freq=inv)
            outs.append(s8.attn_paged_cached(qr, *cache, table, lens))
        graphs.append(graph)
    start = [t.clone() for t in (*cache, lens)]
    replayed = []
    for i in (0, 1, 1, 0):
        graphs[i].replay()
        replayed.append(outs[i].clone())
    for t, s in zip((*cache, lens), start):
        t.copy_(s)
    for i in range(4):
        lens.add_(1)
        qr = s8.kv_append_paged(k, v, *cache, table, lens, q=q, inv_freq=inv)
        assert torch.equal(s8.attn_paged_cached(qr, *cache, table, lens), replayed[i])


def test_refusals(device, binding):
    D, page = 64, 16
    cache = s8.empty_paged_cache(4, 2, page, D, device)
    table = torch.zeros(2, 3, dtype=torch.int32, device=device)
    lens = torch.ones(2, dtype=torch.int32, device=device)
    q = torch.zeros(2, 4, 1, D, device=device, dtype=torch.float16)
    k = q[:, :2]
    inv = freqs(D).to(device)

    def cached(i, t):
        return [t if j == i else c for j, c in enumerate(cache)]

    bad = [
        ("CUDA", lambda: s8.attn_paged_cached(q.cpu(), *cache, table, lens)),
        ("float16 or bfloat16", lambda: s8.attn_paged_cached(q.float(), *cache, table, lens)),
        ("must be int8", lambda: s8.attn_paged_cached(q, *cached(0, cache[0].half()), table, lens)),
        ("contiguous", lambda: s8.attn_paged_cached(q, *cached(2, cache[2][:3]), table, lens)),
        ("scales must be", lambda: s8.attn_paged_cached(q, *cached(1, cache[1].half()), table, lens)),
        ("scales must be", lambda: s8.attn_paged_cached(q, *cached(3, cache[3][:, :1]), table, lens)),
        ("block_table", lambda: s8.attn_paged_cached(q, *cache, table.long(), lens)),
        ("block_table", lambda: s8.attn_paged_cached(q, *cache, table.t().contiguous().t(), lens)),
        ("context_lens", lambda: s8.attn_paged_cached(q, *cache, table, lens.long())),
        ("context_lens", lambda: s8.attn_paged_cached(q, *cache, table, lens[:1])),
        ("query_lens", lambda: s8.attn_paged_cached(q, *cache, table, lens, query_lens=lens.long())),
        ("divisible", lambda: s8.attn_paged_cached(q[:, :3], *cache, table, lens)),
        ("batch and head dim", lambda: s8.attn_paged_cached(q[:1], *cache, table, lens)),
        ("batch and head dim", lambda: s8.attn_paged_cached(q[..., :32], *cache, table, lens)),
        ("page size", lambda: s8.attn_paged_cached(q, *[c[:, :, :8].contiguous() if c.dim() == 4 else c for c in cache], table, lens)),
        ("head dim", lambda: s8.attn_paged_cached(q[..., :48], *[c[..., :48].contiguous() if c.dim() == 4 else c for c in cache], table, lens)),
        ("one dtype", lambda: s8.kv_append_paged(k, k.bfloat16(), *cache, table, lens)),
        ("one shape", lambda: s8.kv_append_paged(k, k[:, :1], *cache, table, lens)),
        ("must match the cache", lambda: s8.kv_append_paged(q, q, *cache, table, lens)),
        ("new_lens", lambda: s8.kv_append_paged(k, k, *cache, table, lens, new_lens=lens.float())),
        ("need inv_freq", lambda: s8.kv_append_paged(k, k, *cache, table, lens, q=q)),
        ("multiple of 16", lambda: s8.kv_append_paged(k, k, *cache, table, lens, inv_freq=inv[:3])),
        ("dtype of k", lambda: s8.kv_append_paged(k, k, *cache, table, lens, q=q.bfloat16(), inv_freq=inv)),
        ("need freq_axis", lambda: s8.kv_append_paged(k, k, *cache, table, lens, inv_freq=inv, positions=torch.zeros(2, 2, 1, dtype=torch.long, device=device))),
        ("not supported", lambda: s8.attn_paged_cached(q, *cache, table, lens, backend=_lib.SL8_BACKEND_TCGEN05_2Q)),
        ("negative", lambda: s8.kv_read_paged(*cache, table, lens, -1)),
        ("first", lambda: s8.kv_read_paged(*cache, table, lens, 1, first=lens.long())),
        ("dtype", lambda: s8.kv_read_paged(*cache, table, lens, 1, dtype=torch.float32)),
    ]
    for words, call in bad:
        with pytest.raises(RuntimeError, match=words):
            call()
    # nothing to do
    assert s8.attn_paged_cached(q[:, :, :0], *cache, table, lens).shape == (2, 4, 0, D)
    assert s8.attn_paged_cached(q[:0], *cache, table[:0], lens[:0]).shape == (0, 4, 1, D)
    assert s8.kv_append_paged(k[:, :, :0], k[:, :, :0], *cache, table, lens, q=q[:, :, :0], inv_freq=inv).shape == (2, 4, 0, D)
    assert s8.kv_append_paged(k[:0], k[:0], *cache, table[:0], lens[:0]) is None
