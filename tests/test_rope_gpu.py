"""Rotary positions against their definition in 64 bits: types, layouts, axes, far positions, strides, the
gradient (against the formula and against differences) and the refusals."""

import pytest
import torch

import paged_oracle as po
import superl8_b200 as s8
from superl8_b200 import _C

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["compiled", "ctypes"], autouse=True)
def binding(request):
    if request.param == "compiled" and _C._ext is None:
        pytest.skip("the compiled extension is not built")
    prev = _C.use_binding(request.param)
    yield
    _C.use_binding(prev)


def freqs(rot, base=10000.0):
    return (base ** (-torch.arange(rot // 2, dtype=torch.float64) / max(1, rot // 2))).float()


def held_to(y, x, dtype, pos, inv, axis=None, interleaved=False, inverse=False):
    ref, size = po.rotate(x, pos, inv, axis, interleaved, inverse)
    tol = size * po.ROTATE_ERR
    tol = tol + po.rounded(ref.abs() + tol, dtype)
    assert ((y.cpu().double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,Hq,Hkv,S,D,rot", [(1, 8, 2, 1, 128, 128), (2, 5, 5, 37, 64, 32), (1, 3, 1, 130, 72, 72),
                                              (2, 4, 2, 9, 80, 80), (1, 2, 1, 33, 256, 64), (3, 1, 1, 2, 6, 2),
                                              (1, 2, 2, 5, 72, 36), (1, 2, 1, 4, 32, 0)])
def test_rope_types_and_shapes(device, dtype, interleaved, B, Hq, Hkv, S, D, rot):
    g = torch.Generator().manual_seed(S + D)
    q, k = torch.randn(B, Hq, S, D, generator=g).to(dtype), torch.randn(B, Hkv, S, D, generator=g).to(dtype)
    pos = torch.randint(0, 5000, (B, S), generator=g)
    inv = freqs(rot)
    yq, yk = s8.apply_rope(q.to(device), k.to(device), pos.to(device), inv.to(device), interleaved=interleaved)
    assert yq.shape == q.shape and yq.dtype == dtype and yk.shape == k.shape
    held_to(yq, q, dtype, pos, inv, None, interleaved)
    held_to(yk, k, dtype, pos, inv, None, interleaved)
    if rot < D:
        assert torch.equal(yq[..., rot:].cpu(), q[..., rot:])


@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("pos_dtype", [torch.int32, torch.int64])
def test_rope_axes(device, mixed, pos_dtype):
    g = torch.Generator().manual_seed(11)
    q, k = torch.randn(2, 4, 75, 128, generator=g).bfloat16(), torch.randn(2, 1, 75, 128, generator=g).bfloat16()
    i = torch.arange(75)
    pos = torch.stack([torch.stack([i, i // 8 % 9, i % 8]), torch.stack([i + 3, i // 5 % 7, i % 5])], 1).to(pos_dtype)
    axis = s8.rope_freq_axis((16, 24, 24), mixed=mixed)
    assert sorted(axis.tolist()) == [0] * 16 + [1] * 24 + [2] * 24
    inv = freqs(128, 1e6)
    yq, yk = s8.apply_rope(q.to(device), k.to(device), pos.to(device), inv.to(device), freq_axis=axis.to(device))
    held_to(yq, q, torch.bfloat16, pos, inv, axis)
    held_to(yk, k, torch.bfloat16, pos, inv, axis)
    # equal positions on all axes are one axis; an axis number past the last reads the last
    same = i.to(pos_dtype).expand(3, 1, 75).to(device)
    one, _ = s8.apply_rope(q.to(device), None, i.to(pos_dtype).to(device), inv.to(device))
    three, _ = s8.apply_rope(q.to(device), None, same, inv.to(device), freq_axis=axis.to(device) * 100)
    assert torch.equal(one, three)


def test_rope_far_positions(device):
    """At position 2^31 - 1 a 32-bit product would be off by tens of radians."""
    g = torch.Generator().manual_seed(12)
    q = torch.randn(1, 2, 6, 64, generator=g)
    pos = torch.tensor([0, -7, 99_999, 1_000_003, -123_456_789, 2**31 - 1])
    inv = freqs(64)
    y, none = s8.apply_rope(q.to(device), None, pos.to(device), inv.to(device))
    assert none is None
    # the 64-bit product and reduction: 2^31 * 2^-52 rad on top of the bound
    held_to(y, q, torch.float32, pos, inv)
    y16, _ = s8.apply_rope(q.to(device), None, pos.int().to(device), inv.to(device))
    assert torch.equal(y, y16)


def test_rope_strides_and_empty(device):
    g = torch.Generator().manual_seed(13)
    inv = freqs(64).to(device)
    qkv = torch.randn(2, 19, 3, 4, 72, generator=g).half().to(device)           # a fused projection's output
    pos = torch.arange(19, device=device)
    views = {"token-major": qkv[:, :, 0, :, :64].transpose(1, 2), "unaligned": qkv[:, :, 1, :, 3:67].transpose(1, 2),
             "channels strided": torch.randn(2, 64, 4, 19, device=device).half().permute(0, 2, 3, 1),
             "batch of one expanded": qkv[:1, :, 2, :, :64].transpose(1, 2).expand(2, 4, 19, 64)}
    for name, x in views.items():
        ref, _ = s8.apply_rope(x.contiguous(), None, pos, inv)
        y, yk = s8.apply_rope(x, x[:, :2], pos, inv)
        assert torch.equal(y, ref) and torch.equal(yk, ref[:, :2]), name
    for shape in ((0, 4, 5, 64), (2, 0, 5, 64), (2, 4, 0, 64)):
        x = torch.empty(shape, device=device, dtype=torch.float16)
        y, _ = s8.apply_rope(x, None, torch.arange(shape[2], device=device), inv)
        assert y.shape == shape


@pytest.mark.parametrize("S,D", [(16, 32), (40, 32)])
def test_rope_of_overlapping_rows(device, S, D):
    """Rows one element apart, and heads that are one tensor seen several times."""
    flat = torch.randn(200, generator=torch.Generator().manual_seed(5)).half()
    pos, inv = torch.arange(S), freqs(D)
    for strides in ((0, 0, 1, 1), (0, 1, 0, 1), (0, 0, 2, 1), (0, 0, 0, 1)):
        q = flat.as_strided((1, 3, S, D), strides)
        y, none = s8.apply_rope(flat.to(device).as_strided((1, 3, S, D), strides), None, pos.to(device), inv.to(device))
        assert none is None
        held_to(y, q, torch.float16, pos, inv)


def test_rope_gradient_against_the_formula_and_differences(device):
    g = torch.Generator().manual_seed(14)
    pos, inv = torch.randint(0, 300, (3, 2, 21), generator=g), freqs(48)
    axis = s8.rope_freq_axis((8, 8, 8), mixed=True)
    for dtype in (torch.float32, torch.bfloat16):
        q, k = torch.randn(2, 4, 21, 64, generator=g).to(dtype), torch.randn(2, 2, 21, 64, generator=g).to(dtype)
        gq, gk = torch.randn(q.shape, generator=g).to(dtype), torch.randn(k.shape, generator=g).to(dtype)
        qd, kd = q.to(device).requires_grad_(), k.to(device).requires_grad_()
        yq, yk = s8.apply_rope(qd, kd, pos.to(device), inv.to(device), freq_axis=axis.to(device))
        dq, dk = torch.autograd.grad((yq, yk), (qd, kd), (gq.to(device), gk.to(device)))
        held_to(yq.detach(), q, dtype, pos, inv, axis)
        held_to(dq, gq, dtype, pos, inv, axis, inverse=True)
        held_to(dk, gk, dtype, pos, inv, axis, inverse=True)
    # differences of the fp32 operator: linear, so a step of 1 has no truncation error
    e = torch.zeros(2, 4, 21, 64)
    e[1, 2, 17, 5] = 1.0
    up, _ = s8.apply_rope((q.float() + e).to(device), None, pos.to(device), inv.to(device), freq_axis=axis.to(device))
    down, _ = s8.apply_rope((q.float() - e).to(device), None, pos.to(device), inv.to(device), freq_axis=axis.to(device))
    qd = q.float().to(device).requires_grad_()
    y, _ = s8.apply_rope(qd, None, pos.to(device), inv.to(device), freq_axis=axis.to(device))
    (d,) = torch.autograd.grad(y, qd, gq.float().to(device))
    by_difference = ((up.double() - down.double()) / 2 * gq.to(device).double()).sum()
    # two rotated elements of size <= |x| + 1, each off by fp32 roundings, times |gq|
    assert abs(float(d[1, 2, 17, 5]) - float(by_difference)) <= 4 * (q.abs().max().item() + 1) * gq.abs().max().item() * po.ROTATE_ERR * 2
    # only one side asked for, an unused output, and a second derivative
    kd = k.float().to(device).requires_grad_()
    yq, yk = s8.apply_rope(q.float().to(device), kd, pos.to(device), inv.to(device), freq_axis=axis.to(device))
    (dk,) = torch.autograd.grad(yk.square().sum(), kd, create_graph=True)
    (ddk,) = torch.autograd.grad(dk.sum(), kd)
    assert (ddk - 2).abs().max() <= 2 * 2 * 4 * po.ROTATE_ERR        # d/dk sum(2 R'R k) = 2
    w = torch.randn(2, 1, 21, 64, device=device, requires_grad=True)  # a broadcast input: its gradient is summed
    yq, _ = s8.apply_rope(w.expand(2, 4, 21, 64), None, pos.to(device), inv.to(device), freq_axis=axis.to(device))
    yq.sum().backward()
    assert w.grad.shape == w.shape


def test_rope_streams_graphs_and_the_next_operator(device):
    """On another stream, captured with its backward, and into the attention operators it feeds."""
    g = torch.Generator(device=device).manual_seed(15)
    q = torch.randn(1, 4, 256, 64, device=device, generator=g).half().requires_grad_()
    k = torch.randn(1, 2, 256, 64, device=device, generator=g).half().requires_grad_()
    pos, inv = torch.arange(256, device=device), freqs(64).to(device)
    go = torch.randn(q.shape, device=device, generator=g).half()

    def step():
        yq, yk = s8.apply_rope(q, k, pos, inv)
        return (yq.detach(), *torch.autograd.grad((yq, yk), (q, k), (go, go[:, :2])))

    eager = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream(device).wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    with torch.no_grad():
        q.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    # twice the input is twice the output, bit for bit, except below 2^-14: there fp16's step is 2^-24 whatever
    # the value, round(2y) is off by at most 2^-25 and 2 round(y) by at most 2^-24
    off = (captured[0].detach().float() - 2 * eager[0].float()).abs()
    assert (off <= torch.where(eager[0].abs() < 2.0 ** -14, 3 * 2.0 ** -25, 0.0)).all()
    assert torch.equal(captured[1], eager[1])
    with torch.no_grad():
        yq, yk = s8.apply_rope(q, k, pos, inv)
        out = s8.attn_fp16_fwd(yq, yk, yk, causal=True)
    assert torch.isfinite(out.float()).all()


def test_rope_refusals(device):
    q = torch.zeros(2, 4, 8, 64, device=device, dtype=torch.float16)
    pos, inv = torch.arange(8, device=device), freqs(64).to(device)
    axis = s8.rope_freq_axis((16, 16)).to(device)
    bad = [
        ("CUDA", lambda: s8.apply_rope(q.cpu(), None, pos, inv)), ("CUDA", lambda: s8.apply_rope(q, None, pos.cpu(), inv)),
        ("B,H,S,D", lambda: s8.apply_rope(q[0], None, pos, inv)), ("float16", lambda: s8.apply_rope(q.double(), None, pos, inv)),
        ("one dtype", lambda: s8.apply_rope(q, q.float(), pos, inv)), ("agree", lambda: s8.apply_rope(q, q[:, :, :4], pos, inv)),
        ("int32 or int64", lambda: s8.apply_rope(q, None, pos.float(), inv)),
        ("positions must be", lambda: s8.apply_rope(q, None, pos[:5], inv)),
        ("positions must be", lambda: s8.apply_rope(q, None, pos.expand(3, 8), inv)),
        ("need freq_axis", lambda: s8.apply_rope(q, None, pos.expand(2, 2, 8), inv)),
        ("float32", lambda: s8.apply_rope(q, None, pos, inv.double())), ("head dim", lambda: s8.apply_rope(q[..., :32], None, pos, inv)),
        ("even", lambda: s8.apply_rope(q[..., :63], None, pos, inv[:4])),
        ("freq_axis must be", lambda: s8.apply_rope(q, None, pos, inv, freq_axis=axis.int())),
        ("freq_axis must be", lambda: s8.apply_rope(q, None, pos, inv, freq_axis=axis[:3])),
        ("constant", lambda: s8.apply_rope(q, None, pos, inv.clone().requires_grad_())),
    ]
    for words, call in bad:
        with pytest.raises(RuntimeError, match=words):
            call()
    with pytest.raises(ValueError):
        s8.rope_freq_axis(())
