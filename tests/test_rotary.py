"""Rotary positions (devspace_amd.ops.fused.rotary*) against the rotation written in 64 bits."""
import math

import pytest
import torch

from devspace_amd.ops import fused

gpu = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    fused.ext()
    return torch.device("cuda")


def _ref(x, pos, freqs, interleaved, magnitude, sign=1.0):
    """float64: each pair of columns as a complex number times m e^(i pos f); also sum |pair| per column."""
    x = x.detach().double()
    r = freqs.numel()
    first = slice(0, 2 * r, 2) if interleaved else slice(0, r)
    second = slice(1, 2 * r, 2) if interleaved else slice(r, 2 * r)
    turns = pos.double()[..., None] * (freqs / (2 * math.pi))
    z = torch.polar(torch.full_like(turns, magnitude), sign * 2 * math.pi * (turns - turns.round()))[..., None, :]
    y, size = x.clone(), x.abs() * 0
    c = torch.complex(x[..., first], x[..., second]) * z
    y[..., first], y[..., second] = c.real, c.imag
    size[..., first] = size[..., second] = magnitude * (x[..., first].abs() + x[..., second].abs())
    return y, size


def _check(got, ref, size):
    """The output's rounding is half a step, eps / 2 of the value (fp16: at least half its smallest step,
    2^-25). Before it, in 32 bits with u = 2^-24: the reduced angle is off by at most 2 pi 2^-25 = 3.2 u,
    the sine and cosine by 4 u (two units in the last place), the magnitude's product, the two products and
    the sum by u each: under 12 u of |a| + |b|."""
    tol = 12 * 2.0 ** -24 * size + torch.finfo(got.dtype).eps / 2 * 1.0001 * ref.abs() + 2.0 ** -25 * (got.dtype == torch.float16)
    bad = (got.double() - ref).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((got.double() - ref).abs() - tol).max()))


def test_frequencies():
    f, m = fused.rotary_frequencies(8)
    assert m == 1.0 and f.dtype == torch.float64
    torch.testing.assert_close(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64))
    torch.testing.assert_close(fused.rotary_frequencies(8, scaling="linear", factor=4)[0], f / 4)
    n = fused.rotary_frequencies(8, scaling="ntk", factor=4)[0]
    assert n[0] == 1.0 and abs(n[-1].item() - f[-1].item() / 4) < 1e-18
    y, m = fused.rotary_frequencies(64, scaling="yarn", factor=16, original_length=4096)
    f = fused.rotary_frequencies(64)[0]
    assert abs(m - (0.1 * math.log(16) + 1)) < 1e-15
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(y[turns >= 32], f[turns >= 32])
    torch.testing.assert_close(y[turns <= 1], f[turns <= 1] / 16)
    between = (turns > 1) & (turns < 32)
    assert between.any() and (y[between] < f[between]).all() and (y[between] > f[between] / 16).all()
    for bad in (dict(dim=7), dict(dim=0), dict(dim=8, scaling="cubic"), dict(dim=8, factor=0.5), dict(dim=8, fast=1.0)):
        with pytest.raises(ValueError):
            fused.rotary_frequencies(**bad)


@pytest.mark.parametrize("interleaved", [False, True])
def test_cpu_form_matches_reference_and_its_gradient_differences(interleaved):
    torch.manual_seed(0)
    f, m = fused.rotary_frequencies(6, scaling="yarn", factor=4)
    x = torch.randn(2, 3, 2, 9, dtype=torch.float64, requires_grad=True)
    pos = torch.tensor([[0, 5, 100000], [7, 8, 9]])
    y = fused.rotary(x, pos, f, interleaved, m)
    torch.testing.assert_close(y, _ref(x, pos, f, interleaved, m)[0], atol=1e-9, rtol=0)
    assert torch.autograd.gradcheck(lambda t: fused.rotary(t, pos, f, interleaved, m), (x,))
    qkv = torch.randn(2, 3, 3, 2, 9)
    out = fused.rotary_qkv(qkv, pos, f, interleaved, m)
    q, k = fused.rotary_qk(qkv[:, :, 0], qkv[:, :, 1], pos, f, interleaved, m)
    assert torch.equal(out, torch.stack([q, k, qkv[:, :, 2]], 2))


def test_module_keeps_exact_frequencies():
    r = fused.Rotary(16, scaling="linear", factor=3.0)
    f = r.freqs.clone()
    r = r.to(torch.bfloat16)
    assert r.freqs.dtype == torch.float64 and torch.equal(r.freqs, f) and not r.state_dict()
    qkv = torch.randn(1, 4, 3, 2, 16)
    q, k = r(qkv[:, :, 0], qkv[:, :, 1], positions=2)
    assert torch.equal(torch.stack([q, k, qkv[:, :, 2]], 2), r(qkv, positions=2))


def test_refusals_cpu():
    f = fused.rotary_frequencies(8)[0]
    x = torch.randn(2, 3, 2, 8)
    for call in (lambda: fused.rotary(x[0], 0, f), lambda: fused.rotary(x, 0, f.float()),
                 lambda: fused.rotary(x[..., :6], 0, f), lambda: fused.rotary(x, torch.zeros(2), f),
                 lambda: fused.rotary(x, torch.zeros(4, dtype=torch.long), f),
                 lambda: fused.rotary(x, torch.zeros(3), f), lambda: fused.rotary_qkv(x[:, :, None], 0, f),
                 lambda: fused.rotary_qk(x, x[:1], 0, f), lambda: fused.rotary_qk(x, x.double(), 0, f)):
        with pytest.raises(ValueError):
            call()


CASES = [  # dtype, B, T, H, N, D, R, interleaved, scaling
    ("bf16", 2, 37, 4, 4, 64, 64, False, "none"),
    ("bf16", 3, 1, 16, 2, 128, 64, True, "yarn"),
    ("fp16", 1, 513, 2, 1, 80, 40, False, "ntk"),
    ("fp16", 2, 5, 3, 1, 72, 36, True, "linear"),
    ("fp32", 1, 9, 5, 5, 72, 18, False, "none"),
    ("fp32", 2, 33, 2, 2, 7, 2, True, "yarn"),
    ("bf16", 1, 3, 1, 1, 256, 250, False, "ntk"),
    ("bf16", 1, 1, 1, 1, 2, 2, False, "none"),
    ("fp32", 4, 700, 8, 1, 64, 64, True, "none"),
    ("bf16", 1, 4, 33, 31, 256, 256, True, "none"),
    ("bf16", 2, 21, 3, 2, 128, 66, True, "yarn"),  # 33 pairs and 62 copied columns: neither a whole number of accesses
    ("fp16", 2, 21, 3, 2, 127, 66, False, "none"),
    ("fp32", 1, 40, 2, 2, 99, 46, False, "linear"),
]


@gpu
@pytest.mark.parametrize("dtype,b,t,h,n,d,r,interleaved,scaling", CASES)
def test_qk_forward_and_backward(dtype, b, t, h, n, d, r, interleaved, scaling):
    dev, dt = _cuda(), DTYPES[dtype]
    gen = torch.Generator(device=dev)
    gen.manual_seed(1)
    f, m = fused.rotary_frequencies(r, scaling=scaling, factor=8.0, device=dev)
    q = torch.randn(b, t, h, d, device=dev, generator=gen).to(dt).requires_grad_()
    k = torch.randn(b, t, n, d, device=dev, generator=gen).to(dt).requires_grad_()
    pos = torch.randint(0, 1 << 20, (b, t), device=dev, generator=gen)
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    yq, yk = fused.rotary_qk(q, k, pos, f, interleaved, m)
    gq, gk = torch.autograd.grad((yq, yk), (q, k), (dq, dk))
    for got, x, sign in ((yq, q, 1.0), (yk, k, 1.0), (gq, dq, -1.0), (gk, dk, -1.0)):
        assert got.dtype == dt and got.shape == x.shape
        ref, size = _ref(x, pos, f, interleaved, m, sign)
        _check(got, ref, size)
        assert torch.equal(got[..., r:], x[..., r:])  # columns behind the turned ones are carried over
    assert torch.equal(fused.rotary(q, pos, f, interleaved, m), yq)  # alone, the same bits


@gpu
@pytest.mark.parametrize("dtype,b,t,h,d,r,interleaved", [("bf16", 2, 129, 3, 64, 64, False), ("fp16", 1, 7, 2, 40, 20, True),
                                                       ("fp32", 2, 1, 2, 64, 32, False)])
def test_packed_forward_and_backward(dtype, b, t, h, d, r, interleaved):
    dev, dt = _cuda(), DTYPES[dtype]
    torch.manual_seed(2)
    f, m = fused.rotary_frequencies(r, device=dev)
    qkv = torch.randn(b, t, 3, h, d, device=dev).to(dt).requires_grad_()
    dout = torch.randn_like(qkv)
    y = fused.rotary_qkv(qkv, 11, f, interleaved, m)
    (g,) = torch.autograd.grad(y, qkv, dout)
    pos = torch.arange(t, device=dev) + 11
    for got, x, sign in ((y, qkv, 1.0), (g, dout, -1.0)):
        for i in range(2):
            _check(got[:, :, i], *_ref(x[:, :, i], pos, f, interleaved, m, sign))
        assert torch.equal(got[:, :, 2], x[:, :, 2])


@gpu
def test_strides_and_forms_of_positions():
    dev = _cuda()
    torch.manual_seed(3)
    f, m = fused.rotary_frequencies(32, device=dev)
    base = torch.randn(2, 6, 3, 4, 64, device=dev).bfloat16()
    dense = base[:, :, 1].contiguous()
    pos = torch.arange(6, device=dev) + 5
    want = fused.rotary(dense, pos, f)
    heads_first = dense.transpose(1, 2).contiguous().transpose(1, 2)  # memory [B, H, T, D]
    shifted = torch.empty(dense.numel() + 1, device=dev, dtype=dense.dtype)[1:].view_as(dense).copy_(dense)  # odd address
    columns = dense.transpose(2, 3).contiguous().transpose(2, 3)  # last stride is not 1
    for x in (base[:, :, 1], heads_first, shifted, columns):
        assert torch.equal(fused.rotary(x, pos, f), want)
    wide = torch.arange(12, device=dev).view(6, 2)[:, 0] // 2 + 5  # a strided tensor of positions
    for p in (5, pos.int(), pos[None], pos.expand(2, 6), pos.repeat(2, 1), wide):
        assert torch.equal(fused.rotary(dense, p, f), want)
    assert torch.equal(fused.rotary(dense, None, f), fused.rotary(dense, 0, f))
    one = dense[:1].expand(2, -1, -1, -1)  # a broadcast input: its gradient is the sum
    leaf = dense[:1].detach().clone().requires_grad_()
    g = torch.randn_like(dense)
    (got,) = torch.autograd.grad(fused.rotary(leaf.expand(2, -1, -1, -1), pos, f), leaf, g)
    torch.testing.assert_close(got, sum(fused._rotary_hip(g[i:i + 1], None, False, -pos, f, False, 1.0)[0] for i in range(2)))
    assert torch.equal(fused.rotary(one, pos, f)[0], fused.rotary(one, pos, f)[1])


@gpu
def test_far_and_negative_positions():
    dev = _cuda()
    torch.manual_seed(4)
    f, m = fused.rotary_frequencies(64, device=dev)
    x = torch.randn(1, 6, 2, 64, device=dev)
    pos = torch.tensor([0, -1, -(1 << 20), (1 << 24) + 1, (1 << 31) + 7, 1 << 40], device=dev)
    ref, size = _ref(x, pos, f, False, 1.0)
    # turns in 64 bits: two roundings of 2^-53 of up to 2^40 / 2 pi turns here, and two in the reference
    _check(fused.rotary(x, pos, f), ref, size * (1 + 4 * 2.0 ** 40 * 2.0 ** -53 / (12 * 2.0 ** -24)))
    back = fused.rotary(fused.rotary(x, pos, f), -pos, f)
    torch.testing.assert_close(back, x, atol=1e-4, rtol=0)  # a turn and its inverse: 2 * 12 u of |a| + |b| < 20


@gpu
def test_gradient_is_the_transpose():
    """<dy, J dx> = <J^T dy, dx>, with J dx taken as a difference of two calls (the rotation is linear)."""
    dev = _cuda()
    torch.manual_seed(5)
    f, m = fused.rotary_frequencies(20, scaling="yarn", factor=4.0, device=dev)
    x = torch.randn(2, 19, 3, 24, device=dev, requires_grad=True)
    dx, dy = torch.randn_like(x), torch.randn_like(x)
    y = fused.rotary(x, 3, f, True, m)
    (g,) = torch.autograd.grad(y, x, dy)
    step = (fused.rotary(x.detach() + dx, 3, f, True, m) - fused.rotary(x.detach() - dx, 3, f, True, m)).double() / 2
    left, right = (dy.double() * step).sum(), (g.double() * dx.double()).sum()
    # 12 u of |a| + |b| <= 20 on each of 2736 terms of random sign: sqrt(2736) * 20 * 12 * 2^-24 * |dy|
    assert abs(left - right) < 4 * math.sqrt(x.numel()) * 20 * 12 * 2.0 ** -24


@gpu
def test_empty_and_missing_gradients():
    dev = _cuda()
    f, m = fused.rotary_frequencies(8, device=dev)
    for shape in ((0, 4, 2, 8), (2, 0, 2, 8), (2, 4, 0, 8)):
        x = torch.randn(shape, device=dev).requires_grad_()
        y = fused.rotary(x, 0, f)
        assert y.shape == x.shape
        assert torch.autograd.grad(y.sum(), x)[0].shape == x.shape
    q = torch.randn(1, 3, 2, 8, device=dev, requires_grad=True)
    k = torch.randn(1, 3, 1, 8, device=dev, requires_grad=True)
    yq, yk = fused.rotary_qk(q, k, 1, f)
    gq, gk = torch.autograd.grad(yk.sum(), (q, k), allow_unused=True)  # a sum's gradient has no strides of its own
    assert gq is None or not gq.any()
    _check(gk, *_ref(torch.ones_like(k), torch.arange(3, device=dev) + 1, f, False, 1.0, -1.0))
    y = fused.rotary(q, 1, f)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(y.sum(), q, create_graph=True)


@gpu
def test_refusals_gpu():
    dev = _cuda()
    f = fused.rotary_frequencies(8, device=dev)[0]
    x = torch.randn(2, 3, 2, 8, device=dev)
    for call in (lambda: fused.rotary(x, torch.zeros(3, device=dev), f),
                 lambda: fused.rotary(x, torch.zeros(4, dtype=torch.long, device=dev), f),
                 lambda: fused.rotary(x, torch.zeros(3, 2, dtype=torch.long, device=dev), f),
                 lambda: fused.rotary(x, torch.zeros(3, dtype=torch.long), f),
                 lambda: fused.rotary(x, 0, f.cpu()), lambda: fused.rotary(x, 0, f.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="rotary"):
            call()


@gpu
def test_captured_and_replayed_on_another_stream():
    dev = _cuda()
    torch.manual_seed(6)
    f, m = fused.rotary_frequencies(64, device=dev)
    q, k = torch.randn(4, 1, 8, 64, device=dev).half(), torch.randn(4, 1, 2, 64, device=dev).half()
    pos = torch.zeros(4, 1, dtype=torch.long, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fused.rotary_qk(q, k, pos, f)
    torch.cuda.current_stream().wait_stream(side)
    leaf = torch.randn(2, 9, 3, 4, 64, device=dev).half().requires_grad_()
    start, grad = torch.zeros(9, dtype=torch.int32, device=dev), torch.randn(2, 9, 3, 4, 64, device=dev).half()

    def train():
        y = fused.rotary_qkv(leaf, start, f, interleaved=True)
        return [y.detach(), *torch.autograd.grad(y, leaf, grad)]

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        yq, yk = fused.rotary_qk(q, k, pos, f)
        trained = train()
    for step in range(4):
        pos += 1000 * step + 1
        start += 7
        g.replay()
        torch.cuda.synchronize()
        eq, ek = fused.rotary_qk(q, k, pos, f)
        assert torch.equal(yq, eq) and torch.equal(yk, ek)
        for a, b in zip(trained, train()):
            assert torch.equal(a, b)


@gpu
def test_more_tokens_than_one_launch_takes():
    """2^24 blocks of 256 threads are 2^32 work items, one more than a launch holds: refused by name."""
    dev = _cuda()
    f = fused.rotary_frequencies(2, device=dev)[0]
    x = torch.ones(1, 1, 1, 2, device=dev, dtype=torch.bfloat16).expand(3, 1_500_000_000, 1, 2)
    with pytest.raises(RuntimeError, match="rotary: too many tokens"):
        fused.rotary(x, 0, f)
