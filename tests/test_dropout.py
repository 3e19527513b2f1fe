"""Dropout from a counter (devspace_amd.ops.fused.dropout*) against its definition in 64 bits."""
import math

import numpy as np
import pytest
import torch

from devspace_amd.ops import fused

gpu = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SEED = 0x1234567_89ABCDEF


def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    fused.ext()
    return torch.device("cuda")


def _philox(counter, key):
    """Ten rounds of Philox 4x32 on Python's whole numbers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def _factor(shape, p, seed, offset=0):
    """The same on numpy's 64-bit words: 1 / (1 - p) where an element stays, else 0."""
    u = np.uint64
    d = shape[-1]
    rows = int(np.prod(shape[:-1]))
    n = (d + 3) // 4
    low = u(0xFFFFFFFF)
    row = np.repeat(np.arange(rows, dtype=u), n)
    c = [np.tile(np.arange(n, dtype=u), rows), row & low, row >> u(32), np.full(rows * n, offset, dtype=u)]
    k = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> u(32)) ^ c[1] ^ u(k[0]), b & low, (a >> u(32)) ^ c[3] ^ u(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    words = np.stack(c, -1).reshape(rows, 4 * n)[:, :d].reshape(shape)
    return torch.from_numpy((words >= u(round(p * 2 ** 32))).astype(np.float64)) * (1 / (1 - p) if p < 1 else 0.0)


def _half_step(t):
    return torch.finfo(t).eps / 2


def _close(got, ref, before, extra=0.0):
    """Half a step of the output's type on the result, and `before` (a tensor: what the 32-bit steps may
    be off), 2^-25 for half a step of the smallest halves."""
    tol = _half_step(got.dtype) * (1 + 1e-4) * ref.abs() + before + (2.0 ** -25 if got.dtype == torch.float16 else 0.0) + extra
    err = (got.double().cpu() - ref).abs()
    assert (err <= tol).all(), float((err - tol).max())


U = 2.0 ** -24


def test_published_words():
    """The known answers of Philox 4x32-10 that its authors give for zeros and for all ones."""
    assert _philox([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert _philox([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_cpu_mask_is_the_definition():
    shape = (3, 5, 11)
    want = _factor(shape, 0.3, SEED, offset=9)
    x = torch.ones(shape, dtype=torch.float64)
    assert torch.equal(fused.dropout(x, 0.3, SEED, offset=9), want)
    assert torch.equal(fused.dropout(x, 0.3, torch.tensor(SEED), offset=9), want)
    word = _philox([10 // 4, 7, 0, 9], [SEED & 0xFFFFFFFF, SEED >> 32])[10 % 4]
    assert (want.view(15, 11)[7, 10] != 0) == (word >= round(0.3 * 2 ** 32))
    big = (1 << 64) - 3  # a seed over 63 bits is the same 64 bits as its negative
    assert torch.equal(fused.dropout(x, 0.3, big), fused.dropout(x, 0.3, -3))
    assert not torch.equal(fused.dropout(x, 0.3, 1), fused.dropout(x, 0.3, 2))
    assert torch.equal(fused.dropout(x, 0.0, 1), x) and not fused.dropout(x, 1.0, 1).any()


def test_cpu_gradients_against_differences():
    torch.manual_seed(0)
    x, d = (torch.randn(2, 3, 5, dtype=torch.float64, requires_grad=True) for _ in range(2))
    w = torch.randn(5, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda a: fused.dropout(a, 0.4, 7), (x,))
    assert torch.autograd.gradcheck(lambda a, b: fused.dropout_add(a, b, 0.4, 7), (x, d))
    assert torch.autograd.gradcheck(lambda a, b, c: fused.dropout_add_rms_norm(a, b, c, 0.4, 7, eps=1e-5), (x, d, w))


def test_kept_share():
    """Of n independent elements a share within 5 sqrt(p (1 - p) / n) of 1 - p stays (a chance of 6e-7)."""
    for p in (0.1, 0.5, 0.9):
        kept = (fused.dropout(torch.ones(400, 1000), p, 3) != 0).double().mean().item()
        assert abs(kept - (1 - p)) < 5 * math.sqrt(p * (1 - p) / 400000)


def test_refusals_cpu():
    x, w = torch.randn(2, 4), torch.randn(4)
    for call in (lambda: fused.dropout(x.long(), 0.1, 0), lambda: fused.dropout(x, -0.1, 0), lambda: fused.dropout(x, 1.1, 0), lambda: fused.dropout(x, 0.1, 1 << 64),
                 lambda: fused.dropout(x, 0.1, 0, offset=1 << 32), lambda: fused.dropout(x, 0.1, torch.zeros(2).long()),
                 lambda: fused.dropout(x, float("nan"), 0), lambda: fused.dropout_add(x, x[:1], 0.1, 0),
                 lambda: fused.dropout_add(x, x.double(), 0.1, 0), lambda: fused.dropout_add_rms_norm(x, x, w[:2], 0.1, 0),
                 lambda: fused.dropout_add_rms_norm(x, x, w.double(), 0.1, 0), lambda: fused.Dropout(2.0)):
        with pytest.raises(ValueError):
            call()


def test_module_repeats_with_the_generator():
    m = fused.Dropout(0.5)
    x, r = torch.randn(4, 64), torch.randn(4, 64)
    torch.manual_seed(5)
    a, b = m(x), m(x)
    torch.manual_seed(5)
    assert torch.equal(a, m(x)) and not torch.equal(a, b)
    torch.manual_seed(5)
    torch.testing.assert_close(m(x, r), r + a)
    m.eval()
    assert m(x) is x and torch.equal(m(x, r), r + x)


SHAPES = [((1, 1), 0.5), ((3, 7), 0.1), ((2, 5, 8), 0.25), ((4, 1023), 0.9), ((33, 1024), 0.1), ((5, 4100), 0.5), ((70001, 3), 0.3)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,p", SHAPES)
def test_dropout_and_add_forward_and_backward(dtype, shape, p):
    dev, dt = _cuda(), DTYPES[dtype]
    torch.manual_seed(1)
    x, d = (torch.randn(shape, device=dev).to(dt).requires_grad_() for _ in range(2))
    g = torch.randn_like(x)
    factor = _factor(shape, p, SEED, 3)
    y = fused.dropout(x, p, SEED, offset=3)
    (gx,) = torch.autograd.grad(y, x, g)
    for got, src in ((y, x), (gx, g)):  # one product in 32 bits, its factor rounded too: 2 u
        ref = src.detach().double().cpu() * factor
        _close(got, ref, 2 * U * ref.abs())
        assert torch.equal((got.detach() == 0).cpu(), (ref == 0))
    s = fused.dropout_add(x, d, p, SEED, offset=3)
    ga, gd = torch.autograd.grad(s, (x, d), g)
    add = d.detach().double().cpu() * factor
    ref = x.detach().double().cpu() + add
    _close(s, ref, U * (2 * add.abs() + ref.abs()))
    assert torch.equal(ga, g) and torch.equal(gd, gx)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 24), (37, 768), (64, 1023), (5, 2048), (9, 2051), (6, 4096), (3, 8191), (2, 16384),
                                      (4097, 64), (20003, 22), (777, 100), (301, 130)])
@pytest.mark.parametrize("use", ["both", "y", "s"])
def test_dropout_add_rms_norm_forward_and_backward(dtype, rows, dim, use):
    dev, dt = _cuda(), DTYPES[dtype]
    torch.manual_seed(2)
    p, eps = 0.2, 1e-5
    x, d = (torch.randn(rows, dim, device=dev).to(dt).requires_grad_() for _ in range(2))
    w = (1 + 0.1 * torch.randn(dim, device=dev)).to(dt).requires_grad_()
    dy, ds = torch.randn_like(x), torch.randn_like(x)
    s, y = fused.dropout_add_rms_norm(x, d, w, p, SEED, eps=eps)
    outs, gs = {"both": ((s, y), (ds, dy)), "y": ((y,), (dy,)), "s": ((s,), (ds,))}[use]
    gx, gd, gw = torch.autograd.grad(outs, (x, d, w), gs)

    f64 = lambda t: t.detach().double().cpu()  # noqa: E731
    factor = _factor((rows, dim), p, SEED)
    t = f64(x) + f64(d) * factor
    r = (t.square().mean(-1, keepdim=True) + eps).rsqrt()
    # the sum in 32 bits: 3 u of its parts; a sum of D squares by at most D / 64 + 16 steps, so r by that many u
    part = (f64(x).abs() + 2 * f64(d).abs() * factor) * U
    steps = dim / 64 + 16
    _close(s, t, part)
    _close(y, t * r * f64(w), part * r * f64(w).abs() + steps * U * (t * r * f64(w)).abs())
    cy = f64(dy) if use != "s" else torch.zeros_like(t)
    cs = f64(ds) if use != "y" else torch.zeros_like(t)
    u = cy * f64(w)
    dot = (u * t).sum(-1, keepdim=True)
    g = cs + r * u - t * r ** 3 * dot / dim
    # the backward pass in 32 bits: the sum is off by 3 u of its parts, its row's sum by `steps` u of its terms' sizes
    size = (u * t).abs().sum(-1, keepdim=True) + (u.abs() * part / U).sum(-1, keepdim=True)
    before = t.abs() * r ** 3 / dim * 4 * steps * U * size + part * r ** 3 / dim * dot.abs() + \
        4 * steps * U * (cs.abs() + (r * u).abs())
    _close(gx, g, before)
    _close(gd, g * factor, before * factor + 2 * U * (g * factor).abs())
    terms = (cy * r).abs() * (t.abs() + part / U)
    _close(gw, (cy * t * r).sum(0), (steps + rows / 8 + 40) * U * terms.sum(0), extra=1e-30)


@gpu
def test_not_finite_and_edge_probabilities():
    dev = _cuda()
    x = torch.tensor([[math.inf, -math.inf, math.nan, 1.0] * 16] * 4, device=dev)
    factor = _factor((4, 64), 0.5, 1).to(dev)
    y = fused.dropout(x, 0.5, 1)
    assert (y[factor == 0] == 0).all()
    assert torch.equal(y[factor != 0].nan_to_num(7.0), (2 * x)[factor != 0].nan_to_num(7.0))
    assert torch.equal(fused.dropout_add(torch.ones_like(x), x, 1.0, 1), torch.ones_like(x))
    assert not fused.dropout(x, 1.0, 1).any()
    assert torch.equal(fused.dropout(x[:, 3:4], 0.0, 1), x[:, 3:4])


@gpu
def test_cpu_and_gpu_masks_agree_and_strides():
    dev = _cuda()
    x = torch.randn(6, 5, 37)
    want = fused.dropout(x, 0.3, -5, offset=(1 << 32) - 1)
    y = x.to(dev)
    turned = y.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.empty(y.numel() + 1, device=dev)[1:].view_as(y).copy_(y)
    seed = torch.tensor([-5], device=dev)
    for z, s in ((y, -5), (turned, -5), (odd, (1 << 64) - 5), (y, seed)):
        torch.testing.assert_close(fused.dropout(z, 0.3, s, offset=(1 << 32) - 1).cpu(), want, atol=0, rtol=2 * U)
    leaf = torch.randn(37, device=dev, requires_grad=True)  # broadcast over rows: each row has its own mask
    (g,) = torch.autograd.grad(fused.dropout(leaf.expand(8, 37), 0.3, 4).sum(), leaf)
    torch.testing.assert_close(g.double().cpu(), _factor((8, 37), 0.3, 4).sum(0), atol=1e-5, rtol=0)


@gpu
def test_empty_and_refusals_gpu():
    dev = _cuda()
    for shape in ((0, 4), (4, 0)):
        x = torch.randn(shape, device=dev, requires_grad=True)
        w = torch.ones(shape[-1], device=dev, requires_grad=True)
        assert fused.dropout(x, 0.1, 0).shape == shape
        s, y = fused.dropout_add_rms_norm(x, x, w, 0.1, 0)
        assert torch.autograd.grad(y.sum(), w)[0].shape == w.shape
    scalar = torch.ones((), device=dev)
    assert fused.dropout(scalar, 0.5, 0).shape == ()
    x, w = torch.randn(2, 16385, device=dev), torch.ones(16385, device=dev)
    for call in (lambda: fused.dropout_add_rms_norm(x, x, w, 0.1, 0), lambda: fused.dropout(x, 0.1, torch.tensor(1)),
                 lambda: fused.dropout_add_rms_norm(x[:, :4], x[:, :4], torch.ones(4), 0.1, 0)):
        with pytest.raises(RuntimeError, match="dropout"):
            call()
    x = torch.randn(2, 8, device=dev, requires_grad=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(fused.dropout(x, 0.1, 0).sum(), x, create_graph=True)
    seed = torch.tensor([3], device=dev)
    y = fused.dropout(x, 0.1, seed)
    seed += 1  # the backward pass would draw another mask
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@gpu
def test_captured_step_reads_its_seed_at_each_replay():
    dev = _cuda()
    torch.manual_seed(3)
    x, d = (torch.randn(64, 256, device=dev).bfloat16().requires_grad_() for _ in range(2))
    w = torch.ones(256, device=dev).bfloat16().requires_grad_()
    seed = torch.tensor([1], device=dev)
    gs, gy = torch.randn_like(x), torch.randn_like(x)

    def step():
        s, y = fused.dropout_add_rms_norm(x, d, w, 0.3, seed, offset=2)
        z = fused.dropout(y, 0.5, seed)
        grads = torch.autograd.grad((s, z), (x, d, w), (gs, gy))
        return [s.detach(), y.detach(), z.detach(), *grads]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step()
    masks = []
    for n in range(4):
        seed.fill_(100 + n)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step()):
            assert torch.equal(a, b)
        masks.append(outs[0].clone())
    assert not torch.equal(masks[0], masks[1])


@gpu
def test_more_than_two_to_the_31_elements():
    """Rows past 2^32 bytes and 2^31 elements: the last rows against a call that sees only their counters."""
    dev = _cuda()
    rows, d = (1 << 21) + 5, 1032
    x = torch.ones(rows, d, device=dev, dtype=torch.float16)
    y = fused.dropout(x, 0.5, SEED)
    for row in (0, 1 << 20, (1 << 31) // d + 1, rows - 1):
        block = [_philox([c // 4, row, 0, 0], [SEED & 0xFFFFFFFF, SEED >> 32])[c % 4] for c in range(d)]
        want = torch.tensor([2.0 if b >= 1 << 31 else 0.0 for b in block], dtype=torch.float16)
        assert torch.equal(y[row].cpu(), want), row
    share = (y != 0).sum(dtype=torch.int64).item() / y.numel()
    assert abs(share - 0.5) < 5 * 0.5 / math.sqrt(y.numel())


@gpu
def test_norm_of_more_rows_than_one_launch_takes():
    """Rows beyond 2^22 blocks of four: x = 0 and delta = 1, so that s is the mask and y follows from its count."""
    dev = _cuda()
    rows, d = (1 << 24) + 6, 136
    s, y = fused.dropout_add_rms_norm(torch.zeros(rows, d, device=dev, dtype=torch.bfloat16),
                                      torch.ones(rows, d, device=dev, dtype=torch.bfloat16),
                                      torch.ones(d, device=dev, dtype=torch.bfloat16), 0.5, SEED, eps=0.0)
    for row in (0, (1 << 24) - 1, 1 << 24, rows - 1):
        words = [_philox([c // 4, row, 0, 0], [SEED & 0xFFFFFFFF, SEED >> 32])[c % 4] for c in range(d)]
        want = torch.tensor([2.0 if v >= 1 << 31 else 0.0 for v in words], dtype=torch.float64)
        assert torch.equal(s[row].double().cpu(), want), row
        ref = want * want.square().mean().rsqrt()
        assert ((y[row].double().cpu() - ref).abs() <= 1.01 * 2.0 ** -8 * ref).all(), row


def test_module_draws_from_the_cpu_generator_whatever_the_default_device():
    """On a GPU as default device the seed would come from the GPU's generator, and the call would wait for it; on
    `meta` there is none to draw from."""
    m, x = fused.Dropout(0.5), torch.randn(4, 64)
    torch.manual_seed(5)
    want = m(x)
    torch.manual_seed(5)
    with torch.device("meta"):
        seed_of_the_call = []
        real = fused.dropout
        fused.dropout = lambda t, p, seed, offset=0: seed_of_the_call.append(seed)
        try:
            m(x)
        finally:
            fused.dropout = real
    assert torch.equal(fused.dropout(x, 0.5, seed_of_the_call[0]), want)


@gpu
def test_module_draws_from_the_cpu_generator_with_a_gpu_as_default_device():
    dev = _cuda()
    m, x = fused.Dropout(0.5), torch.randn(4, 64, device=dev)
    torch.manual_seed(5)
    want = m(x)
    torch.cuda.manual_seed(99)  # another state of the GPU's generator changes nothing
    torch.default_generator.manual_seed(5)
    with dev:
        assert torch.equal(m(x), want)
