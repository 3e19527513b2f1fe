"""Cross attention (devspace_amd.ops.fused.cross_attention) against its formulas in 64 bits."""
import math

import pytest
import torch

from devspace_amd.ops import fused

gpu = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0 ** -24


def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    fused.ext()
    return torch.device("cuda")


def _inputs(dev, dt, b, tq, tk, h, g, d, seed=1, big=1.0):
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    q = (big * torch.randn(b, tq, h, d, device=dev, generator=gen)).to(dt).requires_grad_()
    kv = torch.randn(b, tk, 2, h // g, d, device=dev, generator=gen).to(dt).requires_grad_()
    return q, kv, torch.randn(b, tq, h, d, device=dev, generator=gen).to(dt)


def _tiny(dt):
    """What rounding or flushing takes from a value below the type's normal range: half of fp16's smallest step;
    bf16 and fp32 values below 2^-126 may become 0."""
    return 2.0 ** -25 if dt == torch.float16 else 2.0 ** -126


def _reference(q, kv, do, lengths, scale, h_step, tiny=0.0):
    """The results in 64 bits and, for each, how far a computation may be off that rounds the probabilities
    and dS to the 16-bit type (half a step h each) and does all else in 32 bits (u = 2^-24). Worst cases,
    not averages:
      scores: D products and sums, so (D + 8) u of scale sum |q k|; a probability is off by that share (twice:
        in the sum, too), by the sums over the keys, (n + 16) u, and by its rounding
      O: that share of sum P |v|; the output's rounding is added where the results are compared
      the backward pass's row sum dO . O reads the rounded O
      dS = P (dP - sum): P's share, and what dP and the sum are off; then rounded
      and for each probability, each dS and each of their products that is below the normal range: `tiny`
    """
    q, kv, do = (t.detach().double().cpu() for t in (q, kv, do))
    b, tq, hh, d = q.shape
    tk, n = kv.shape[1], kv.shape[3]
    grp = hh // n
    out = {k: torch.zeros_like(t) for k, t in (("o", q), ("dq", q), ("dkv", kv))}
    off = {k: torch.zeros_like(t) for k, t in out.items()}
    for i in range(b):
        m = tk if lengths is None else max(0, min(tk, int(lengths[i])))
        for j in range(hh if m else 0):
            k, v = kv[i, :m, 0, j // grp], kv[i, :m, 1, j // grp]
            x, y = q[i, :, j], do[i, :, j]
            s = scale * (x @ k.T)
            e_s = (d + 8) * U * (scale * (x.abs() @ k.abs().T)).amax(-1, keepdim=True)
            p = torch.softmax(s, -1)
            o = p @ v
            e_p = 2 * e_s + (m + 16) * U  # relative, without the rounding
            e_o = (h_step + e_p) * (p @ v.abs()) + tiny * (v.abs().sum(0) + m)
            out["o"][i, :, j], off["o"][i, :, j] = o, e_o
            dp = y @ v.T
            row = (y * o).sum(-1, keepdim=True)
            e_row = (y.abs() * (e_o * (1 + h_step) + h_step * o.abs())).sum(-1, keepdim=True) + \
                (d + 2) * U * (y.abs() * o.abs()).sum(-1, keepdim=True)
            ds = p * (dp - row)
            e_ds = h_step * ds.abs() + (1 + h_step) * p * (
                e_p * (dp - row).abs() + (d + 2) * U * (y.abs() @ v.abs().T) + e_row) + tiny * ((dp - row).abs() + 1)
            steps = (max(m, tq * grp) + 16) * U  # sums over the keys or over the rows
            out["dq"][i, :, j] = scale * ds @ k
            off["dq"][i, :, j] = scale * ((e_ds + steps * ds.abs()) @ k.abs() + tiny * m)
            out["dkv"][i, :m, 0, j // grp] += scale * ds.T @ x
            off["dkv"][i, :m, 0, j // grp] += scale * ((e_ds + steps * ds.abs()).T @ x.abs() + tiny * tq)
            out["dkv"][i, :m, 1, j // grp] += p.T @ y
            off["dkv"][i, :m, 1, j // grp] += ((h_step + e_p + steps) * p + tiny).T @ y.abs() + tiny * tq
    return out, off


def _check(name, got, ref, off):
    h = torch.finfo(got.dtype).eps / 2
    tol = off + h * (ref.abs() + off) + _tiny(got.dtype)
    err = (got.detach().double().cpu() - ref).abs()
    assert bool((err <= tol).all()), (name, float((err - tol).max()), float((err / tol).max()))


def _run(q, kv, do, lengths, scale=None):
    o = fused.cross_attention(q, kv, lengths, scale)
    dq, dkv = torch.autograd.grad(o, (q, kv), do)
    return {"o": o, "dq": dq, "dkv": dkv}


def _hold(got, q, kv, do, lengths, scale=None, tiny=None):
    ref, off = _reference(q, kv, do, lengths, q.shape[-1] ** -0.5 if scale is None else scale,
                          torch.finfo(q.dtype).eps / 2, _tiny(q.dtype) if tiny is None else tiny)
    for k in ref:
        assert got[k].shape == ref[k].shape and got[k].dtype == q.dtype
        _check(k, got[k], ref[k], off[k])


def test_cpu_form_and_its_gradients():
    torch.manual_seed(0)
    q = torch.randn(2, 3, 4, 8, dtype=torch.float64, requires_grad=True)
    kv = torch.randn(2, 5, 2, 2, 8, dtype=torch.float64, requires_grad=True)
    do = torch.randn_like(q)
    for lengths in (None, torch.tensor([3, 0])):
        got = _run(q, kv, do, lengths)
        ref, _ = _reference(q, kv, do, lengths, 8 ** -0.5, 0.0)
        for k in ref:
            torch.testing.assert_close(got[k], ref[k], atol=1e-12, rtol=0)
        assert torch.autograd.gradcheck(lambda a, b: fused.cross_attention(a, b, lengths), (q, kv))
    bad = kv.detach().clone()
    bad[0, 3:] = math.nan
    bad[1] = math.inf
    got = _run(q, bad.requires_grad_(), do, torch.tensor([3, 0]))
    assert all(t.isfinite().all() for t in got.values())


def test_refusals_cpu():
    q, kv = torch.randn(2, 3, 4, 8), torch.randn(2, 5, 2, 2, 8)
    for call in (lambda: fused.cross_attention(q[0], kv), lambda: fused.cross_attention(q, kv[:, :, 0]),
                 lambda: fused.cross_attention(q[:1], kv), lambda: fused.cross_attention(q, kv[..., :4]),
                 lambda: fused.cross_attention(q, kv.double()), lambda: fused.cross_attention(q[:, :, :3], kv),
                 lambda: fused.cross_attention(q, kv, torch.tensor([1])), lambda: fused.cross_attention(q, kv, torch.ones(2)),
                 lambda: fused.cross_attention(q, kv, scale=0.0), lambda: fused.cross_attention(q, kv, scale=math.inf)):
        with pytest.raises(ValueError):
            call()


CASES = [  # dtype, B, Tq, Tk, H, G, D, lengths
    ("bf16", 1, 1, 1, 1, 1, 8, None),
    ("bf16", 2, 1, 100, 4, 1, 64, (100, 37)),
    ("fp16", 3, 1, 333, 8, 8, 128, (0, 1, 333)),
    ("bf16", 1, 1, 5000, 16, 4, 128, None),
    ("bf16", 2, 8, 700, 8, 4, 80, (700, 129)),
    ("fp16", 2, 33, 65, 2, 1, 64, (64, 65)),
    ("bf16", 1, 11, 63, 6, 3, 40, None),
    ("bf16", 2, 130, 257, 2, 1, 96, (257, 128)),
    ("fp16", 3, 77, 190, 8, 4, 72, (190, 0, 5)),
    ("bf16", 1, 257, 130, 4, 2, 128, None),
    ("fp16", 1, 513, 64, 2, 1, 64, None),
    ("bf16", 4, 64, 512, 4, 1, 64, (512, 1, 300, 449)),
    ("bf16", 1, 2000, 31, 2, 1, 104, None),
    ("fp16", 1, 3, 2000, 2, 1, 16, (1999,)),
    ("fp16", 2, 40, 2, 4, 1, 64, None),  # few states: dO . O nearly equals dP
    ("bf16", 1, 1000, 3000, 1, 1, 64, None),  # both axes split
    ("bf16", 1, 200, 900, 14, 7, 128, (899,)),  # tiles that begin inside a token's group of heads
    ("fp16", 2, 31, 64, 5, 5, 88, (64, 63)),
    ("bf16", 3, 800, 1500, 2, 1, 64, (1500, 0, 600)),  # many rows joined
]


@gpu
@pytest.mark.parametrize("dtype,b,tq,tk,h,g,d,lengths", CASES)
def test_forward_and_backward(dtype, b, tq, tk, h, g, d, lengths):
    dev = _cuda()
    q, kv, do = _inputs(dev, DTYPES[dtype], b, tq, tk, h, g, d)
    n = None if lengths is None else torch.tensor(lengths, device=dev, dtype=torch.int32)
    got = _run(q, kv, do, n)
    _hold(got, q, kv, do, n)
    again = _run(q, kv, do, None if n is None else n.long())
    for k in got:
        assert torch.equal(got[k], again[k]), k
    with torch.no_grad():
        assert torch.equal(fused.cross_attention(q, kv, n), got["o"])


@gpu
@pytest.mark.parametrize("dtype,tq,g,d", [("bf16", 1, 1, 64), ("fp16", 70, 2, 128), ("bf16", 40, 4, 80)])
def test_a_single_state(dtype, tq, g, d):
    """Its softmax is constant: O = V to the bit, dQ = dK = 0 exactly."""
    dev = _cuda()
    q, kv, do = _inputs(dev, DTYPES[dtype], 2, tq, 5, 4, g, d, big=3.0)
    n = torch.tensor([1, 0], device=dev)
    for x, lengths in ((kv, n), (kv[:, :1], None)):
        x = x.detach().clone().requires_grad_()
        got = _run(q, x, do, lengths)
        _hold(got, q, x, do, lengths)
        assert not got["dq"].any() and not got["dkv"][:, :, 0].any()
        assert torch.equal(got["o"][0], x[0, :1, 1].repeat_interleave(g, 1).expand(tq, -1, -1))


@gpu
def test_frozen_states_and_frozen_queries():
    dev = _cuda()
    q, kv, do = _inputs(dev, torch.bfloat16, 2, 50, 1000, 4, 2, 64)
    want = _run(q, kv, do, None)
    (dq,) = torch.autograd.grad(fused.cross_attention(q, kv.detach()), q, do)
    (dkv,) = torch.autograd.grad(fused.cross_attention(q.detach(), kv), kv, do)
    assert torch.equal(dq, want["dq"]) and torch.equal(dkv, want["dkv"])


@gpu
@pytest.mark.parametrize("tq,g", [(1, 1), (40, 2)])
def test_sharp_rows_and_another_scale(tq, g):
    """Scores of tens: the running maximum moves, most probabilities vanish."""
    dev = _cuda()
    q, kv, do = _inputs(dev, torch.bfloat16, 2, tq, 300, 4, g, 64, big=6.0)
    _hold(_run(q, kv, do, None, 0.3), q, kv, do, None, 0.3)


@gpu
def test_fp16_keeps_small_probabilities_and_large_gradients():
    """A long source: each probability is far below fp16's normal range (2^-14), where half a step would be 2^-25. They
    are lifted by 2^15, so that is 2^-40; dS by as much as its column's largest allows, so 2^-39 of that (under 8)."""
    dev = _cuda()
    q, kv, do = _inputs(dev, torch.float16, 1, 20, 30000, 2, 1, 64)
    do = do * 64  # gradients in the normal range
    _hold(_run(q, kv, do, None), q, kv, do, None, tiny=2.0 ** -36 * 64)
    one = q.detach()[:, :1].clone().requires_grad_()
    _hold(_run(one, kv, do[:, :1].contiguous(), None), one, kv, do[:, :1], None, tiny=2.0 ** -36 * 64)
    # few states, large gradients of the output: dS beyond 65504, all results within it
    q, kv, do = _inputs(dev, torch.float16, 1, 2, 3, 2, 1, 128, big=1e-3)
    kv = (kv.detach() * torch.tensor([1.0, 2.0], device=dev).half()[:, None, None]).requires_grad_()
    do = (do * 2e4).clamp(-6e4, 6e4)  # (3.3 standard deviations of them are beyond fp16)
    got = _run(q, kv, do, None)
    assert all(t.isfinite().all() for t in got.values())
    _hold(got, q, kv, do, None)


@gpu
@pytest.mark.parametrize("tq", [1, 100])
def test_states_behind_the_length_are_never_read(tq):
    dev = _cuda()
    n = torch.tensor([70, 0, 128], device=dev)
    q, kv, do = _inputs(dev, torch.float16, 3, tq, 200, 4, 2, 64)
    want = _run(q, kv, do, n)
    poisoned = kv.detach().clone()
    for i, m in enumerate(n.tolist()):
        poisoned[i, m:] = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(torch.float16).min] * 16, device=dev).half()
    got = _run(q, poisoned.requires_grad_(), do, n)
    for k in want:
        assert torch.equal(got[k], want[k])
    assert not got["o"][1].any() and not got["dq"][1].any() and not got["dkv"][1].any() and not got["dkv"][0, 70:].any()
    clamped = _run(q, kv, do, torch.tensor([70, -5, 1000], device=dev))["o"]
    assert torch.equal(clamped[1], want["o"][1])
    assert torch.equal(clamped[2], _run(q, kv, do, None)["o"][2])


@gpu
@pytest.mark.parametrize("tq", [1, 64])
def test_not_finite_states(tq):
    dev = _cuda()
    q, kv, _ = _inputs(dev, torch.bfloat16, 1, tq, 256, 2, 1, 64)
    q, kv = q.detach().abs(), kv.detach()
    kv[0, :96, 0] = -math.inf  # whole tiles of scores of -inf in front: those states do not count
    want = fused.cross_attention(q, kv[:, 96:].contiguous()).float()
    torch.testing.assert_close(fused.cross_attention(q, kv).float(), want, atol=2 * 2.0 ** -8 * want.abs().max().item(), rtol=0)
    kv[0, :, 0] = -math.inf
    assert fused.cross_attention(q, kv).isnan().all()  # as a softmax of nothing but -inf
    kv[0, :, 0] = 0.0
    kv[0, 200, 1, 0, 3] = math.nan
    o = fused.cross_attention(q, kv)
    assert o[0, :, 0, 3].isnan().all() and o.isnan().sum() == tq


@gpu
def test_strides():
    dev = _cuda()
    q, kv, do = _inputs(dev, torch.bfloat16, 2, 37, 90, 4, 2, 64)
    n = torch.tensor([90, 41], device=dev)
    want = _run(q, kv, do, n)
    a, c = q.detach(), kv.detach()

    def odd(t):  # an address that is no multiple of 16
        return torch.empty(t.numel() + 1, device=dev, dtype=t.dtype)[1:].view_as(t).copy_(t)

    heads_first = lambda t: t.transpose(1, -2).contiguous().transpose(1, -2)  # noqa: E731
    last = lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2)  # noqa: E731
    longer = torch.cat((c, torch.full_like(c, math.nan)), 1)[:, :90]
    for x, y, g in ((heads_first(a), c, do), (a, heads_first(c), do), (odd(a), odd(c), odd(do)), (last(a), last(c), last(do)),
                    (a, longer, heads_first(do))):
        got = _run(x.requires_grad_(), y.requires_grad_(), g, n)
        for k in want:
            assert torch.equal(got[k], want[k])
    one = c[:1].clone().requires_grad_()  # one source for both sequences: its gradient is the sum
    full = one.detach().expand(2, -1, -1, -1, -1).contiguous().requires_grad_()
    x = a.clone().requires_grad_()
    o = fused.cross_attention(x, one.expand(2, -1, -1, -1, -1), n)
    (g1,) = torch.autograd.grad(o, one, do)
    o2 = fused.cross_attention(x, full, n)
    (g2,) = torch.autograd.grad(o2, full, do)
    assert torch.equal(o, o2)
    torch.testing.assert_close(g1[0].float(), g2.float().sum(0), atol=0, rtol=2.0 ** -7)
    step = torch.arange(4, device=dev)[::2] * 0 + torch.tensor([90, 41], device=dev)
    strided = torch.stack((step, step), 1)[:, 0]
    assert torch.equal(fused.cross_attention(a, c, strided), want["o"])


@gpu
def test_gradient_against_differences():
    """A step along a random direction, both ways: the loss's difference against <gradient, direction>."""
    dev = _cuda()
    q, kv, do = _inputs(dev, torch.float16, 1, 40, 70, 2, 1, 64, seed=7)
    n = torch.tensor([61], device=dev)
    got = _run(q, kv, do, n)
    f64 = lambda t: t.detach().double().cpu()  # noqa: E731
    for name, x in (("dq", q), ("dkv", kv)):
        d = torch.randn(x.shape, dtype=torch.float64)
        losses = []
        for sign in (1, -1):
            a = f64(q) + (1e-4 * sign * d if name == "dq" else 0)
            c = f64(kv) + (1e-4 * sign * d if name == "dkv" else 0)
            losses.append((fused.cross_attention(a, c, n.cpu()) * f64(do)).sum())
        slope = (losses[0] - losses[1]) / 2e-4
        ref, off = _reference(q, kv, do, n, 64 ** -0.5, 2.0 ** -11, 2.0 ** -25)
        tol = ((off[name] + 2.0 ** -11 * (ref[name].abs() + off[name]) + 2.0 ** -25) * d.abs()).sum()
        assert abs(slope - (f64(got[name]) * d).sum()) <= tol + 1e-5 * abs(slope)


@gpu
def test_empty_and_refusals_gpu():
    dev = _cuda()
    for b, tq, tk in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q, kv, do = _inputs(dev, torch.bfloat16, b, tq, tk, 2, 1, 64)
        got = _run(q, kv, do, None)
        assert got["o"].shape == q.shape and got["dkv"].shape == kv.shape
        assert not any(t.any() for t in got.values())
    q, kv, do = _inputs(dev, torch.bfloat16, 1, 2, 3, 2, 1, 64)
    for call in (lambda: fused.cross_attention(q[..., :12], kv[..., :12]),
                 lambda: fused.cross_attention(torch.cat([q] * 3, -1), torch.cat([kv] * 3, -1))):
        with pytest.raises(RuntimeError, match="multiple of 8 up to 128"):
            call()
    many = torch.zeros(1 << 24, 1, 1, 8, device=dev, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="workgroups"):
        fused.cross_attention(many, many[:, :, None].expand(-1, -1, 2, -1, -1))
    with pytest.raises(RuntimeError, match="2\\^20"):
        fused.cross_attention(torch.zeros(1, 1, 1 << 15, 64, device=dev).half(), torch.zeros(1, 1, 2, 1, 64, device=dev).half())
    with pytest.raises(ValueError, match="lengths"):
        fused.cross_attention(q, kv, torch.tensor([3]))
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(fused.cross_attention(q, kv).sum(), q, create_graph=True)
    wide = fused.cross_attention(q.float(), kv.float())  # 32 bits: PyTorch ops
    torch.testing.assert_close(wide, fused.cross_attention(q.double(), kv.double()).float(), atol=1e-5, rtol=0)


@gpu
def test_far_offsets():
    """More than 2^32 elements of states: only the last one counts."""
    dev = _cuda()
    tk, heads, d = 1_100_003, 8, 128
    q = torch.randn(2, 1, heads, d, device=dev).bfloat16()
    kv = torch.zeros(2, tk, 2, heads, d, device=dev, dtype=torch.bfloat16)
    assert kv.numel() > 1 << 32
    kv[:, -1, 0] = 40 * q[:, 0]
    kv[:, -1, 1] = torch.randn(2, heads, d, device=dev).bfloat16()
    # its score is 40 |q|^2 / sqrt(128) > 200, all others 0: their probabilities are 0 in 32 bits
    assert torch.equal(fused.cross_attention(q, kv)[:, 0], kv[:, -1, 1])


@gpu
def test_far_offsets_trained():
    """The same for tiles of rows and their gradients: 2.25 * 2^30 elements of states in one sequence."""
    dev = _cuda()
    tk, heads, d, tq = 1_100_003, 8, 128, 40
    q = torch.randn(1, 1, heads, d, device=dev).bfloat16().expand(1, tq, heads, d).contiguous().requires_grad_()
    kv = torch.zeros(1, tk, 2, heads, d, device=dev, dtype=torch.bfloat16)
    kv[:, -1, 0] = 40 * q[:, 0].detach()
    kv[:, -1, 1] = torch.randn(1, heads, d, device=dev).bfloat16()
    kv.requires_grad_()
    do = torch.randn(1, tq, heads, d, device=dev).bfloat16()
    o = fused.cross_attention(q, kv)
    assert torch.equal(o, kv[:, -1:, 1].expand_as(o))
    dq, dkv = torch.autograd.grad(o, (q, kv), do)
    want = do.double().sum(1)  # P = 1 for the last state: 40 terms summed in 32 bits, rounded once
    off = (dkv[:, -1, 1].double() - want).abs()
    assert (off <= 2.0 ** -8 * want.abs() + 40 * U * do.double().abs().sum(1)).all()
    assert not dkv[:, :-1].any()
    # dS = dP - dO . O: both sums of 128 products in 32 bits; times K of up to 40 * 5 and its scale
    assert dq.abs().max() <= 256 * U * 128 * 25 * 200


@gpu
def test_captured_with_lengths_read_at_each_replay():
    dev = _cuda()
    q, kv, do = _inputs(dev, torch.bfloat16, 2, 40, 600, 4, 2, 64)
    one = torch.randn(2, 1, 4, 64, device=dev).bfloat16()
    n = torch.tensor([600, 10], device=dev)

    def step():
        o = fused.cross_attention(q, kv, n)
        return [o.detach(), *torch.autograd.grad(o, (q, kv), do), fused.cross_attention(one, kv.detach(), n)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step()
    for lengths in ((600, 10), (1, 599), (0, 300), (64, 65)):
        n.copy_(torch.tensor(lengths))
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step()):
            assert torch.equal(a, b)


def _short_reference(q, kv, do, lengths, scale, h_step, tiny):
    """_reference's gradients of sequences of 1 to 64 states, where the row sum is taken from the unrounded P and dP, in
    32 bits: it is off by P's share and dP's of each of its terms and by (m + 8) u of their sizes, not by O's
    rounding. A single state's dQ and dK are 0 exactly."""
    q, kv, do = (t.detach().double().cpu() for t in (q, kv, do))
    b, tq, hh, d = q.shape
    grp = hh // kv.shape[3]
    dq, dkv = torch.zeros_like(q), torch.zeros_like(kv)
    off_q, off_kv = torch.zeros_like(q), torch.zeros_like(kv)
    for i, m in enumerate(lengths):
        for j in range(hh if m else 0):
            k, v = kv[i, :m, 0, j // grp], kv[i, :m, 1, j // grp]
            x, y = q[i, :, j], do[i, :, j]
            p = torch.softmax(scale * (x @ k.T), -1)
            e_p = 2 * (d + 8) * U * (scale * (x.abs() @ k.abs().T)).amax(-1, keepdim=True) + (m + 16) * U
            steps = (max(m, tq * grp) + 16) * U
            dkv[i, :m, 1, j // grp] += p.T @ y
            off_kv[i, :m, 1, j // grp] += ((h_step + e_p + steps) * p + tiny).T @ y.abs() + tiny * tq
            if m == 1:
                continue
            dp = y @ v.T
            e_dp = (d + 2) * U * (y.abs() @ v.abs().T)
            row = (p * dp).sum(-1, keepdim=True)
            e_row = (p * ((e_p + (m + 8) * U) * dp.abs() + e_dp)).sum(-1, keepdim=True)
            ds = p * (dp - row)
            e_ds = h_step * ds.abs() + (1 + h_step) * p * (e_p * (dp - row).abs() + e_dp + e_row) + tiny * ((dp - row).abs() + 1)
            dq[i, :, j] = scale * ds @ k
            off_q[i, :, j] = scale * ((e_ds + steps * ds.abs()) @ k.abs() + tiny * m)
            dkv[i, :m, 0, j // grp] += scale * ds.T @ x
            off_kv[i, :m, 0, j // grp] += scale * ((e_ds + steps * ds.abs()).T @ x.abs() + tiny * tq)
    return {"dq": (dq, off_q), "dkv": (dkv, off_kv)}


@gpu
@pytest.mark.parametrize("dtype,b,tq,tk,h,g,d,lengths,big", [
    ("bf16", 5, 40, 1500, 2, 1, 64, (1500, 1, 2, 64, 0), 1.0),
    ("bf16", 4, 17, 1500, 4, 4, 128, (1, 63, 3, 1499), 4.0),
    ("fp16", 3, 1, 6000, 2, 2, 80, (2, 1, 33), 1.0),
    ("fp16", 3, 300, 770, 1, 1, 96, (1, 5, 64), 4.0),
    ("bf16", 3, 40, 64, 2, 1, 64, (2, 1, 64), 4.0),  # one tile, for comparison: no split
])
def test_short_sources_beside_long_ones(dtype, b, tq, tk, h, g, d, lengths, big):
    """How exact a sequence's gradients are goes by its own length: a long axis beside it, for which the launch is split,
    changes nothing."""
    dev = _cuda()
    q, kv, do = _inputs(dev, DTYPES[dtype], b, tq, tk, h, g, d, big=big)
    n = torch.tensor(lengths, device=dev)
    got = _run(q, kv, do, n)
    _hold(got, q, kv, do, n)
    short = [i for i, m in enumerate(lengths) if m <= 64]
    ref = _short_reference(q[short], kv[short], do[short], [lengths[i] for i in short], d ** -0.5,
                           torch.finfo(q.dtype).eps / 2, _tiny(q.dtype))
    for k, (want, off) in ref.items():
        _check(k, got[k][short], want, off)
    for i in short:
        if lengths[i] <= 1:
            assert not got["dq"][i].any() and not got["dkv"][i, :, 0].any()
    # the same bits as with nothing but its first 64 states around it
    alone = _run(q, kv.detach()[:, :64].clone().requires_grad_(), do, n.clamp(max=64))
    for i in short:
        assert torch.equal(alone["dq"][i], got["dq"][i]) and torch.equal(alone["dkv"][i], got["dkv"][i, :64])


@gpu
@pytest.mark.parametrize("tk", [(1 << 31) - 1_000_000, (1 << 31) - 129])
@pytest.mark.parametrize("tq", [1, 33])
def test_almost_two_to_the_31_states(tk, tq):
    """Sums of positions that pass 32 bits: where parts end, how many parts there are, tiles fetched ahead. The last two
    states have equal scores of 1018, the others 0: their probabilities are 0 in 32 bits, together too (2^31 e^-1018)."""
    dev = _cuda()
    if torch.cuda.get_device_properties(0).total_memory < 200 << 30:
        pytest.skip("needs 140 GB for the states and their gradients")
    torch.cuda.empty_cache()
    kv = torch.zeros(1, tk, 2, 1, 8, device=dev, dtype=torch.bfloat16)
    gen = torch.Generator(device=dev)
    gen.manual_seed(1)
    kv[0, -2:, 0, 0] = torch.tensor([[120.0] * 8, [240.0, 0.0] * 4], device=dev).bfloat16()
    kv[0, -2:, 1] = torch.randn(2, 1, 8, device=dev, generator=gen).bfloat16()
    q = torch.full((1, tq, 1, 8), 3.0, device=dev, dtype=torch.bfloat16).requires_grad_()
    do = torch.randn(1, tq, 1, 8, device=dev, generator=gen).bfloat16()
    last = kv[:, -2:].clone()
    o = fused.cross_attention(q, kv.requires_grad_())
    dq, dkv = torch.autograd.grad(o, (q, kv), do)
    _hold({"o": o, "dq": dq, "dkv": dkv[:, -2:]}, q, last, do, None)
    assert dq.any() and not dkv[:, :-2].any()
    # a source that ends where the parts of its axis are being counted
    n = torch.tensor([tk - 1], device=dev)
    with torch.no_grad():
        assert torch.equal(fused.cross_attention(q, kv, n), last[:, :1, 1].expand(1, tq, 1, 8))
    del kv, dkv
    torch.cuda.empty_cache()


@gpu
def test_almost_two_to_the_31_rows():
    """The same for the rows, over which dK and dV are split: only the last rows have a gradient."""
    dev = _cuda()
    if torch.cuda.get_device_properties(0).total_memory < 200 << 30:
        pytest.skip("needs 160 GB for the rows and their gradients")
    torch.cuda.empty_cache()
    rows = (1 << 31) - 129
    q = torch.zeros(1, rows, 1, 8, device=dev, dtype=torch.bfloat16)
    do = torch.zeros_like(q)
    gen = torch.Generator(device=dev)
    gen.manual_seed(1)
    q[:, -9:] = torch.randn(1, 9, 1, 8, device=dev, generator=gen).bfloat16()
    do[:, -9:] = torch.randn(1, 9, 1, 8, device=dev, generator=gen).bfloat16()
    kv = torch.randn(1, 5, 2, 1, 8, device=dev, generator=gen).bfloat16().requires_grad_()
    last, grad = q[:, -9:].clone(), do[:, -9:].clone()
    o = fused.cross_attention(q.requires_grad_(), kv)
    dq, dkv = torch.autograd.grad(o, (q, kv), do)
    _hold({"o": o[:, -9:], "dq": dq[:, -9:], "dkv": dkv}, last, kv, grad, None)
    assert not dq[:, :-9].any()
    del q, do, o, dq
    torch.cuda.empty_cache()


@gpu
def test_more_blocks_of_states_than_a_launch_takes():
    """2^24 blocks of 128 states, all of one source, so that the call itself is small: the states' gradient is refused,
    the rest is not."""
    dev = _cuda()
    source = torch.ones(1, 1 << 19, 2, 1, 8, device=dev, dtype=torch.bfloat16, requires_grad=True)
    q = torch.ones(1 << 12, 1, 1, 8, device=dev, dtype=torch.bfloat16, requires_grad=True)
    o = fused.cross_attention(q, source.expand(1 << 12, -1, -1, -1, -1))
    assert torch.equal(o, q)
    (dq,) = torch.autograd.grad(o.sum(), q, retain_graph=True)
    # V is constant: dS is P times what O's rounding and two sums of 8 products leave, its sum with K = 1 no more
    assert not dq.float().abs().max() > 2 * 8 * 2.0 ** -8
    with pytest.raises(RuntimeError, match="blocks of 128 states"):
        torch.autograd.grad(o.sum(), source)
