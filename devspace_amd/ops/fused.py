"""Autograd wrappers around the gfx950 fused ops (fused_ops.hip, rotary.hip, dropout.hip, cross_attention.hip).

    from devspace_amd.ops import fused
    norm = fused.RMSNorm(dim)             # drop-in for nn.RMSNorm
    x, h = fused.add_rms_norm(x, delta, norm.weight)  # x += delta; h = norm(x), one kernel
    y = fused.swiglu(h)                   # silu(h[..., :H]) * h[..., H:]
    loss = fused.cross_entropy(logits, t) # mean CE on bf16 logits [N, V]
    qkv = fused.rotary_qkv(qkv, positions, freqs)     # q and k turned by their positions
    x, h = fused.dropout_add_rms_norm(x, delta, norm.weight, p, seed)  # no mask is stored
    o = fused.cross_attention(q, kv, lengths)         # over an encoder's states of another length

On a GPU the HIP kernels are mandatory for the types and sizes that an operator's docstring names: if
the in-tree extension is missing or broken the first call raises (no silent eager fallback). Other types
on a GPU (float64; float32 in cross_attention) and CPU tensors (tests, CPU smoke runs) take the plain
PyTorch formulation. The kernels have first derivatives in reverse mode; rotary, dropout and cross
attention refuse second and forward-mode ones on a GPU.
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

_ext = None
_ext_error = None


def _load_cached():
    """A copy of this package vendored into a project (`devspace init`, rocm-pytorch) has no
    in-tree build: compile into the cache (done at image build by the template's Dockerfile,
    else once on the first pod start) and load it from there."""
    import importlib.util

    from . import build

    path = build.ensure_fused_cached()
    spec = importlib.util.spec_from_file_location(f"{__package__}._fused_ops", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def ext():
    """The compiled extension module (raises with the build error on a GPU box)."""
    global _ext, _ext_error
    if _ext is None and _ext_error is None:
        try:
            from . import _fused_ops  # noqa: WPS433 - the in-tree (or image-built) extension

            _check_source(_fused_ops)  # a stale build raises here, on every call
            _ext = _fused_ops
        except ImportError as e:  # pragma: no cover - depends on the build
            try:
                _ext = _load_cached()
            except Exception as e2:  # no hipcc / ROCm headers in the image, build error
                _ext_error = f"{e}; building it failed: {e2}"
    if _ext is None:
        raise RuntimeError(f"devspace_amd fused HIP ops are not built ({_ext_error}); run "
                           "`python -m devspace_amd.ops.build --fused`")
    return _ext


def _check_source(mod) -> None:
    """An in-tree build must come from the sources next to it: kernels older than an edit of
    them must not run (an error, not a silent fallback)."""
    import os

    from . import build

    if os.path.exists(os.path.join(build.HERE, "fused_ops.hip")):
        built, src = getattr(mod, "source_sha", "unknown"), build.source_sha()
        if built != src:
            raise RuntimeError(f"the fused-ops extension is stale: built from source {built[:12]}, the source is "
                               f"{src[:12]}; run `python -m devspace_amd.ops.build --fused`")


def check_fresh() -> str:
    """The loaded extension was built from the sources next to it: returns their SHA-256, raises
    on a stale build (kernels older than the sources)."""
    from . import build

    _check_source(ext())
    return build.source_sha()


def backend() -> str:
    """"hip" when the gfx950 kernels are loaded (loading or compiling them now), else
    "eager (<why>)". For the training script's start-up line: never a silent fallback."""
    if not torch.cuda.is_available():
        return "eager (no GPU)"
    try:
        ext()
        return "hip"
    except RuntimeError as e:
        return f"eager ({e})"


def _use_hip(t: torch.Tensor) -> bool:
    return t.is_cuda and t.dtype == torch.bfloat16


# ------------------------------------------------------------------------------ ops
# The differentiable entry points are C++ autograd nodes inside the extension (no Python on
# the forward/backward path of the training step).


def _rmsnorm_kernel_default() -> bool:
    import os

    return os.environ.get("DEVSPACE_FUSED_RMSNORM", "1") != "0"


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float | None = None, kernel: bool | None = None) -> torch.Tensor:
    """RMSNorm alone: the gfx950 kernel by default (`kernel=False` or DEVSPACE_FUSED_RMSNORM=0 for
    PyTorch's fused rms_norm). Fwd+bwd on [4096x1024] it takes 25.2 us of device time against
    41.4 us (1.64x, replayed from a HIP graph); issued one call at a time from Python, both are
    bound by the host's dispatch (39.4 vs 40.6 us, 1.03x; round 5 measured 0.97x that way and
    kept it off). profiles/r6_fused_ops_ab_graph.txt. In a training step the device clock is the
    one that counts: the step is queued ahead of the GPU."""
    if eps is None:
        eps = torch.finfo(x.dtype).eps
    use = _rmsnorm_kernel_default() if kernel is None else kernel
    if use and _use_hip(x) and weight.dtype == torch.bfloat16 and ext().rmsnorm_supported(x.shape[-1]):
        return ext().rms_norm(x, weight, float(eps))
    return F.rms_norm(x, (x.shape[-1],), weight, eps)


def add_rms_norm(x: torch.Tensor, delta: torch.Tensor, weight: torch.Tensor, eps: float | None = None):
    """Residual add fused into the following RMSNorm: returns (s, y) with s = x + delta and
    y = rms_norm(s) * weight. On the GPU one kernel each way (no separate add kernel forward,
    no gradient-accumulation add backward)."""
    if eps is None:
        eps = torch.finfo(x.dtype).eps
    if (_use_hip(x) and delta.dtype == torch.bfloat16 and weight.dtype == torch.bfloat16 and delta.shape == x.shape
            and ext().rmsnorm_supported(x.shape[-1])):
        s, y = ext().add_rms_norm(x, delta, weight, float(eps))
        return s, y
    s = x + delta
    return s, F.rms_norm(s, (s.shape[-1],), weight, eps)


class RMSNorm(nn.Module):
    """nn.RMSNorm(dim) with the fused HIP forward/backward (same parameters, same eps default)."""

    def __init__(self, dim: int, eps: float | None = None):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim))

    def forward(self, x):
        return rms_norm(x, self.weight, self.eps)


def swiglu(h: torch.Tensor) -> torch.Tensor:
    """silu(g) * u for h = cat([g, u], -1) (the gate/up projection output)."""
    if _use_hip(h) and h.shape[-1] % 4 == 0:
        return ext().swiglu(h)
    g, u = h.chunk(2, dim=-1)
    return F.silu(g) * u


def cross_entropy(logits: torch.Tensor, target: torch.Tensor, ignore_index: int = -100) -> torch.Tensor:
    """Mean cross-entropy of [N, V] logits (computed in fp32 from bf16 logits, no fp32 copy)."""
    if _use_hip(logits) and logits.dim() == 2 and logits.shape[1] % 8 == 0 and target.dtype == torch.long:
        return ext().cross_entropy(logits, target, int(ignore_index))
    return F.cross_entropy(logits.float(), target, ignore_index=ignore_index)


def attention(qkv: torch.Tensor, causal: bool = True, scale: float | None = None) -> torch.Tensor:
    """Multi-head attention on the packed projection output qkv [B, T, 3, H, D] -> [B, T, H, D].

    HIP flash attention (MFMA, fwd + bwd) for bf16, D == 64, T % 128 == 0; otherwise
    F.scaled_dot_product_attention on transposed views."""
    b, t, three, h, d = qkv.shape
    if three != 3:
        raise ValueError("qkv must be [B, T, 3, H, D]")
    if scale is None:
        scale = d ** -0.5
    if _use_hip(qkv) and ext().attention_supported(qkv):
        return ext().attention(qkv, bool(causal), float(scale))
    q, k, v = qkv.unbind(2)
    o = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), is_causal=causal,
                                       scale=scale)
    return o.transpose(1, 2)


def cross_attention(q: torch.Tensor, kv: torch.Tensor, lengths: torch.Tensor | None = None,
                    scale: float | None = None) -> torch.Tensor:
    """Attention of queries q [B, Tq, H, D] over another sequence's states, kv [B, Tk, 2, N, D] (its packed
    key and value projection; N divides H, and H / N neighbouring heads share a key head) -> [B, Tq, H, D].

    lengths: int32 or int64 [B], how many of the Tk states each sequence has (None: all; values outside
    0..Tk are taken as the nearest). States behind them are never read, whatever they hold, and their
    gradients are 0; a sequence of no states gives 0. Any strides; Tq and Tk of any length, one query token
    included (serving). bfloat16 and float16 run the gfx950 kernels on a GPU (MFMA, forward and backward),
    with D a multiple of 8 up to 128, H times D up to 2^20 and fewer than 2^24 blocks (one per sequence, key head
    and 128 stacked query rows; the backward pass for kv, one per 128 states); float32 and float64 are computed in
    PyTorch ops."""
    if q.dim() != 4 or kv.dim() != 5 or kv.shape[2] != 2:
        raise ValueError("cross_attention: q must be [B, Tq, H, D] and kv [B, Tk, 2, N, D]")
    b, _, h, d = q.shape
    if kv.shape[0] != b or kv.shape[4] != d or q.dtype != kv.dtype or q.device != kv.device:
        raise ValueError("cross_attention: q and kv must agree in B, D, type and device")
    if kv.shape[3] == 0 or h == 0 or h % kv.shape[3]:
        raise ValueError("cross_attention: N must divide H")
    if lengths is not None and (lengths.shape != (b,) or lengths.dtype not in (torch.int32, torch.int64)
                                or lengths.device != q.device):
        raise ValueError("cross_attention: lengths must be int32 or int64 [B] on the device of q")
    if scale is None:
        scale = d ** -0.5
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError("cross_attention: scale must be positive")
    if q.is_cuda and q.dtype in (torch.bfloat16, torch.float16):
        return ext().cross_attention(q, kv, lengths, float(scale))
    return _cross_attention_eager(q, kv, lengths, scale)


def _cross_attention_eager(q, kv, lengths, scale):
    b, tq, h, d = q.shape
    tk, n = kv.shape[1], kv.shape[3]
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    kv = kv.to(wide)
    if lengths is not None:
        off = torch.arange(tk, device=q.device) >= lengths[:, None]
        kv = kv.masked_fill(off[:, :, None, None, None], 0.0)
    k, v = kv.permute(2, 0, 3, 1, 4)  # [B, N, Tk, D]
    rows = q.to(wide).reshape(b, tq, n, h // n, d).permute(0, 2, 3, 1, 4).reshape(b, n, -1, d)
    s = rows @ k.transpose(2, 3).contiguous() * scale
    if lengths is not None:
        s = s.masked_fill(off[:, None, None], -math.inf)
        p = torch.softmax(s, -1).masked_fill((lengths <= 0)[:, None, None, None], 0.0)
    else:
        p = torch.softmax(s, -1)
    return (p @ v.contiguous()).view(b, n, h // n, tq, d).permute(0, 3, 1, 2, 4).reshape(b, tq, h, d).to(q.dtype)


# ------------------------------------------------------------------------------ rotary positions


def rotary_frequencies(dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       original_length: int = 4096, fast: float = 32.0, slow: float = 1.0, device=None):
    """(freqs, magnitude) for rotary positions on the first `dim` columns of a head: freqs is a float64
    tensor of dim / 2 angles per position, base^(-2i/dim), scaled for contexts `factor` times as long:

      "linear"  every frequency divided by the factor (positions squeezed)
      "ntk"     the base raised to base * factor^(dim / (dim - 2)): the fastest pair keeps its
                frequency, the slowest is divided by the factor
      "yarn"    pairs that turn at least `fast` times within `original_length` keep their frequency,
                those that turn at most `slow` times are divided by the factor, a ramp between them;
                q and k are multiplied by the magnitude 0.1 ln(factor) + 1
    """
    if dim < 2 or dim % 2:
        raise ValueError("rotary_frequencies: dim must be even and at least 2")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise ValueError(f"rotary_frequencies: unknown scaling {scaling!r}")
    if base <= 0 or factor < 1 or original_length < 1 or fast <= slow:
        raise ValueError("rotary_frequencies: base > 0, factor >= 1, original_length >= 1 and fast > slow wanted")
    if scaling == "ntk" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    freqs = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    magnitude = 1.0
    if scaling == "linear":
        freqs = freqs / factor
    elif scaling == "yarn":
        turns = original_length * freqs / (2 * math.pi)
        keep = ((turns - slow) / (fast - slow)).clamp(0, 1)
        freqs = freqs * keep + freqs / factor * (1 - keep)
        magnitude = 0.1 * math.log(factor) + 1.0
    return freqs.to(device), magnitude


def _check_rotary(x, dims, freqs):
    if x.dim() != dims:
        raise ValueError("rotary: heads must be [B, T, H, D]" if dims == 4 else "rotary: qkv must be [B, T, 3, H, D]")
    if freqs.dtype != torch.float64 or freqs.dim() != 1 or not 1 <= freqs.numel() <= x.shape[-1] // 2:
        raise ValueError("rotary: freqs must be a 1-D float64 tensor of 1 to head_dim / 2 values")


def _rotary_eager(x, positions, freqs, interleaved, magnitude):
    """The formula in PyTorch ops (x [B, T, H, D]): angles in 64 bits, the turn in 32 (64 for float64)."""
    b, t, _, d = x.shape
    if not isinstance(positions, torch.Tensor):
        positions = torch.arange(t, device=x.device) + int(positions or 0)
    if positions.shape not in ((t,), (1, t), (b, t)) or positions.dtype not in (torch.int64, torch.int32):
        raise ValueError("rotary: positions must be int64 or int32 and [T], [1, T] or [B, T]")
    angle = (positions.double()[..., None] * freqs)[..., None, :]
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    cos, sin = (angle.cos() * magnitude).to(wide), (angle.sin() * magnitude).to(wide)
    n = freqs.numel()
    y = x.to(wide)
    u, v = (y[..., 0:2 * n:2], y[..., 1:2 * n:2]) if interleaved else (y[..., :n], y[..., n:2 * n])
    turned = (u * cos - v * sin, u * sin + v * cos)
    turned = torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1)
    return torch.cat((turned, y[..., 2 * n:]), -1).to(x.dtype)


_HIP_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def _rotary_hip(x, k, packed, positions, freqs, interleaved, magnitude):
    pos = positions if isinstance(positions, torch.Tensor) else None
    return ext().rotary(x, k, packed, pos, 0 if pos is not None else int(positions or 0), freqs, bool(interleaved),
                        float(magnitude))


def rotary(x: torch.Tensor, positions, freqs: torch.Tensor, interleaved: bool = False,
           magnitude: float = 1.0) -> torch.Tensor:
    """Rotary positions on heads x [B, T, H, D] (any strides): pair i of the first 2 * len(freqs) columns
    is turned by position * freqs[i] and multiplied by `magnitude`; the other columns are carried over.

    positions: an int64 or int32 tensor [T], [1, T] or [B, T], or a whole number: the position of
    token 0 (None: 0). interleaved: pairs are neighbouring columns (2i, 2i + 1) instead of
    (i, i + len(freqs)). Gradients flow to x. bfloat16, float16 and float32 run the gfx950 kernel on a GPU."""
    _check_rotary(x, 4, freqs)
    if x.is_cuda and x.dtype in _HIP_FLOATS:
        return _rotary_hip(x, None, False, positions, freqs, interleaved, magnitude)[0]
    return _rotary_eager(x, positions, freqs, interleaved, magnitude)


def rotary_qk(q: torch.Tensor, k: torch.Tensor, positions, freqs: torch.Tensor, interleaved: bool = False,
              magnitude: float = 1.0):
    """rotary() of queries [B, T, H, D] and keys [B, T, N, D] in one launch: (q', k')."""
    _check_rotary(q, 4, freqs)
    _check_rotary(k, 4, freqs)
    if q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3] or q.dtype != k.dtype or q.device != k.device:
        raise ValueError("rotary: q and k must agree in B, T, D, type and device")
    if q.is_cuda and q.dtype in _HIP_FLOATS:
        return tuple(_rotary_hip(q, k, False, positions, freqs, interleaved, magnitude))
    return tuple(_rotary_eager(x, positions, freqs, interleaved, magnitude) for x in (q, k))


def rotary_qkv(qkv: torch.Tensor, positions, freqs: torch.Tensor, interleaved: bool = False,
               magnitude: float = 1.0) -> torch.Tensor:
    """rotary() of the q and k of a packed projection [B, T, 3, H, D], v carried over: what attention()
    reads, in one launch."""
    _check_rotary(qkv, 5, freqs)
    if qkv.shape[2] != 3:
        raise ValueError("rotary: qkv must be [B, T, 3, H, D]")
    if qkv.is_cuda and qkv.dtype in _HIP_FLOATS:
        return _rotary_hip(qkv, None, True, positions, freqs, interleaved, magnitude)[0]
    q, k, v = qkv.unbind(2)
    return torch.stack([_rotary_eager(x, positions, freqs, interleaved, magnitude) for x in (q, k)] + [v], 2)


class Rotary(nn.Module):
    """Rotary positions of a model: keeps the frequencies (a buffer that stays float64 when the module is
    cast) and applies them to a packed qkv or to q and k."""

    def __init__(self, dim: int, interleaved: bool = False, base: float = 10000.0, scaling: str = "none",
                 factor: float = 1.0, original_length: int = 4096):
        super().__init__()
        self.interleaved = interleaved
        freqs, self.magnitude = rotary_frequencies(dim, base, scaling, factor, original_length)
        self.register_buffer("freqs", freqs, persistent=False)

    def _apply(self, fn, recurse=True):
        exact = self.freqs
        super()._apply(fn, recurse)
        if self.freqs.dtype != torch.float64:  # .bfloat16() and the like: move, but keep the exact values
            self.freqs = exact.to(self.freqs.device)
        return self

    def forward(self, q, k=None, positions=None):
        if k is None:
            return rotary_qkv(q, positions, self.freqs, self.interleaved, self.magnitude)
        return rotary_qk(q, k, positions, self.freqs, self.interleaved, self.magnitude)


# ------------------------------------------------------------------------------ dropout


def _check_dropout(op, p, seed, offset, dtype=torch.float32):
    if not dtype.is_floating_point:
        raise ValueError(f"{op}: floating-point data wanted")
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{op}: p must be within 0 and 1")
    if not 0 <= offset < 1 << 32:
        raise ValueError(f"{op}: offset must be within 0 and 2^32 - 1")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise ValueError(f"{op}: a seed tensor must hold one int64")
        return 0, seed
    if not -(1 << 63) <= seed < 1 << 64:
        raise ValueError(f"{op}: seed must fit 64 bits")
    return (int(seed) + (1 << 63)) % (1 << 64) - (1 << 63), None  # the same 64 bits with a sign


def _dropout_factor(shape, p, seed, offset, device):
    """1 / (1 - p) where an element of `shape` stays and 0 where it is dropped (float64): the words of
    Philox 4x32-10 in PyTorch ops, the gfx950 kernels' own."""
    low = (1 << 32) - 1
    d = shape[-1] if len(shape) else 1
    rows = math.prod(shape[:-1])
    c0 = torch.arange((d + 3) // 4, device=device).expand(rows, -1)
    row = torch.arange(rows, device=device)[:, None].expand_as(c0)
    c1, c2, c3 = row & low, row >> 32, torch.full_like(c0, offset)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # modulo 2^64: both halves are right
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack((c0, c1, c2, c3), -1).flatten(1)[:, :d].reshape(shape)
    return (words >= round(p * 2.0 ** 32)).double() * (1.0 / (1.0 - p) if p < 1.0 else 0.0)


def _dropped(x, p, seed, seed_at, offset):
    """x dropped and scaled, unrounded (float32, or float64 for float64)."""
    factor = _dropout_factor(x.shape, p, int(seed_at) if seed_at is not None else seed, offset, x.device)
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    return torch.where(factor != 0, x.to(wide) * factor.to(wide), torch.zeros((), dtype=wide, device=x.device))


def dropout(x: torch.Tensor, p: float, seed, offset: int = 0) -> torch.Tensor:
    """x with each element dropped with probability p, the others divided by 1 - p. The mask is a
    function of (seed, offset, row, column) of x seen as [rows, last dimension]; it is computed again
    in the backward pass and never stored. Dropped elements are 0, whatever they were.

    seed: a whole number of 64 bits, or a tensor of one int64 on the data's device (a captured graph
    reads it anew at each replay; it must not change between a forward pass and its backward pass).
    offset: 0 to 2^32 - 1, to tell the dropouts of one step apart. The masks are the same on every device."""
    seed, at = _check_dropout("dropout", p, seed, offset, x.dtype)
    if x.is_cuda and x.dtype in _HIP_FLOATS:
        return ext().dropout(x, None, float(p), seed, at, offset)
    return _dropped(x, p, seed, at, offset).to(x.dtype)


def dropout_add(x: torch.Tensor, delta: torch.Tensor, p: float, seed, offset: int = 0) -> torch.Tensor:
    """x + dropout(delta, p, seed, offset) in one kernel, rounded once."""
    seed, at = _check_dropout("dropout_add", p, seed, offset, x.dtype)
    if x.shape != delta.shape or x.dtype != delta.dtype or x.device != delta.device:
        raise ValueError("dropout_add: x and delta must agree in shape, type and device")
    if x.is_cuda and x.dtype in _HIP_FLOATS:
        return ext().dropout(delta, x, float(p), seed, at, offset)
    return (x + _dropped(delta, p, seed, at, offset)).to(x.dtype)


def dropout_add_rms_norm(x: torch.Tensor, delta: torch.Tensor, weight: torch.Tensor, p: float, seed,
                         eps: float | None = None, offset: int = 0):
    """add_rms_norm() of a residual stream with dropout: returns (s, y) with
    s = x + dropout(delta, p, seed, offset) and y = rms_norm(s) * weight, one kernel each way (and a
    small one for the weight's gradient). y and the gradients are made of the sum before it is rounded
    to s: the backward pass sums x and delta again. On a GPU rows (the last dimension) of up to 16384
    elements."""
    seed, at = _check_dropout("dropout_add_rms_norm", p, seed, offset, x.dtype)
    if x.shape != delta.shape or x.dtype != delta.dtype or x.device != delta.device:
        raise ValueError("dropout_add_rms_norm: x and delta must agree in shape, type and device")
    if x.dim() < 1 or weight.shape != x.shape[-1:] or weight.dtype != x.dtype:
        raise ValueError("dropout_add_rms_norm: weight must be [D] and of the data's type")
    if eps is None:
        eps = torch.finfo(x.dtype).eps
    if x.is_cuda and x.dtype in _HIP_FLOATS:
        return tuple(ext().dropout_add_rms_norm(x, delta, weight, float(eps), float(p), seed, at, offset))
    s = x + _dropped(delta, p, seed, at, offset)
    return s.to(x.dtype), (s * torch.rsqrt(s.square().mean(-1, keepdim=True) + eps) * weight).to(x.dtype)


class Dropout(nn.Module):
    """nn.Dropout(p) on the fused kernels. Each call takes its seed from PyTorch's CPU generator (so
    torch.manual_seed and checkpointed recomputation repeat it); `residual` is added in the same kernel.
    A captured graph keeps the seeds of its capture: inside one, call dropout() with a seed tensor."""

    def __init__(self, p: float = 0.5):
        super().__init__()
        _check_dropout("Dropout", p, 0, 0)
        self.p = p

    def forward(self, x, residual=None):
        if not self.training or self.p == 0.0:
            return x if residual is None else residual + x
        seed = int(torch.randint(-(1 << 63), (1 << 63) - 1, (), device="cpu"))  # whatever the default device is
        return dropout(x, self.p, seed) if residual is None else dropout_add(residual, x, self.p, seed)


# ------------------------------------------------------------------------------ AdamW


def _hip_ok(t: torch.Tensor) -> bool:
    return _use_hip(t) and t.is_contiguous() and t.data_ptr() % 16 == 0


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW (decoupled weight decay, no amsgrad) with a multi-tensor HIP update for
    bf16 GPU parameters: one launch per <= 48 tensors, moments kept in the parameter dtype like
    torch's fused AdamW. Other parameters (CPU, fp32, non-contiguous) take the same math in
    plain PyTorch ops."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2):
        if lr < 0 or eps < 0 or not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError("invalid AdamW hyper-parameters")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            lr, (b1, b2), eps, wd = group["lr"], group["betas"], group["eps"], group["weight_decay"]
            buckets = {}  # step -> lists for one multi-tensor launch
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW does not support sparse gradients")
                st = self.state[p]
                if not st:
                    st["step"] = 0
                    st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                    st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                st["step"] += 1
                g = p.grad
                if all(_hip_ok(t) for t in (p, g, st["exp_avg"], st["exp_avg_sq"])):
                    b = buckets.setdefault(st["step"], ([], [], [], []))
                    for lst, t in zip(b, (p, g, st["exp_avg"], st["exp_avg_sq"])):
                        lst.append(t)
                else:
                    _adamw_eager(p, g, st["exp_avg"], st["exp_avg_sq"], lr, b1, b2, eps, wd, st["step"])
            for step, (ps, gs, ms, vs) in buckets.items():
                ext().adamw_step(ps, gs, ms, vs, lr, b1, b2, eps, wd, step)
        return loss


def _adamw_eager(p, g, m, v, lr, b1, b2, eps, wd, step):
    pf, gf = p.float(), g.float()
    mf = m.float().mul_(b1).add_(gf, alpha=1 - b1)
    vf = v.float().mul_(b2).addcmul_(gf, gf, value=1 - b2)
    pf.mul_(1 - lr * wd)
    denom = vf.sqrt().div_((1 - b2 ** step) ** 0.5).add_(eps)
    pf.addcdiv_(mf, denom, value=-lr / (1 - b1 ** step))
    p.copy_(pf)
    m.copy_(mf)
    v.copy_(vf)
