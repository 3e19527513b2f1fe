// Rotary positions for gfx950: the pairs of columns of every head turned by pos * f_i.
//
//   theta = pos * f_i,  a' = m (a cos theta - b sin theta),  b' = m (a sin theta + b cos theta)
//   pair i of the first R columns: (i, i + R/2), or (2i, 2i + 1) interleaved; columns >= R are copied.
//   The backward pass is the same turn by -theta.
//
// The angle is held in turns and in 64 bits until its whole turns are taken off (a position of a
// million times a frequency of one, in 32 bits, is off by 0.06), then the sine and cosine are taken in
// 32 bits. They are computed, not read from a table: a block takes a few tokens, computes their R/2
// sines and cosines once into LDS and uses them for every head of q, k (and the packed v's copy), so
// their cost shrinks with the number of heads and any position works. Bound by memory: each element is
// read once and written once, in accesses of up to 16 bytes, neighbouring lanes on neighbouring
// columns and heads of a token. MI355X: 32749 tokens x 40 heads x 128 bf16, 126 us a pass (5.3 TB/s, a large
// copy reaches 5.0); 8 x 512 packed tokens x 16 heads x 64, 12 us; 16 single tokens 4 us, a launch's latency.
#include "fused_common.h"

#include <vector>

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 256;  // tokens per block at most

struct RotarySegment {  // the heads of one tensor
  const void* in;
  void* out;
  int64_t ib, it, ih, ob, ot, oh;  // strides in elements
  int heads;
  bool turn;  // false: copied (the packed projection's v)
};

struct RotaryParams {
  RotarySegment seg[3];
  const void* pos;   // null: start + t
  const double* freq;  // R/2 angles per position, radians
  int64_t start, pb, pt;
  int64_t tokens;  // B * T
  int nseg, D, R, T;
  int tokens_per_block, per_token, per_head;  // work items: of a token, of a head
  int turned, pad;                            // a head's items of turned pairs; floats of a token's cosines in LDS
  FastDiv by_token, by_head, by_T, by_half;
  float magnitude, sign;
  bool pos64;
};

// n values from LDS at 4 x N bytes' alignment
template <int N>
__device__ __forceinline__ void lds_floats(const float* p, float (&v)[N]) {
  if constexpr (N >= 4) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 x = *reinterpret_cast<const float4*>(p + i);
      v[i] = x.x, v[i + 1] = x.y, v[i + 2] = x.z, v[i + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = p[i];
  }
}

// The W pairs of a head from `pair` on, their cosines and sines at cs and sn.
template <typename E, int W, bool INTERLEAVED>
__device__ __forceinline__ void turn(const typename E::S* in, typename E::S* out, int pair, int half, const float* cs,
                                     const float* sn) {
  typedef typename E::S S;
  float c[W], s[W];
  lds_floats(cs, c);
  lds_floats(sn, s);
  if (INTERLEAVED) {
    auto x = load_pack<S, 2 * W>(in + 2 * pair);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float a = E::get(x.v[2 * i]), b = E::get(x.v[2 * i + 1]);
      x.v[2 * i] = E::put(a * c[i] - b * s[i]);
      x.v[2 * i + 1] = E::put(a * s[i] + b * c[i]);
    }
    store_pack<S, 2 * W>(out + 2 * pair, x);
  } else {
    auto x = load_pack<S, W>(in + pair), y = load_pack<S, W>(in + half + pair);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float a = E::get(x.v[i]), b = E::get(y.v[i]);
      x.v[i] = E::put(a * c[i] - b * s[i]);
      y.v[i] = E::put(a * s[i] + b * c[i]);
    }
    store_pack<S, W>(out + pair, x);
    store_pack<S, W>(out + half + pair, y);
  }
}

// The last n < 2 W pairs (or columns to copy) in pieces of W, W / 2, ... 1.
template <typename E, int W, bool INTERLEAVED>
__device__ __forceinline__ void turn_rest(const typename E::S* in, typename E::S* out, int pair, int half, const float* cs,
                                          const float* sn) {
  if ((half - pair) & W) {
    turn<E, W, INTERLEAVED>(in, out, pair, half, cs, sn);
    pair += W, cs += W, sn += W;
  }
  if constexpr (W > 1) turn_rest<E, W / 2, INTERLEAVED>(in, out, pair, half, cs, sn);
}
template <typename S, int W>
__device__ __forceinline__ void copy_rest(const S* in, S* out, int n) {
  if (n & W) {
    store_pack<S, W>(out, load_pack<S, W>(in));
    in += W, out += W;
  }
  if constexpr (W > 1) copy_rest<S, W / 2>(in, out, n);
}

// One work item: V pairs of one head of one token, or 2 V columns to copy; the last item of either kind may have
// fewer.
template <typename E, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rotary_kernel(RotaryParams p) {
  typedef typename E::S S;
  extern __shared__ __attribute__((aligned(16))) float lds[];  // [tokens][cos | sin], each padded to p.pad
  const int half = p.R >> 1;
  const int64_t token0 = (int64_t)blockIdx.x * p.tokens_per_block;
  const int n = (int)min((int64_t)p.tokens_per_block, p.tokens - token0);
  const int64_t b0 = token0 / p.T;
  const int t0 = (int)(token0 - b0 * p.T);
  for (unsigned u = threadIdx.x; u < (unsigned)(n * half); u += kThreads) {
    unsigned i;
    const unsigned j = p.by_half.divmod(u, i);
    const unsigned wrap = p.by_T.div(t0 + j);
    const int64_t b = b0 + wrap, t = t0 + j - (int64_t)wrap * p.T;
    double x = (double)(p.start + t);
    if (p.pos) {
      const int64_t at = b * p.pb + t * p.pt;
      x = p.pos64 ? (double)static_cast<const int64_t*>(p.pos)[at] : (double)static_cast<const int*>(p.pos)[at];
    }
    const double turns = x * (p.freq[i] * 0.15915494309189533577);
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    lds[2 * j * p.pad + i] = c * p.magnitude;
    lds[(2 * j + 1) * p.pad + i] = s * p.magnitude * p.sign;
  }
  __syncthreads();
  const unsigned items = (unsigned)n * p.per_token;
  for (unsigned u = threadIdx.x; u < items; u += kThreads) {
    unsigned rest, item;
    const unsigned j = p.by_token.divmod(u, rest);
    int h = (int)p.by_head.divmod(rest, item);
    int k = 0;
    while (k + 1 < p.nseg && h >= p.seg[k].heads) h -= p.seg[k++].heads;
    const RotarySegment& sg = p.seg[k];
    const unsigned wrap = p.by_T.div(t0 + j);
    const int64_t b = b0 + wrap, t = t0 + j - (int64_t)wrap * p.T;
    const S* in = static_cast<const S*>(sg.in) + b * sg.ib + t * sg.it + h * sg.ih;
    S* out = static_cast<S*>(sg.out) + b * sg.ob + t * sg.ot + h * sg.oh;
    const int pair = (int)item * V;
    if (sg.turn && pair < half) {
      const float* cs = lds + 2 * j * p.pad + pair;
      const float* sn = cs + p.pad;
      if (pair + V <= half) turn<E, V, INTERLEAVED>(in, out, pair, half, cs, sn);
      else if constexpr (V > 1) turn_rest<E, V / 2, INTERLEAVED>(in, out, pair, half, cs, sn);
    } else {
      const int c = sg.turn ? p.R + 2 * (pair - p.turned * V) : 2 * pair;
      if (c + 2 * V <= p.D) store_pack<S, 2 * V>(out + c, load_pack<S, 2 * V>(in + c));
      else if (c < p.D) copy_rest<S, V>(in + c, out + c, p.D - c);
    }
  }
}

void check_positions(const c10::optional<at::Tensor>& pos, int64_t B, int64_t T, const at::Device& dev) {
  if (!pos) return;
  TORCH_CHECK(pos->device() == dev, "rotary: positions must be on the device of the heads");
  TORCH_CHECK(pos->scalar_type() == at::kLong || pos->scalar_type() == at::kInt, "rotary: positions must be int64 or int32");
  TORCH_CHECK((pos->dim() == 1 && pos->size(0) == T) ||
                  (pos->dim() == 2 && (pos->size(0) == B || pos->size(0) == 1) && pos->size(1) == T),
              "rotary: positions must be [T], [1, T] or [B, T]");
}

template <typename E>
void launch_rotary(RotaryParams& p, bool interleaved, hipStream_t st) {
  // accesses of 16 bytes; of the half's size where that is less
  constexpr int kWide = 16 / (int)sizeof(typename E::S);
  const int half = p.R / 2;
  int v = kWide;
  while (v > half) v /= 2;
  p.turned = (half + v - 1) / v;
  // a head's items: its turned pairs, then its copied columns; a copied head needs no more than that
  p.per_head = std::max(p.turned + (p.D - p.R + 2 * v - 1) / (2 * v), (p.D + 2 * v - 1) / (2 * v));
  p.pad = (half + 3) / 4 * 4;
  int heads = 0;
  for (int i = 0; i < p.nseg; ++i) heads += p.seg[i].heads;
  TORCH_CHECK((int64_t)heads * p.per_head * kMaxTokens < (1ll << 31), "rotary: too many heads");
  p.per_token = heads * p.per_head;
  // about four items per thread, so that the sines' latency is shared, but not fewer blocks than CUs
  int tb = std::max(1, std::min(kMaxTokens, 4 * kThreads / std::max(1, p.per_token)));
  while (tb > 1 && ((p.tokens + tb - 1) / tb < 512 || tb * p.pad * 8 > 32768)) tb /= 2;
  p.tokens_per_block = tb;
  p.by_token = FastDiv((unsigned)p.per_token);
  p.by_head = FastDiv((unsigned)p.per_head);
  p.by_T = FastDiv((unsigned)p.T);
  p.by_half = FastDiv((unsigned)half);
  const int64_t blocks = (p.tokens + tb - 1) / tb;
  TORCH_CHECK(blocks < (1ll << 32) / kThreads, "rotary: too many tokens for one launch of fewer than 2^32 work items");
  const size_t lds = (size_t)tb * 2 * p.pad * sizeof(float);
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kThreads), lds, st, p); };
#define ROTARY_CASE(W)                                                                        \
  case W:                                                                                     \
    if constexpr (W <= kWide) {                                                               \
      interleaved ? go(rotary_kernel<E, W, true>) : go(rotary_kernel<E, W, false>);           \
    }                                                                                         \
    break;
  switch (v) {
    ROTARY_CASE(8)
    ROTARY_CASE(4)
    ROTARY_CASE(2)
    ROTARY_CASE(1)
  }
#undef ROTARY_CASE
  LAUNCH_CHECK();
}

at::Tensor unit_last(const at::Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }

// Turns each tensor [B, T, H_i, D] of `xs` (null ones are skipped); `packed`: one [B, T, 3, H, D], whose
// last slot is copied.
std::vector<at::Tensor> rotary_apply(std::vector<at::Tensor> xs, bool packed, const c10::optional<at::Tensor>& pos,
                                     int64_t start, const at::Tensor& freq, bool interleaved, double magnitude,
                                     bool inverse) {
  at::Tensor first;
  for (auto& x : xs)
    if (x.defined()) first = x;
  c10::DeviceGuard guard(first.device());
  const int64_t B = first.size(0), T = first.size(1), D = first.size(-1);
  RotaryParams p{};
  p.D = (int)D;
  p.R = (int)(2 * freq.numel());
  p.T = (int)T;
  p.tokens = B * T;
  p.start = start;
  p.magnitude = (float)magnitude;
  p.sign = inverse ? -1.f : 1.f;
  at::Tensor f = freq.contiguous();
  p.freq = f.data_ptr<double>();
  if (pos) {
    p.pos = pos->data_ptr();
    p.pos64 = pos->scalar_type() == at::kLong;
    p.pt = pos->stride(-1);
    p.pb = pos->dim() == 2 && pos->size(0) > 1 ? pos->stride(0) : 0;
  }
  std::vector<at::Tensor> outs;
  for (auto& x0 : xs) {
    if (!x0.defined()) {
      outs.emplace_back();
      continue;
    }
    auto x = unit_last(x0);
    x0 = x;  // stays alive until the launch
    auto y = at::empty(x.sizes(), x.options());
    outs.push_back(y);
    const int slots = packed ? 3 : 1, hd = packed ? 3 : 2;
    for (int k = 0; k < slots; ++k) {
      RotarySegment& s = p.seg[p.nseg++];
      s.in = static_cast<const char*>(x.data_ptr()) + (packed ? k * x.stride(2) * x.element_size() : 0);
      s.out = static_cast<char*>(y.data_ptr()) + (packed ? k * y.stride(2) * y.element_size() : 0);
      s.ib = x.stride(0), s.it = x.stride(1), s.ih = x.stride(hd);
      s.ob = y.stride(0), s.ot = y.stride(1), s.oh = y.stride(hd);
      s.heads = (int)x.size(hd);
      s.turn = k < 2;
    }
  }
  int64_t heads = 0;
  for (int i = 0; i < p.nseg; ++i) heads += p.seg[i].heads;
  if (p.tokens == 0 || heads == 0) return outs;
  switch (first.scalar_type()) {
    case at::kBFloat16: launch_rotary<BF16>(p, interleaved, stream()); break;
    case at::kHalf: launch_rotary<FP16>(p, interleaved, stream()); break;
    default: launch_rotary<FP32>(p, interleaved, stream()); break;
  }
  return outs;
}

void check_rotary(const at::Tensor& x, const char* name, const at::Tensor& freq) {
  TORCH_CHECK(x.is_cuda(), "rotary: ", name, " must be a GPU tensor");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf || x.scalar_type() == at::kFloat,
              "rotary: ", name, " must be bfloat16, float16 or float32");
  TORCH_CHECK(freq.scalar_type() == at::kDouble && freq.dim() == 1 && freq.device() == x.device(),
              "rotary: freqs must be a 1-D float64 tensor on the device of ", name);
  TORCH_CHECK(!freq.requires_grad(), "rotary: no gradient flows to freqs");
  TORCH_CHECK(freq.numel() >= 1 && 2 * freq.numel() <= x.size(-1), "rotary: freqs must hold 1 to head_dim / 2 values");
  TORCH_CHECK(x.size(-1) <= 4096 && x.size(1) < (1ll << 31) - kMaxTokens, "rotary: head_dim <= 4096 and T < 2^31 wanted");
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct RotaryFn : public torch::autograd::Function<RotaryFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const c10::optional<at::Tensor>& k, bool packed,
                               const c10::optional<at::Tensor>& pos, int64_t start, const at::Tensor& freq,
                               bool interleaved, double magnitude) {
    ctx->save_for_backward({pos ? *pos : at::Tensor(), freq});
    ctx->saved_data["start"] = start;
    ctx->saved_data["packed"] = packed;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["magnitude"] = magnitude;
    ctx->set_materialize_grads(false);  // a tensor whose result was not used costs nothing
    std::vector<at::Tensor> xs{q};
    if (k) xs.push_back(*k);
    return rotary_apply(std::move(xs), packed, pos, start, freq, interleaved, magnitude, false);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_order("rotary");
    auto s = ctx->get_saved_variables();
    c10::optional<at::Tensor> pos;
    if (s[0].defined()) pos = s[0];
    bool any = false;
    for (auto& g : grads) any |= g.defined();
    variable_list d(grads.size());
    if (any)
      d = rotary_apply(grads, ctx->saved_data["packed"].toBool(), pos, ctx->saved_data["start"].toInt(), s[1],
                       ctx->saved_data["interleaved"].toBool(), ctx->saved_data["magnitude"].toDouble(), true);
    at::Tensor none;
    return {d[0], d.size() > 1 ? d[1] : none, none, none, none, none, none, none};
  }
};

std::vector<at::Tensor> rotary(const at::Tensor& q, const c10::optional<at::Tensor>& k, bool packed,
                               const c10::optional<at::Tensor>& pos, int64_t start, const at::Tensor& freq,
                               bool interleaved, double magnitude) {
  no_tangents("rotary", q, or_none(k), freq);
  check_rotary(q, packed ? "qkv" : "q", freq);
  TORCH_CHECK(q.dim() == (packed ? 5 : 4) && (!packed || q.size(2) == 3), "rotary: ",
              packed ? "qkv must be [B, T, 3, H, D]" : "heads must be [B, T, H, D]");
  if (k) {
    check_rotary(*k, "k", freq);
    TORCH_CHECK(k->dim() == 4 && k->size(0) == q.size(0) && k->size(1) == q.size(1) && k->size(3) == q.size(3) &&
                    k->scalar_type() == q.scalar_type() && k->device() == q.device(),
                "rotary: q and k must agree in B, T, D, type and device");
  }
  check_positions(pos, q.size(0), q.size(1), q.device());
  if (at::GradMode::is_enabled() && (q.requires_grad() || (k && k->requires_grad())))
    return RotaryFn::apply(q, k, packed, pos, start, freq, interleaved, magnitude);
  std::vector<at::Tensor> xs{q};
  if (k) xs.push_back(*k);
  return rotary_apply(std::move(xs), packed, pos, start, freq, interleaved, magnitude, false);
}

}  // namespace

void register_rotary(pybind11::module_& m) {
  m.def("rotary", &rotary, "rotary positions of [B, T, H, D] heads (one or two tensors) or a packed [B, T, 3, H, D]");
}
