// Dropout for gfx950 whose mask is computed from a counter and never stored, alone, with the residual's
// add, and with the residual's add and RMSNorm.
//
//   keep(row, col) <=> word[col % 4] of Philox(key = seed, counter = (col / 4, row, row >> 32, offset))
//                      >= round(p 2^32)
//   dropout               y = keep ? x / (1 - p) : 0
//   dropout_add           s = x + dropout(delta)
//   dropout_add_rms_norm  s as above, y = s r w, r = rsqrt(mean s^2 + eps)
//   backward of the last  g = ds + r w dy - s r^3 / D sum(w dy s), dx = g, ddelta = dropout(g),
//                         dw = sum over rows of dy s r, with s summed again from x and delta: the rounded
//                         s would weigh in dw (up to 1.75 times the rounding of dw itself)
//
// Philox 4x32 with ten rounds (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3",
// 2011): the backward pass computes the same words again instead of reading a mask. A block of four words
// belongs to four neighbouring columns of a row, so that eight elements (one access of 16 bytes in 16-bit
// types) are two blocks whatever the row's length. All of a row's math is in fp32; each output is rounded
// once, and y is made of the sum before its rounding.
//
// Bound by memory, the generator's work hidden behind it. MI355X: 32768 x 8192 bf16 forward and backward 381 us
// (5.6 TB/s, a large copy reaches 5.0); 4096 x 1024 bf16 add + norm 9.8 us forward (3.4 TB/s), 14.0 + 3.9 us
// backward (3.6 TB/s), a few us of each being the launch; 4095 x 1023 fp16 7.2 us a pass.
#include "fused_common.h"

#include <algorithm>
#include <type_traits>
#include <vector>

namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxNormDim = 16384;

struct Drop {
  const int64_t* seed_at;  // null: seed
  uint64_t seed;
  unsigned offset;
  unsigned last;  // the largest dropped word
  bool none;      // p rounds to 0: nothing is dropped
  float scale;    // 1 / (1 - p); 0 where p is 1
};

struct Key {
  unsigned k0, k1, offset, last;
  bool none;
  float scale;
  __device__ __forceinline__ explicit Key(const Drop& d) : offset(d.offset), last(d.last), none(d.none), scale(d.scale) {
    const uint64_t s = d.seed_at ? (uint64_t)*d.seed_at : d.seed;
    k0 = (unsigned)s;
    k1 = (unsigned)(s >> 32);
  }
};

__device__ __forceinline__ void philox(unsigned c0, unsigned c1, unsigned c2, unsigned c3, unsigned k0, unsigned k1,
                                       unsigned w[4]) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (unsigned)(b >> 32) ^ c1 ^ k0;
    c2 = (unsigned)(a >> 32) ^ c3 ^ k1;
    c1 = (unsigned)b;
    c3 = (unsigned)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0, w[1] = c1, w[2] = c2, w[3] = c3;
}

// Which of the eight elements at column 8 v of a row stay, a bit each.
__device__ __forceinline__ unsigned keep8(int64_t row, unsigned v, const Key& k) {
  unsigned bits = 0;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    unsigned w[4];
    philox(2 * v + q, (unsigned)row, (unsigned)((uint64_t)row >> 32), k.offset, k.k0, k.k1, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) bits |= (w[i] > k.last || k.none) ? 1u << (4 * q + i) : 0u;
  }
  return bits;
}
// They are scaled; what is dropped becomes 0 whatever it was (a product with the mask would make NaN of an infinity).
__device__ __forceinline__ void drop8(float f[8], unsigned bits, float scale) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = bits >> i & 1 ? f[i] * scale : 0.f;
}
__device__ __forceinline__ void drop8(float f[8], int64_t row, unsigned v, const Key& k) { drop8(f, keep8(row, v, k), k.scale); }

// Up to eight elements of a row as they are stored, 0 behind its end: one wide access, or the row's last n in pieces
// of four, two and one. EVEN: rows are whole groups of eight. They are widened where they are used, so that no load
// waits for another's values.
template <typename S, bool EVEN>
__device__ __forceinline__ Pack<S, 8> load8(const S* p, int n) {
  if (EVEN || n >= 8) return load_pack<S, 8>(p);
  const bool four = n & 4, two = n & 2, one = n & 1;
  const S zero = (S)0;
  Pack<S, 4> a = {{zero, zero, zero, zero}};
  Pack<S, 2> b = {{zero, zero}};
  S c = zero;
  if (four) a = load_pack<S, 4>(p);
  if (two) b = load_pack<S, 2>(p + (n & 4));
  if (one) c = p[n & 6];
  Pack<S, 8> x;
  x.v[0] = four ? a.v[0] : two ? b.v[0] : c;
  x.v[1] = four ? a.v[1] : b.v[1];
  x.v[2] = four ? a.v[2] : two ? c : zero;
  x.v[3] = a.v[3];
  x.v[4] = four ? (two ? b.v[0] : c) : zero;
  x.v[5] = four ? b.v[1] : zero;
  x.v[6] = four && two ? c : zero;
  x.v[7] = zero;
  return x;
}
template <typename E>
__device__ __forceinline__ void widen(const Pack<typename E::S, 8>& x, float f[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = E::get(x.v[i]);
}
template <typename E, bool EVEN>
__device__ __forceinline__ void store8(typename E::S* p, int n, const float f[8]) {
  typedef typename E::S S;
  Pack<S, 8> x;
#pragma unroll
  for (int i = 0; i < 8; ++i) x.v[i] = E::put(f[i]);
  if (EVEN || n >= 8) {
    store_pack<S, 8>(p, x);
  } else {
    const bool four = n & 4, two = n & 2;
    if (four) store_pack<S, 4>(p, Pack<S, 4>{{x.v[0], x.v[1], x.v[2], x.v[3]}});
    if (two) store_pack<S, 2>(p + (n & 4), Pack<S, 2>{{four ? x.v[4] : x.v[0], four ? x.v[5] : x.v[1]}});
    if (n & 1) p[n & 6] = four ? (two ? x.v[6] : x.v[4]) : (two ? x.v[2] : x.v[0]);
  }
}

// ------------------------------------------------------------------------------ dropout, dropout + add

// y = [x +] drop(d). Eight elements per work item; a launch covers rows row0.. with fewer than 2^31 items.
template <typename E, bool ADD, bool EVEN>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const typename E::S* __restrict__ d,
                                                           const typename E::S* __restrict__ x,
                                                           typename E::S* __restrict__ y, unsigned items, int64_t row0,
                                                           int D, FastDiv by_row, Drop drop) {
  const Key key(drop);
  for (unsigned u = blockIdx.x * kThreads + threadIdx.x; u < items; u += gridDim.x * kThreads) {
    unsigned v;
    const unsigned r = by_row.divmod(u, v);
    const int64_t row = row0 + r;
    const int64_t at = row * D + 8 * (int64_t)v;
    const int n = D - 8 * (int)v;
    const auto rd = load8<typename E::S, EVEN>(d + at, n);
    Pack<typename E::S, 8> rx;
    if (ADD) rx = load8<typename E::S, EVEN>(x + at, n);
    float f[8], g[8];
    widen<E>(rd, f);
    if (ADD) widen<E>(rx, g);
    drop8(f, row, v, key);
    if (ADD) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] += g[i];
    }
    store8<E, EVEN>(y + at, n, f);
  }
}

// ------------------------------------------------------------------------------ dropout + add + norm

// threads of a block that gives each row LANES lanes
constexpr int threads_for(int lanes) { return lanes < kThreads ? kThreads : lanes; }

// Sum over the lanes that share a row: part of a wave, a wave, or the block's waves through LDS, in their order.
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = (LANES < 64 ? LANES : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if constexpr (LANES <= 64) {
    return v;
  } else {
    __syncthreads();  // the last row's sums have been read
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < LANES / 64; ++i) t += red[i];
    return t;
  }
}

// LANES lanes per row (4 to 64, or the block's 256 to 1024), VPL groups of eight elements per lane: lane l owns groups l, l + LANES, ...
// and keeps them in registers between the sum of squares and the scaled store, so that each tensor passes once.
template <typename E, int LANES, int VPL, bool EVEN>
__global__ void __launch_bounds__(threads_for(LANES)) drop_norm_fwd_kernel(const typename E::S* __restrict__ x,
                                                                 const typename E::S* __restrict__ delta,
                                                                 const typename E::S* __restrict__ w,
                                                                 typename E::S* __restrict__ sum,
                                                                 typename E::S* __restrict__ y, float* __restrict__ rstd,
                                                                 int64_t row0, int64_t R, int D, float eps, Drop drop) {
  __shared__ float red[16];
  constexpr int kRows = threads_for(LANES) / LANES;  // of a block
  const int lane = threadIdx.x & (LANES - 1);
  const int64_t row = row0 + (int64_t)blockIdx.x * kRows + threadIdx.x / LANES;
  if (kRows > 1 && row >= R) return;
  const Key key(drop);
  const int nvec = (D + 7) >> 3;
  const int64_t base = row * D;
  // the weight is loaded with the row, not behind its sum
  Pack<typename E::S, 8> rx[VPL], rd[VPL], rw[VPL];
  float s[VPL][8];
#pragma unroll
  for (int k = 0; k < VPL; ++k) {
    const int i = lane + LANES * k;
    if (i < nvec) {
      rx[k] = load8<typename E::S, EVEN>(x + base + 8 * i, D - 8 * i);
      rd[k] = load8<typename E::S, EVEN>(delta + base + 8 * i, D - 8 * i);
      rw[k] = load8<typename E::S, EVEN>(w + 8 * i, D - 8 * i);
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < VPL; ++k) {
    const int i = lane + LANES * k;
    if (i < nvec) {
      float d[8];
      widen<E>(rx[k], s[k]);
      widen<E>(rd[k], d);
      drop8(d, row, i, key);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s[k][j] += d[j];
        ss += s[k][j] * s[k][j];  // columns behind the row are 0
      }
      store8<E, EVEN>(sum + base + 8 * i, D - 8 * i, s[k]);
    }
  }
  ss = row_sum<LANES>(ss, red);
  const float r = rsqrtf(ss / (float)D + eps);
  if (lane == 0) rstd[row] = r;
#pragma unroll
  for (int k = 0; k < VPL; ++k) {
    const int i = lane + LANES * k;
    if (i < nvec) {
      float wv[8];
      widen<E>(rw[k], wv);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[k][j] *= r * wv[j];
      store8<E, EVEN>(y + base + 8 * i, D - 8 * i, s[k]);
    }
  }
}

// A block owns rows_per_block rows (its groups of LANES lanes take turns); each lane adds the weight gradient of
// its columns in registers, and the block writes one fp32 row of partial sums, which part_sum_kernel adds in a
// fixed order.
template <typename E, int LANES, int VPL, bool EVEN>
__global__ void __launch_bounds__(threads_for(LANES)) drop_norm_bwd_kernel(
    const typename E::S* __restrict__ dy, const typename E::S* __restrict__ ds, const typename E::S* __restrict__ x,
    const typename E::S* __restrict__ delta, const typename E::S* __restrict__ w, const float* __restrict__ rstd, typename E::S* __restrict__ dx,
    typename E::S* __restrict__ dd, float* __restrict__ part, int64_t R, int D, int rows_per_block, Drop drop) {
  __shared__ float red[16];
  constexpr int kStep = threads_for(LANES) / LANES;  // groups
  extern __shared__ float sdw[];                     // [kStep][D], with more than one
  const int lane = threadIdx.x & (LANES - 1);
  const Key key(drop);
  const int nvec = (D + 7) >> 3;
  float acc[VPL][8];
#pragma unroll
  for (int k = 0; k < VPL; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[k][j] = 0.f;
  const int64_t r0 = (int64_t)blockIdx.x * rows_per_block, r1 = min(R, r0 + rows_per_block);
  const float inv_d = 1.0f / (float)D;
  typedef Pack<typename E::S, 8> Raw;
  Raw rw[VPL], rr[VPL], rg[VPL], rx[VPL], rd[VPL];
#pragma unroll
  for (int k = 0; k < VPL; ++k) {
    if (lane + LANES * k < nvec) rw[k] = load8<typename E::S, EVEN>(w + 8 * (lane + LANES * k), D - 8 * (lane + LANES * k));
  }
  for (int64_t row = r0 + threadIdx.x / LANES; row < r1; row += kStep) {
    const int64_t base = row * D;
    float g[VPL][8], sv[VPL][8];
    unsigned keep[VPL];
    float dot = 0.f;
    const float r = rstd[row];
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
      const int i = lane + LANES * k, n = D - 8 * i;
      if (i < nvec) {
        if (dy) rg[k] = load8<typename E::S, EVEN>(dy + base + 8 * i, n);
        rx[k] = load8<typename E::S, EVEN>(x + base + 8 * i, n);
        rd[k] = load8<typename E::S, EVEN>(delta + base + 8 * i, n);
        if (ds) rr[k] = load8<typename E::S, EVEN>(ds + base + 8 * i, n);
      }
    }
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
      if (lane + LANES * k < nvec) {
        float wv[8], d[8];
        keep[k] = keep8(row, lane + LANES * k, key);
        widen<E>(rg[k], g[k]);
        widen<E>(rx[k], sv[k]);
        widen<E>(rd[k], d);
        widen<E>(rw[k], wv);
        drop8(d, keep[k], key.scale);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          sv[k][j] += d[j];
          if (!dy) g[k][j] = 0.f;
          acc[k][j] += g[k][j] * sv[k][j] * r;
          g[k][j] *= wv[j];
          dot += g[k][j] * sv[k][j];
        }
      }
    }
    dot = row_sum<LANES>(dot, red);
    const float c = dot * r * r * r * inv_d;
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
      const int i = lane + LANES * k, n = D - 8 * i;
      if (i < nvec) {
        float rv[8];
        widen<E>(rr[k], rv);
#pragma unroll
        for (int j = 0; j < 8; ++j) g[k][j] = r * g[k][j] - sv[k][j] * c + (ds ? rv[j] : 0.f);
        store8<E, EVEN>(dx + base + 8 * i, n, g[k]);
        drop8(g[k], keep[k], key.scale);
        store8<E, EVEN>(dd + base + 8 * i, n, g[k]);
      }
    }
  }
  float* out = part + (int64_t)blockIdx.x * D;
  if constexpr (kStep > 1) {
    float* mine = sdw + threadIdx.x / LANES * D;
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
      const int i = lane + LANES * k;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (8 * i + j < D) mine[8 * i + j] = acc[k][j];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < D; c += kThreads) {
      float t = 0.f;
#pragma unroll
      for (int g = 0; g < kStep; ++g) t += sdw[g * D + c];
      out[c] = t;
    }
  } else {
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
      const int i = lane + LANES * k;
      if (i < nvec) store8<FP32, EVEN>(out + 8 * i, D - 8 * i, acc[k]);
    }
  }
}

// out[c] = sum over rows of part[row][c]: 32 columns per block, 32 groups of rows, added in a fixed order.
template <typename E>
__global__ void __launch_bounds__(1024) part_sum_kernel(const float* __restrict__ part, int rows, int D,
                                                        typename E::S* __restrict__ out) {
  __shared__ float red[32][33];
  const int cl = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + cl;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < D) {
    int r = g;
    for (; r + 3 * 32 < rows; r += 4 * 32) {
#pragma unroll
      for (int u = 0; u < 4; ++u) s[u] += part[(int64_t)(r + 32 * u) * D + c];
    }
    for (; r < rows; r += 32) s[0] += part[(int64_t)r * D + c];
  }
  red[g][cl] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (threadIdx.x < 32 && c < D) {
    float t = 0.f;
#pragma unroll 8
    for (int k = 0; k < 32; ++k) t += red[k][cl];
    out[c] = E::put(t);
  }
}

// ------------------------------------------------------------------------------ host side

Drop make_drop(double p, int64_t seed, const c10::optional<at::Tensor>& seed_at, int64_t offset) {
  Drop d{};
  d.seed = (uint64_t)seed;
  if (seed_at) d.seed_at = seed_at->data_ptr<int64_t>();
  d.offset = (unsigned)offset;
  const double words = std::nearbyint(p * 4294967296.0);  // words below this one are dropped
  d.none = words < 1.0;
  d.last = d.none ? 0u : (unsigned)(words - 1.0);
  d.scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.f;
  return d;
}

void check_drop(const char* op, const at::Tensor& x, double p, const c10::optional<at::Tensor>& seed_at, int64_t offset) {
  TORCH_CHECK(x.is_cuda(), op, ": GPU tensors wanted");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf || x.scalar_type() == at::kFloat, op,
              ": bfloat16, float16 or float32 wanted");
  TORCH_CHECK(p >= 0.0 && p <= 1.0, op, ": p must be within 0 and 1");
  TORCH_CHECK(offset >= 0 && offset < (1ll << 32), op, ": offset must be within 0 and 2^32 - 1");
  TORCH_CHECK(!seed_at || (seed_at->scalar_type() == at::kLong && seed_at->numel() == 1 && seed_at->device() == x.device()),
              op, ": a seed tensor must hold one int64 on the device of the data");
  TORCH_CHECK(x.dim() == 0 || x.size(-1) < (1ll << 31) - 8, op, ": rows of fewer than 2^31 elements wanted");
}

void same(const char* op, const char* name, const at::Tensor& a, const at::Tensor& b) {
  TORCH_CHECK(a.sizes() == b.sizes() && a.scalar_type() == b.scalar_type() && a.device() == b.device(), op, ": ", name,
              " must agree in shape, type and device");
}

template <typename F>
void by_type(at::ScalarType t, F&& f) {
  switch (t) {
    case at::kBFloat16: f(BF16{}); break;
    case at::kHalf: f(FP16{}); break;
    default: f(FP32{}); break;
  }
}

// drop(d), or x + drop(d); contiguous inputs
at::Tensor dropout_apply(const at::Tensor& d, const at::Tensor& x, const Drop& drop) {
  c10::DeviceGuard guard(d.device());
  auto y = at::empty_like(d);
  if (d.numel() == 0) return y;
  const int64_t D = d.dim() ? d.size(-1) : 1, R = d.numel() / D, nvec = (D + 7) / 8;
  const int64_t most = std::max<int64_t>(1, ((1ll << 30)) / nvec);  // rows of one launch: items stay under 2^31
  for (int64_t r0 = 0; r0 < R; r0 += most) {
    const int64_t items = std::min(most, R - r0) * nvec;
    const unsigned blocks = (unsigned)((items + kThreads - 1) / kThreads);
    by_type(d.scalar_type(), [&](auto e) {
      typedef decltype(e) E;
      typedef typename E::S S;
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kThreads), 0, stream(), (const S*)d.data_ptr(),
                           x.defined() ? (const S*)x.data_ptr() : nullptr, (S*)y.data_ptr(), (unsigned)items, r0, (int)D,
                           FastDiv((unsigned)nvec), drop);
      };
      if (D % 8 == 0) x.defined() ? go(dropout_kernel<E, true, true>) : go(dropout_kernel<E, false, true>);
      else x.defined() ? go(dropout_kernel<E, true, false>) : go(dropout_kernel<E, false, false>);
    });
    LAUNCH_CHECK();
  }
  return y;
}

// Lanes per row and groups per lane of the norm kernels: as many lanes as a narrow row has groups (several rows
// per wave: 4128008 rows x 22 forward and backward take 1 wave per row 8709 us, so 619), a wave per row up to 1024
// columns (no barrier, four rows in flight per block), a block per row beyond, never more than two groups a lane.
template <typename F>
void by_width(int64_t D, F&& g) {
  auto f = [&](auto lanes, auto vpl) {
    if (D % 8 == 0) g(lanes, vpl, std::true_type{});
    else g(lanes, vpl, std::false_type{});
  };
  constexpr std::integral_constant<int, 1> one{};
  constexpr std::integral_constant<int, 2> two{};
  const int64_t n = (D + 7) / 8;
  if (n <= 4) f(std::integral_constant<int, 4>{}, one);
  else if (n <= 16) f(std::integral_constant<int, 16>{}, one);
  else if (n <= 64) f(std::integral_constant<int, 64>{}, one);
  else if (n <= 128) f(std::integral_constant<int, 64>{}, two);
  else if (n <= 256) f(std::integral_constant<int, 256>{}, one);
  else if (n <= 512) f(std::integral_constant<int, 256>{}, two);
  else if (n <= 1024) f(std::integral_constant<int, 512>{}, two);
  else f(std::integral_constant<int, 1024>{}, two);
}

struct NormForward {
  at::Tensor sum, y, rstd;
};

NormForward drop_norm_fwd(const at::Tensor& x, const at::Tensor& delta, const at::Tensor& w, double eps, const Drop& drop) {
  c10::DeviceGuard guard(x.device());
  const int64_t D = x.size(-1), R = D ? x.numel() / D : 0;
  NormForward o{at::empty_like(x), at::empty_like(x), at::empty({R}, x.options().dtype(at::kFloat))};
  if (R == 0) return o;
  by_type(x.scalar_type(), [&](auto e) {
    typedef decltype(e) E;
    typedef typename E::S S;
    by_width(D, [&](auto lanes, auto vpl, auto even) {
      const int64_t at_once = threads_for(lanes) / lanes, most = at_once << 21;  // rows of one launch
      for (int64_t row0 = 0; row0 < R; row0 += most) {
        const int64_t blocks = (std::min(most, R - row0) + at_once - 1) / at_once;
        hipLaunchKernelGGL((drop_norm_fwd_kernel<E, lanes, vpl, even>), dim3((unsigned)blocks), dim3(threads_for(lanes)), 0, stream(),
                           (const S*)x.data_ptr(), (const S*)delta.data_ptr(), (const S*)w.data_ptr(), (S*)o.sum.data_ptr(),
                           (S*)o.y.data_ptr(), o.rstd.data_ptr<float>(), row0, R, (int)D, (float)eps, drop);
        LAUNCH_CHECK();
      }
    });
  });
  return o;
}

// dy or ds may be undefined (zero)
std::vector<at::Tensor> drop_norm_bwd(const at::Tensor& dy, const at::Tensor& ds, const at::Tensor& x, const at::Tensor& delta,
                                      const at::Tensor& w, const at::Tensor& rstd, const Drop& drop) {
  c10::DeviceGuard guard(x.device());
  const int64_t D = x.size(-1), R = D ? x.numel() / D : 0;
  auto dx = at::empty_like(x), dd = at::empty_like(x), dw = at::empty_like(w);
  if (R == 0) return {dx, dd, dw.zero_()};
  by_type(x.scalar_type(), [&](auto e) {
    typedef decltype(e) E;
    typedef typename E::S S;
    by_width(D, [&](auto lanes, auto vpl, auto even) {
      // two rows per group of lanes; at most 1024 rows of partial sums
      const int64_t at_once = threads_for(lanes) / lanes;
      const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>(1024, (R + 2 * at_once - 1) / (2 * at_once)));
      const int64_t per = (R + blocks - 1) / blocks;
      TORCH_CHECK(per < (1ll << 31), "dropout_add_rms_norm: too many rows");
      auto part = at::empty({blocks, D}, x.options().dtype(at::kFloat));
      hipLaunchKernelGGL((drop_norm_bwd_kernel<E, lanes, vpl, even>), dim3((unsigned)blocks), dim3(threads_for(lanes)),
                         at_once > 1 ? at_once * D * sizeof(float) : 0, stream(), dy.defined() ? (const S*)dy.data_ptr() : nullptr,
                         ds.defined() ? (const S*)ds.data_ptr() : nullptr, (const S*)x.data_ptr(),
                         (const S*)delta.data_ptr(), (const S*)w.data_ptr(),
                         rstd.data_ptr<float>(), (S*)dx.data_ptr(), (S*)dd.data_ptr(), part.data_ptr<float>(), R, (int)D,
                         (int)per, drop);
      LAUNCH_CHECK();
      hipLaunchKernelGGL((part_sum_kernel<E>), dim3((unsigned)((D + 31) / 32)), dim3(1024), 0, stream(),
                         part.data_ptr<float>(), (int)blocks, (int)D, (S*)dw.data_ptr());
      LAUNCH_CHECK();
    });
  });
  return {dx, dd, dw};
}

// ------------------------------------------------------------------------------ autograd

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef c10::optional<at::Tensor> OptTensor;

void save_drop(AutogradContext* ctx, double p, int64_t seed, int64_t offset) {
  ctx->saved_data["p"] = p;
  ctx->saved_data["seed"] = seed;
  ctx->saved_data["offset"] = offset;
}
Drop saved_drop(AutogradContext* ctx, const at::Tensor& seed_at) {
  OptTensor t;
  if (seed_at.defined()) t = seed_at;
  return make_drop(ctx->saved_data["p"].toDouble(), ctx->saved_data["seed"].toInt(), t, ctx->saved_data["offset"].toInt());
}

struct DropoutFn : public torch::autograd::Function<DropoutFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& d, const OptTensor& x, double p, int64_t seed,
                            const OptTensor& seed_at, int64_t offset) {
    ctx->save_for_backward({seed_at ? *seed_at : at::Tensor()});
    save_drop(ctx, p, seed, offset);
    ctx->saved_data["add"] = x.has_value();
    return dropout_apply(d.contiguous(), x ? x->contiguous() : at::Tensor(), make_drop(p, seed, seed_at, offset));
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_order("dropout");
    at::Tensor none, seed_at = ctx->get_saved_variables()[0], dd;
    if (ctx->needs_input_grad(0)) dd = dropout_apply(grads[0].contiguous(), none, saved_drop(ctx, seed_at));
    return {dd, ctx->saved_data["add"].toBool() ? grads[0] : none, none, none, none, none};
  }
};

struct DropNormFn : public torch::autograd::Function<DropNormFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& delta, const at::Tensor& w,
                               double eps, double p, int64_t seed, const OptTensor& seed_at, int64_t offset) {
    auto xc = x.contiguous(), dc = delta.contiguous(), wc = w.contiguous();
    auto o = drop_norm_fwd(xc, dc, wc, eps, make_drop(p, seed, seed_at, offset));
    ctx->save_for_backward({xc, dc, wc, o.rstd, seed_at ? *seed_at : at::Tensor()});
    save_drop(ctx, p, seed, offset);
    ctx->set_materialize_grads(false);
    return {o.sum, o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_order("dropout_add_rms_norm");
    auto s = ctx->get_saved_variables();
    auto dense = [](const at::Tensor& g) { return g.defined() ? g.contiguous() : g; };
    at::Tensor none;
    if (!grads[0].defined() && !grads[1].defined()) return {none, none, none, none, none, none, none, none};
    auto r = drop_norm_bwd(dense(grads[1]), dense(grads[0]), s[0], s[1], s[2], s[3], saved_drop(ctx, s[4]));
    return {r[0], r[1], r[2], none, none, none, none, none};
  }
};

at::Tensor dropout(const at::Tensor& d, const OptTensor& x, double p, int64_t seed, const OptTensor& seed_at,
                   int64_t offset) {
  const char* op = x ? "dropout_add" : "dropout";
  no_tangents(op, d, or_none(x));
  check_drop(op, d, p, seed_at, offset);
  if (x) same(op, "x and delta", *x, d);
  if (at::GradMode::is_enabled() && (d.requires_grad() || (x && x->requires_grad())))
    return DropoutFn::apply(d, x, p, seed, seed_at, offset);
  return dropout_apply(d.contiguous(), x ? x->contiguous() : at::Tensor(), make_drop(p, seed, seed_at, offset));
}

std::vector<at::Tensor> dropout_add_rms_norm(const at::Tensor& x, const at::Tensor& delta, const at::Tensor& w, double eps,
                                             double p, int64_t seed, const OptTensor& seed_at, int64_t offset) {
  const char* op = "dropout_add_rms_norm";
  no_tangents(op, x, delta, w);
  check_drop(op, x, p, seed_at, offset);
  same(op, "x and delta", x, delta);
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) <= kMaxNormDim, op, ": rows of at most ", kMaxNormDim, " elements wanted");
  TORCH_CHECK(w.dim() == 1 && w.numel() == x.size(-1) && w.scalar_type() == x.scalar_type() && w.device() == x.device(), op,
              ": weight must be [D], of the data's type and device");
  if (at::GradMode::is_enabled() && (x.requires_grad() || delta.requires_grad() || w.requires_grad()))
    return DropNormFn::apply(x, delta, w, eps, p, seed, seed_at, offset);
  auto o = drop_norm_fwd(x.contiguous(), delta.contiguous(), w.contiguous(), eps, make_drop(p, seed, seed_at, offset));
  return {o.sum, o.y};
}

}  // namespace

void register_dropout(pybind11::module_& m) {
  m.def("dropout", &dropout, "dropout(delta), or x + dropout(delta), from a seed, an optional seed tensor and an offset");
  m.def("dropout_add_rms_norm", &dropout_add_rms_norm, "(s, y): s = x + dropout(delta), y = rmsnorm(s) * w");
}
