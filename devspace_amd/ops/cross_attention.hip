// Cross attention for gfx950: queries of one sequence over the encoder's states of another length.
//
//   q [B, Tq, H, D], kv [B, Tk, 2, N, D] (packed keys and values, N divides H, G = H / N), len_b <= Tk states
//   S = scale q k^T over the first len_b states, P = softmax(S), O = P V; len_b = 0: O = 0, gradients 0
//   D_r = rowsum(dO * O), dV = P^T dO, dS = P * (dO V^T - D_r), dQ = scale dS K, dK = scale dS^T Q
//
// There is no causal mask, so the G query heads that share a key head are stacked: row m = t G + g, M = G Tq
// rows over one set of keys, each key and value read once for all of them. All products run on
// v_mfma_f32_32x32x16 (bf16 or fp16 in, fp32 out); softmax statistics and sums are in fp32. P and dS are
// rounded to the 16-bit type as operands of the next product (half a step each, averaged over the keys; in fp16
// by powers of two that keep them in its range), as are the outputs; nothing else is.
//
//   cross_fwd_kernel   128 rows (4 waves x 32), key tiles of 64 in LDS
//   cross_few_kernel   up to 32 rows (single tokens): every wave goes through key tiles of its own, keys
//                      straight into registers, values through a small LDS tile of the wave; joined in LDS
//   cross_dq_kernel    128 rows over all key tiles; also D_r
//   cross_dkv_kernel   128 keys over all row tiles; sums over a group's heads in registers, no atomics
// Each can split its long axis over several workgroups where there are too few of them to fill the chip;
// join kernels then add the parts in a fixed order.
//
// S is computed transposed (keys on the matrix rows, query rows on the lanes), so that a row's maximum and sum
// are lane-local plus one exchange of the wave's halves, and the accumulators are the next product's operand
// as they stand; V^T, K^T, Q^T and dO^T come from ds_read_b64_tr_b16 reads of row-major LDS tiles. Tiles come by
// buffer loads that write LDS without passing registers, one or two tiles ahead of their use, one barrier a tile.
//
// What bounds it (MI355X, bf16; a large matrix product reaches 1367 TFLOP/s and a large copy 5.0 TB/s here):
//   long rows      no unit alone: what a wave does between its products (softmax, conversions, LDS reads) is hidden in
//                  part only. 4 x 4096 x 4096, 16 heads of 128: forward 509 us (1080 TFLOP/s), dQ 692 (1192), dK and dV
//                  967 (1137), all three among others 2182; the matrix cores are busy in 54, 63 and 57 % of the cycles,
//                  at 1.8 to 1.9 GHz, LDS conflicts in 0.1 % at the most. Two kernels without atomics compute S and dP
//                  twice: 18 products' work for 14. 16 heads of 64, with as many exponentials for half of the products:
//                  299 us (919), 386 (1068), 521 (1055), matrix cores busy in 45, 57 and 52 %.
//   short rows     latency of a tile and of a launch: 8 x 512 x 512 ragged, 16 heads of 64: 18, 23 and 28 us
//   single tokens  memory: 32 tokens over 1500 ragged states, 16 heads of 64: 37 us (4.0 TB/s); one token over
//                  131071 states, 8 key heads of 128: 104 us with its join (5.2 TB/s)
#include "fused_common.h"

#include <algorithm>
#include <type_traits>
#include <vector>

namespace {

constexpr int kThreads = 256;
constexpr int kRows = 128;  // query rows (forward, dQ) or keys (dK, dV) of a workgroup: 32 per wave
constexpr int kKeys = 64;   // keys of an LDS tile
constexpr int kWanted = 512;  // workgroups that fill the chip: two on each of 256 CUs

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) unsigned char lds_u8;
typedef __attribute__((address_space(3))) void lds_void;

template <typename E>
__device__ __forceinline__ f32x16 mfma(const u16x8& a, const u16x8& b, const f32x16& c) {
  if constexpr (E::kType == at::kBFloat16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// A tile's rows of D <= DP columns take RB bytes. 16-byte chunks are swizzled by the row: the row reads
// (ds_read_b128, 16 rows of one chunk) and the transposed reads (4 neighbouring rows of 4 neighbouring chunks)
// both fall on different banks.
template <int DP>
struct Tile {
  static constexpr int RB = DP <= 64 ? 128 : 256;
  static constexpr int CH = DP / 8;   // chunks of a row
  static constexpr int KS = DP / 16;  // steps of a product over the columns
  static constexpr int NB = DP / 32;  // blocks of 32 columns
  static constexpr int BUFS = DP <= 64 ? 3 : 2;  // tiles in LDS, with two workgroups on a CU
  __device__ static __forceinline__ int off(int row, int chunk) {
    if constexpr (RB == 128) return row * 128 + ((chunk ^ ((row >> 1) & 7) ^ ((row & 2) << 1)) << 4);
    else return row * 256 + ((chunk ^ (((row & 3) << 2) | ((row >> 2) & 3))) << 4);
  }
};

// A lane's places in a tile, the same in every tile and (32 and 16 rows being whole periods of the swizzle) in
// every block of rows: kept in registers, all else is a constant of the instruction.
template <int DP>
struct Places {
  typedef Tile<DP> L;
  int row[L::KS];    // chunk 2 s + hh of row r (r = lane & 31, hh = lane >> 5)
  int tr[L::NB][2];  // the transposed operand's four rows from 4 hh on and from 8 + 4 hh on, 32 columns at nb 32
  __device__ __forceinline__ explicit Places(int lane) {
    const int r = lane & 31, hh = lane >> 5, g = lane >> 4, i = lane & 15;
#pragma unroll
    for (int s = 0; s < L::KS; ++s) row[s] = L::off(r, 2 * s + hh);
#pragma unroll
    for (int nb = 0; nb < L::NB; ++nb) {
      const int col = nb * 32 + 16 * (g & 1) + 4 * (i & 3);
#pragma unroll
      for (int k = 0; k < 2; ++k) tr[nb][k] = L::off(8 * k + 4 * hh + (i >> 2), col >> 3) + ((col & 7) << 1);
    }
  }
  // columns 16 s + 8 hh .. of row r0 + r; r0 a multiple of 32
  __device__ __forceinline__ u16x8 row8(const unsigned char* tile, int r0, int s) const {
    return *reinterpret_cast<const u16x8*>(tile + row[s] + r0 * L::RB);
  }
  // Operand of the transposed tile: column nb 32 + r of rows r0 + 4 hh + {0..3} and r0 + 8 + 4 hh + {0..3}, the
  // order of an accumulator's rows; r0 a multiple of 16.
  __device__ __forceinline__ u16x8 tr8(const unsigned char* tile, int r0, int nb) const {
    lds_u8* base = (lds_u8*)tile + r0 * L::RB;
    s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(base + tr[nb][0]));
    s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(base + tr[nb][1]));
    return __builtin_bit_cast(u16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

// Probabilities become operands of the 16-bit type. fp16 loses bits below 2^-14, and a probability of a long source is
// smaller than that: they are lifted by a power of two, which what they are divided by, or the result, takes off
// again (the sum l in the forward pass, whose P lies within 2^8 of its reference; 2^-kLiftBack in the backward pass,
// whose P is at most 1). 65451 states in fp16: dK and dV were 2.2 times as far off as their own rounding.
template <typename E>
constexpr float kLift = E::kType == at::kHalf ? 7.f : 0.f;
template <typename E>
constexpr float kLiftBack = E::kType == at::kHalf ? 15.f : 0.f;
template <typename E>  // the exponent's constant (a negation costs an instruction nothing, a difference with 0 does)
__device__ __forceinline__ float lift_back(float lse) {
  if constexpr (E::kType == at::kHalf) return kLiftBack<E> - lse;
  else return -lse;
}
template <typename E>
constexpr float kUnliftBack = E::kType == at::kHalf ? 1.f / 32768.f : 1.f;

// 2^x on the transcendental unit; 2^-inf = 0, which masked scores rely on
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

template <typename E>
__device__ __forceinline__ u16x8 to_operand(const f32x16& acc, int s) {
  u16x8 o;
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = E::put(acc[8 * s + j]);
  return o;
}

// row of a 32x32 accumulator in register i of lane half hh
__device__ __forceinline__ int acc_row(int i, int hh) { return (i & 3) + 8 * (i >> 2) + 4 * hh; }

__device__ __forceinline__ u16x8 zero8() {
  u16x8 z;
#pragma unroll
  for (int i = 0; i < 8; ++i) z[i] = 0;
  return z;
}
__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

struct CrossParams {
  const u16 *q, *kv, *o, *dout;
  u16 *out, *dkv;       // O or dQ [B, Tq, H, D]; [B, Tk, 2, N, D]
  float *part;          // split forward: O's parts [split][B N][M][D]; split dQ, dK, dV: parts in the output's layout
  float *part_ml;       // split forward: (m, l) of each part [split][B N][M]
  float *lse, *delta;   // [B N][M]; lse in the log2 domain of the scaled scores
  const void* lengths;  // null: Tk
  int64_t qb, qt, qh;   // strides in elements
  int64_t kb, kt, ks, kh;
  int64_t out_numel, dkv_numel;  // a part's size in the gradients' layout
  int B, N, G, M, Tq, Tk, D;
  int splits, per_split;  // keys (forward, dQ) or rows (dK, dV) of a split: whole tiles
  int blocks;             // workgroups along the rows or keys
  FastDiv by_G;
  float scale, scale_log2;
  bool len64;

  __device__ __forceinline__ int length_of(int b) const {
    if (!lengths) return Tk;
    const int64_t n = len64 ? static_cast<const int64_t*>(lengths)[b] : (int64_t)static_cast<const int*>(lengths)[b];
    return (int)(n < 0 ? 0 : n > Tk ? Tk : n);
  }
  // the same for a sequence that all lanes share
  __device__ __forceinline__ int length(int b) const { return __builtin_amdgcn_readfirstlane(length_of(b)); }
  // Axes come near to 2^31, where begin + per_split does not fit 32 bits: where a split ends, and how many have any of
  // an axis' first len.
  __device__ __forceinline__ int split_end(int begin, int len) const { return begin + min(per_split, len - begin); }
  __device__ __forceinline__ int parts_of(int len) const {
    return (int)(((unsigned)len + (unsigned)per_split - 1u) / (unsigned)per_split);
  }
  // offset of row m of key head n in [B, Tq, H, D] with these strides
  __device__ __forceinline__ int64_t row_at(int m, int b, int n, int64_t sb, int64_t st, int64_t sh) const {
    unsigned g;
    const unsigned t = by_G.divmod((unsigned)m, g);
    return b * sb + (int64_t)t * st + ((int64_t)n * G + g) * sh;
  }
  __device__ __forceinline__ int64_t dense_at(int m, int b, int n) const {
    const int64_t H = (int64_t)N * G;
    return row_at(m, b, n, Tq * H * D, H * D, D);
  }
};

// Which work a workgroup has. Workgroups go to the 8 XCDs in turn; all of one key head are given to one XCD, whose L2
// then serves its keys and values, and neighbouring heads to different XCDs, so that sequences of unlike lengths are
// spread evenly (8 ragged sequences of 16 heads, trained: 62.2 us, with one sequence to an XCD 65.2; 32 single tokens
// 37.2 us for 39.1).
struct Place {
  int block, split, n, b, bn;
  __device__ __forceinline__ explicit Place(const CrossParams& p) {
    const unsigned id = blockIdx.x, each = p.blocks * p.splits, even = (unsigned)(p.B * p.N) & ~7u;
    unsigned rest;
    if (id < even * each) {
      const unsigned slot = id >> 3;
      bn = (int)(slot / each * 8 + (id & 7));
      rest = slot % each;
    } else {  // up to 7 heads more, in turn
      const unsigned over = id - even * each;
      bn = (int)(even + over / each);
      rest = over % each;
    }
    block = rest % p.blocks;
    split = rest / p.blocks;
    n = bn % p.N;
    b = bn / p.N;
  }
};

// Buffer loads know how many bytes there are from their base on, and read 0 behind them: tiles that reach past
// the last row, and columns past D (whose lanes get the offset kOutside), need no branches.
constexpr unsigned kOutside = 0x80000000u;

// bytes from a tile's first row to the end of its last valid one; none for valid <= 0
__device__ __forceinline__ unsigned bytes_of(int valid, int64_t stride, int D) {
  return valid <= 0 ? 0u : (unsigned)min(((int64_t)(valid - 1) * stride + D) * 2, (int64_t)kOutside - 1);
}

// The builtin is younger than the instruction: a compiler without it (a pod's image may have one) gets the intrinsic
// by its name, the same code.
#if defined(__HIP_DEVICE_COMPILE__) && !__has_builtin(__builtin_amdgcn_raw_ptr_buffer_load_lds)
extern "C" __device__ void buffer_load_to_lds(__amdgpu_buffer_rsrc_t src, lds_void* lds, int size, int offset, int soffset,
                                              int at, int aux) __asm("llvm.amdgcn.raw.ptr.buffer.load.lds");
#else
#define buffer_load_to_lds __builtin_amdgcn_raw_ptr_buffer_load_lds
#endif

// BYTES (4 or 16) per lane from `base` plus this lane's offset to `lds` plus BYTES times the lane, without passing
// registers
template <int BYTES>
__device__ __forceinline__ void to_lds(const void* base, unsigned bytes, void* lds, unsigned offset) {
  static_assert(BYTES == 16 || BYTES == 4, "sizes used here");
#ifdef __HIP_DEVICE_COMPILE__  // the buffer's type is the device's
  __amdgpu_buffer_rsrc_t src = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00020000);
  if constexpr (BYTES == 16) buffer_load_to_lds(src, (lds_void*)(lds_u8*)lds, 16, offset, 0, 0, 0);
  else buffer_load_to_lds(src, (lds_void*)(lds_u8*)lds, 4, offset, 0, 0, 0);
#endif
}

// N chunks of 16 bytes at this lane's offsets
template <int N>
__device__ __forceinline__ void to_registers(u16x8 (&to)[N], const void* base, unsigned bytes, const unsigned (&offset)[N]) {
#ifdef __HIP_DEVICE_COMPILE__
  __amdgpu_buffer_rsrc_t src = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00020000);
#pragma unroll
  for (int u = 0; u < N; ++u) to[u] = __builtin_bit_cast(u16x8, __builtin_amdgcn_raw_buffer_load_b128(src, offset[u], 0, 0));
#endif
}

// One wave's share of copying tiles of ROWS rows of two tensors (waves 0 and 1 the first, 2 and 3 the second)
// into LDS: 64 lanes x 16 bytes, a few whole rows each. The swizzle is applied to the source: lane l fills the
// l-th 16 bytes and fetches the chunk that belongs there.
template <int DP, int ROWS>
struct Dma {
  typedef Tile<DP> L;
  static constexpr int kPer = 2 * ROWS * L::RB / (4 * 1024);  // loads of a wave
  static constexpr int kRowsEach = 1024 / L::RB;
  static constexpr int kSlots = L::RB / 16;
  unsigned at[kPer];  // byte offset of this lane's chunk from the tile's first row
  int piece;          // where the wave's part of a tensor's tile begins, bytes

  __device__ static __forceinline__ bool second(int wave) { return wave >= 2; }
  __device__ static __forceinline__ int row(int wave, int lane, int u) {
    return (wave & 1) * (ROWS / 2) + u * kRowsEach + lane / kSlots;
  }
  // offset(row): byte offset of a row of the tile, or kOutside
  template <typename F>
  __device__ __forceinline__ void place(int wave, int lane, int D, F&& offset) {
    piece = (wave & 1) * (ROWS / 2) * L::RB;
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int i = row(wave, lane, u);
      const int chunk = (L::off(i, lane % kSlots) - i * L::RB) >> 4;
      const unsigned o = offset(i);
      at[u] = chunk * 8 < D && o < kOutside ? o + chunk * 16 : kOutside;
    }
  }
  __device__ __forceinline__ void go(const u16* base, unsigned bytes, unsigned char* tile) const {
#pragma unroll
    for (int u = 0; u < kPer; ++u) to_lds<16>(base, bytes, tile + piece + u * 1024, at[u]);
  }
};

// All but the wave's last N loads have arrived, its LDS reads are done, and the other waves are as far.
template <int N>
__device__ __forceinline__ void wait_all_but() {
  static_assert(N < 64, "the counter has six bits");
  if constexpr (N == 0)
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  else
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// this lane's half of a row as KS operands (columns 16 s + 8 hh ..); null: zeros
template <int DP>
__device__ __forceinline__ void load_row(u16x8* f, const u16* row, int hh, int D) {
#pragma unroll
  for (int s = 0; s < Tile<DP>::KS; ++s) {
    const int col = 16 * s + 8 * hh;
    f[s] = row && col < D ? *reinterpret_cast<const u16x8*>(row + col) : zero8();
  }
}

// the larger, or the sum, of this lane's value and that of the other half's lane of the same row
__device__ __forceinline__ void other_half(float x, float& a, float& b) {
  const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  a = __uint_as_float(both[0]);
  b = __uint_as_float(both[1]);
}
__device__ __forceinline__ float half_max(float x) {
  float a, b;
  other_half(x, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float half_sum(float x) {
  float a, b;
  other_half(x, a, b);
  return a + b;
}

// dS as an operand: fp16 neither holds the small values of long sources nor every large one, so each lane's column is
// multiplied by a power of two that fits the largest value met so far (2^9 times the lift at the most). The
// accumulators it goes into are rescaled when that falls; bf16 has the range and passes by.
template <typename E>
struct Gain {
  float up = E::kType == at::kHalf ? 512.f : 1.f;
  template <int NB>
  __device__ __forceinline__ void fit(f32x16& ds, f32x16 (&acc)[NB]) {
    if constexpr (E::kType == at::kHalf) {
      float most = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(ds[i]));
      most = half_max(most);
      if (__any(most * up > 32768.f)) {
        const float fits = most > 0.f ? ldexpf(1.f, 15 - __builtin_amdgcn_frexp_expf(most)) : up;
        const float next = fminf(up, fits), by = next / up;  // powers of two
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[nb][i] *= by;
        up = next;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) ds[i] *= up;
    }
  }
  // what the accumulators are multiplied by to be sums of dS
  __device__ __forceinline__ float down() const { return kUnliftBack<E> / up; }
};

// One tile of scores in the log2 domain: the online softmax of this lane's row. On return s holds P against the
// reference m, which follows the running maximum (less the lift) only when that has left it by more than 2^8: P and
// the sums stay within 2^8 (and the lift) times the number of keys, nothing is lost in their floating types, and O (64
// registers with wide heads) is rarely rescaled. In front of the exponentials, `rescale` gets the factor where any
// row moves.
template <typename E, int KB, typename F>
__device__ __forceinline__ void soften(f32x16* s, float& m, float& l, float scale_log2, F&& rescale) {
  float mt = -INFINITY;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int i = 0; i < 16; ++i) mt = fmaxf(mt, s[kb][i]);
  mt = half_max(mt) * scale_log2;
  if (__any(mt > m + (8.f + kLift<E>))) {
    const float mn = fmaxf(m, mt - kLift<E>);
    const float alpha = exp2_fast(m - (mn == -INFINITY ? 0.f : mn));
    l *= alpha;
    m = mn;
    rescale(alpha);
  }
  const float base = m == -INFINITY ? 0.f : m;  // nothing but -inf so far: all of P is 0
  float ls[2] = {0.f, 0.f};
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float e = exp2_fast(__builtin_fmaf(s[kb][i], scale_log2, -base));
      s[kb][i] = e;
      ls[i & 1] += e;
    }
  l += ls[0] + ls[1];
}

// Four columns of a row of O^T or dQ^T accumulators at a time: column nb 32 + 8 g4 + 4 hh
template <int DP, typename F>
__device__ __forceinline__ void each_quad(int hh, int D, F&& f) {
#pragma unroll
  for (int nb = 0; nb < Tile<DP>::NB; ++nb)
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
      const int col = nb * 32 + 8 * g4 + 4 * hh;
      if (col < D) f(col, nb, 4 * g4);
    }
}
template <typename E>
__device__ __forceinline__ void put4(u16* at, const f32x16& a, int i, float by) {
  u16v<4> o;
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = E::put(a[i + j] * by);
  *reinterpret_cast<u16v<4>*>(at) = o;
}
__device__ __forceinline__ void put4f(float* at, const f32x16& a, int i, float by) {
  *reinterpret_cast<float4*>(at) = make_float4(a[i] * by, a[i + 1] * by, a[i + 2] * by, a[i + 3] * by);
}

// Runs step(tile, position) over positions begin, begin + STEP, ... < end, with the tiles of the next BUFS - 1
// positions on their way: issue(tile, position) starts a tile's PER loads of this wave (positions past the end
// too, so that the number of loads in flight does not depend on the position). A position's loads are waited
// for, then the barrier says that all waves have waited, and have left the tile that is filled next. The tiles
// are separate arrays, so that the compiler knows that reads of one need not wait for loads into another.
template <int PER, int STEP, typename T, typename I, typename S>
__device__ __forceinline__ void pipeline(T& a, T& b, int begin, int end, I&& issue, S&& step) {
  issue(a, begin);
  for (int at = begin;;) {
    wait_all_but<0>();
    issue(b, at + STEP);
    step(a, at);
    if ((at += STEP) >= end) break;
    wait_all_but<0>();
    issue(a, at + STEP);
    step(b, at);
    if ((at += STEP) >= end) break;
  }
  wait_all_but<0>();
}
template <int PER, int STEP, typename T, typename I, typename S>
__device__ __forceinline__ void pipeline(T& a, T& b, T& c, int begin, int end, I&& issue, S&& step) {
  issue(a, begin);
  issue(b, begin + STEP);
  for (int at = begin;;) {
    wait_all_but<PER>();
    issue(c, at + 2 * STEP);
    step(a, at);
    if ((at += STEP) >= end) break;
    wait_all_but<PER>();
    issue(a, at + 2 * STEP);
    step(b, at);
    if ((at += STEP) >= end) break;
    wait_all_but<PER>();
    issue(b, at + 2 * STEP);
    step(c, at);
    if ((at += STEP) >= end) break;
  }
  wait_all_but<0>();
}

template <int DP>
using KeyTile = unsigned char[2][kKeys * Tile<DP>::RB];  // K | V
#define KEY_TILES(DP) __shared__ __attribute__((aligned(16))) KeyTile<DP> tile0, tile1, tile2

// step(K tile, V tile, first key) over the keys [begin, end) of one key head
template <int DP, typename S>
__device__ __forceinline__ void key_loop(KeyTile<DP>& tile0, KeyTile<DP>& tile1, KeyTile<DP>& tile2, const CrossParams& p,
                                         const Place& w, int wave, int lane, int begin, int end, S&& step) {
  typedef Tile<DP> L;
  typedef Dma<DP, kKeys> Copy;
  typedef KeyTile<DP> Pair;
  if (begin >= end) return;
  Copy copy;
  copy.place(wave, lane, p.D, [&](int row) { return (unsigned)(row * (int)p.kt * 2); });
  const bool second = Copy::second(wave);
  const u16* base = p.kv + w.b * p.kb + w.n * p.kh + (second ? p.ks : 0);
  auto issue = [&](Pair& t, int k0) { copy.go(base + (k0 < end ? k0 : 0) * p.kt, bytes_of(end - k0, p.kt, p.D), t[second]); };
  auto use = [&](const Pair& t, int k0) { step(t[0], t[1], k0); };
  if constexpr (L::BUFS == 3) pipeline<Copy::kPer, kKeys>(tile0, tile1, tile2, begin, end, issue, use);
  else pipeline<Copy::kPer, kKeys>(tile0, tile1, begin, end, issue, use);
}

// ------------------------------------------------------------------------------ forward

template <typename E, int DP>
__global__ void __launch_bounds__(kThreads, 2) cross_fwd_kernel(CrossParams p) {
  typedef Tile<DP> L;
  KEY_TILES(DP);
  const Place w(p);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 31, hh = lane >> 5;
  const Places<DP> lds(lane);
  const int m0 = w.block * kRows + wave * 32, row = m0 + r;
  const bool some = m0 < p.M;  // the wave has rows at all
  const int k_begin = w.split * p.per_split, k_end = p.split_end(k_begin, p.length(w.b));
  u16x8 qf[L::KS];
  load_row<DP>(qf, row < p.M ? p.q + p.row_at(row, w.b, w.n, p.qb, p.qt, p.qh) : nullptr, hh, p.D);
  f32x16 o[L::NB];
#pragma unroll
  for (int nb = 0; nb < L::NB; ++nb) o[nb] = zero16();
  float m = -INFINITY, l = 0.f;
  auto step = [&](const unsigned char* Ks, const unsigned char* Vs, int k0) {
    if (!some) return;
    f32x16 s[2] = {zero16(), zero16()};
#pragma unroll
    for (int st = 0; st < L::KS; ++st)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) s[kb] = mfma<E>(lds.row8(Ks, kb * 32, st), qf[st], s[kb]);
    if (k0 + kKeys > k_end) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (k0 + kb * 32 + acc_row(i, hh) >= k_end) s[kb][i] = -INFINITY;
    }
    soften<E, 2>(s, m, l, p.scale_log2, [&](float alpha) {
#pragma unroll
      for (int nb = 0; nb < L::NB; ++nb)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[nb][i] *= alpha;
    });
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const u16x8 pb = to_operand<E>(s[ks >> 1], ks & 1);
#pragma unroll
      for (int nb = 0; nb < L::NB; ++nb) o[nb] = mfma<E>(lds.tr8(Vs, 16 * ks, nb), pb, o[nb]);
    }
  };
  key_loop<DP>(tile0, tile1, tile2, p, w, wave, lane, k_begin, k_end, step);
  if (row >= p.M) return;
  l = half_sum(l);
  const int64_t stat = (int64_t)w.bn * p.M + row;
  if (p.splits == 1) {
    const float inv = k_begin < k_end ? 1.f / l : 0.f;  // no state at all: 0
    u16* to = p.out + p.dense_at(row, w.b, w.n);
    each_quad<DP>(hh, p.D, [&](int col, int nb, int i) { put4<E>(to + col, o[nb], i, inv); });
    if (p.lse && hh == 0) p.lse[stat] = m + __log2f(l);
  } else if (k_begin < k_end) {
    const int64_t at = ((int64_t)w.split * p.B * p.N + w.bn) * p.M + row;
    each_quad<DP>(hh, p.D, [&](int col, int nb, int i) { put4f(p.part + at * p.D + col, o[nb], i, 1.f); });
    if (hh == 0) {
      p.part_ml[2 * at] = m;
      p.part_ml[2 * at + 1] = l;
    }
  }
}

// Up to 32 rows: wave w takes the 32-key tiles w, w + 4, ... of the split. Bound by memory: the loads of two
// tiles are under way per wave (heads of 64; with one, 32 tokens over 1500 states took 45 us for 39).
template <typename E, int DP>
__global__ void __launch_bounds__(kThreads, 2) cross_few_kernel(CrossParams p) {
  typedef Tile<DP> L;
  constexpr int kTile = 32;
  constexpr int kPer = kTile * L::CH / 64;  // chunks of V per lane
  __shared__ __attribute__((aligned(16))) union {
    unsigned char v[4][kTile * L::RB];
    float o[4][32][DP];
  } sm;
  __shared__ float sml[4][2][32];
  const Place w(p);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 31, hh = lane >> 5;
  const Places<DP> lds(lane);
  const int m0 = w.block * 32, row = m0 + r;
  const int rows = min(32, p.M - m0);
  const int k_begin = w.split * p.per_split, k_end = p.split_end(k_begin, p.length(w.b));
  const u16* kbase = p.kv + w.b * p.kb + w.n * p.kh;
  u16x8 qf[L::KS];
  load_row<DP>(qf, row < p.M ? p.q + p.row_at(row, w.b, w.n, p.qb, p.qt, p.qh) : nullptr, hh, p.D);
  f32x16 o[L::NB];
#pragma unroll
  for (int nb = 0; nb < L::NB; ++nb) o[nb] = zero16();
  float m = -INFINITY, l = 0.f;
  unsigned char* Vs = sm.v[wave];
  unsigned at_k[L::KS], at_v[kPer];
#pragma unroll
  for (int st = 0; st < L::KS; ++st) at_k[st] = 16 * st + 8 * hh < p.D ? (unsigned)(r * (int)p.kt + 16 * st + 8 * hh) * 2 : kOutside;
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    const int c = lane + 64 * u, ch = c % L::CH;
    at_v[u] = ch * 8 < p.D ? (unsigned)(c / L::CH * (int)p.kt + ch * 8) * 2 : kOutside;
  }
  struct Keys {  // one tile on its way: keys as operands, values by rows
    u16x8 k[L::KS], v[kPer];
  };
  auto load = [&](Keys& t, unsigned k0) {  // positions past the end pass 2^31, too
    const bool any = k0 < (unsigned)k_end;
    const u16* base = kbase + (any ? k0 : 0u) * p.kt;
    const unsigned bytes = any ? bytes_of((int)((unsigned)k_end - k0), p.kt, p.D) : 0u;
    to_registers(t.k, base, bytes, at_k);
    to_registers(t.v, base + p.ks, bytes, at_v);
  };
  auto step = [&](Keys& t, int k0, int ahead) {
    f32x16 s = zero16();
#pragma unroll
    for (int st = 0; st < L::KS; ++st) s = mfma<E>(t.k[st], qf[st], s);
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int c = lane + 64 * u;
      *reinterpret_cast<u16x8*>(Vs + L::off(c / L::CH, c % L::CH)) = t.v[u];
    }
    load(t, (unsigned)k0 + ahead);
    if (k0 + kTile > k_end) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (k0 + acc_row(i, hh) >= k_end) s[i] = -INFINITY;
    }
    soften<E, 1>(&s, m, l, p.scale_log2, [&](float alpha) {
#pragma unroll
      for (int nb = 0; nb < L::NB; ++nb)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[nb][i] *= alpha;
    });
    // the tile belongs to this wave alone, and a wave's LDS operations stay in order
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const u16x8 pb = to_operand<E>(s, ks);
#pragma unroll
      for (int nb = 0; nb < L::NB; ++nb) o[nb] = mfma<E>(lds.tr8(Vs, 16 * ks, nb), pb, o[nb]);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  };
  // the loads of one more tile, or of two where the registers hold them, are under way
  constexpr int kStride = 4 * kTile;
  int k0 = __builtin_amdgcn_readfirstlane(k_begin + wave * kTile);
  Keys t0, t1;
  load(t0, k0);
  if constexpr (L::BUFS == 3) {
    load(t1, (unsigned)k0 + kStride);
    while (k0 < k_end) {
      step(t0, k0, 2 * kStride);
      if ((k0 += kStride) >= k_end) break;
      step(t1, k0, 2 * kStride);
      k0 += kStride;
    }
  } else {
    for (; k0 < k_end; k0 += kStride) step(t0, k0, kStride);
  }
  // join the four waves: their maxima and sums, then their rows on the common maximum
  l = half_sum(l);
  if (hh == 0) {
    sml[wave][0][r] = m;
    sml[wave][1][r] = l;
  }
  __syncthreads();  // the tiles are done with: their memory takes the rows
  float mj = fmaxf(fmaxf(sml[0][0][r], sml[1][0][r]), fmaxf(sml[2][0][r], sml[3][0][r]));
  const float base = mj == -INFINITY ? 0.f : mj;
  float lj = 0.f;
#pragma unroll
  for (int v = 0; v < 4; ++v) lj += sml[v][1][r] * exp2_fast(sml[v][0][r] - base);
  const float mine = exp2_fast(m - base);
  if (r < rows) each_quad<DP>(hh, DP, [&](int col, int nb, int i) { put4f(&sm.o[wave][r][col], o[nb], i, mine); });
  __syncthreads();
  if (k_begin >= k_end && p.splits > 1) return;  // the join does not look at this part
  if (wave == 0 && hh == 0 && r < rows) {
    if (p.splits == 1) {
      if (p.lse) p.lse[(int64_t)w.bn * p.M + row] = mj + __log2f(lj);
      sml[0][0][r] = k_begin < k_end ? 1.f / lj : 0.f;
    } else {
      const int64_t at = ((int64_t)w.split * p.B * p.N + w.bn) * p.M + row;
      p.part_ml[2 * at] = mj;
      p.part_ml[2 * at + 1] = lj;
    }
  }
  __syncthreads();
  const int quads = p.D >> 2;
  for (int c = threadIdx.x; c < rows * quads; c += kThreads) {
    const int i = c / quads, col = (c - i * quads) * 4;
    float4 a = *reinterpret_cast<const float4*>(&sm.o[0][i][col]);
#pragma unroll
    for (int v = 1; v < 4; ++v) {
      const float4 b = *reinterpret_cast<const float4*>(&sm.o[v][i][col]);
      a.x += b.x, a.y += b.y, a.z += b.z, a.w += b.w;
    }
    if (p.splits == 1) {
      const float inv = sml[0][0][i];
      u16v<4> out;
      out[0] = E::put(a.x * inv), out[1] = E::put(a.y * inv), out[2] = E::put(a.z * inv), out[3] = E::put(a.w * inv);
      *reinterpret_cast<u16v<4>*>(p.out + p.dense_at(m0 + i, w.b, w.n) + col) = out;
    } else {
      const int64_t at = ((int64_t)w.split * p.B * p.N + w.bn) * p.M + m0 + i;
      *reinterpret_cast<float4*>(p.part + at * p.D + col) = a;
    }
  }
}

// Joins the parts of split rows, four columns of a row per thread: for rows enough to fill the chip so.
template <typename E>
__global__ void __launch_bounds__(kThreads) cross_join_many_kernel(CrossParams p, unsigned items, FastDiv by_quads) {
  const unsigned u = blockIdx.x * kThreads + threadIdx.x;
  if (u >= items) return;
  unsigned quad;
  const unsigned stat = by_quads.divmod(u, quad);  // bn M + row
  const int col = (int)quad * 4;
  const int bn = (int)(stat / (unsigned)p.M), row = (int)(stat - (unsigned)bn * p.M);
  const int b = bn / p.N, n = bn - b * p.N;
  const int parts = p.parts_of(p.length_of(b));
  const int64_t step = (int64_t)p.B * p.N * p.M;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + stat;
  float m = -INFINITY;
  for (int s = 0; s < parts; ++s) m = fmaxf(m, ml[s * step].x);
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < parts; ++s) {
    const float2 part = ml[s * step];
    const float4 v = *reinterpret_cast<const float4*>(p.part + (s * step + stat) * p.D + col);
    const float e = exp2_fast(part.x - base);
    l += part.y * e;
    a.x += v.x * e, a.y += v.y * e, a.z += v.z * e, a.w += v.w * e;
  }
  const float inv = parts > 0 ? 1.f / l : 0.f;
  u16v<4> out;
  out[0] = E::put(a.x * inv), out[1] = E::put(a.y * inv), out[2] = E::put(a.z * inv), out[3] = E::put(a.w * inv);
  *reinterpret_cast<u16v<4>*>(p.out + p.dense_at(row, b, n) + col) = out;
  if (p.lse && col == 0) p.lse[stat] = m + __log2f(l);
}

// Joins the parts of a split row: THREADS threads per row, 32 lanes over its columns (four each), THREADS / 32
// groups of them over the parts, whose sums are added in LDS.
template <typename E, int THREADS>
__global__ void __launch_bounds__(THREADS) cross_join_kernel(CrossParams p) {
  constexpr int kGroups = THREADS / 32;
  __shared__ float weight[kWanted], red[2][THREADS / 64];
  __shared__ __attribute__((aligned(16))) float acc[kGroups][128];
  const int64_t stat = blockIdx.x;  // bn M + row
  const int bn = (int)(stat / p.M), row = (int)(stat - (int64_t)bn * p.M);
  const int b = bn / p.N, n = bn - b * p.N;
  const int parts = p.parts_of(p.length(b));
  const int64_t step = (int64_t)p.B * p.N * p.M;
  const int wave = threadIdx.x >> 6;
  float m = -INFINITY;
  for (int s = threadIdx.x; s < parts; s += THREADS) m = fmaxf(m, p.part_ml[2 * (s * step + stat)]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  if ((threadIdx.x & 63) == 0) red[0][wave] = m;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < THREADS / 64; ++v) m = fmaxf(m, red[0][v]);
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  for (int s = threadIdx.x; s < parts; s += THREADS) {
    const int64_t at = s * step + stat;
    const float e = exp2_fast(p.part_ml[2 * at] - base);
    weight[s] = e;
    l += p.part_ml[2 * at + 1] * e;
  }
  l = wave_sum(l);
  if ((threadIdx.x & 63) == 0) red[1][wave] = l;
  __syncthreads();
  l = red[1][0];
#pragma unroll
  for (int v = 1; v < THREADS / 64; ++v) l += red[1][v];
  const int col = (threadIdx.x & 31) * 4, group = threadIdx.x >> 5;
  if (col < p.D) {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = group; s < parts; s += kGroups) {
      const float4 v = *reinterpret_cast<const float4*>(p.part + (s * step + stat) * p.D + col);
      const float e = weight[s];
      a.x += v.x * e, a.y += v.y * e, a.z += v.z * e, a.w += v.w * e;
    }
    *reinterpret_cast<float4*>(&acc[group][col]) = a;
  }
  __syncthreads();
  if (group > 0 || col >= p.D) return;
  const float inv = parts > 0 ? 1.f / l : 0.f;
  u16v<4> out;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float t = acc[0][col + j];
#pragma unroll
    for (int g = 1; g < kGroups; ++g) t += acc[g][col + j];
    out[j] = E::put(t * inv);
  }
  *reinterpret_cast<u16v<4>*>(p.out + p.dense_at(row, b, n) + col) = out;
  if (p.lse && threadIdx.x == 0) p.lse[stat] = m + __log2f(l);
}

// ------------------------------------------------------------------------------ backward

template <typename E, int DP>
__global__ void __launch_bounds__(kThreads, 2) cross_dq_kernel(CrossParams p) {
  typedef Tile<DP> L;
  KEY_TILES(DP);
  const Place w(p);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 31, hh = lane >> 5;
  const Places<DP> lds(lane);
  const int m0 = w.block * kRows + wave * 32, row = m0 + r;
  const bool some = m0 < p.M, mine = row < p.M;
  const int len = p.length(w.b);
  const int k_begin = w.split * p.per_split, k_end = p.split_end(k_begin, len);
  const int64_t dense = mine ? p.dense_at(row, w.b, w.n) : 0, stat = (int64_t)w.bn * p.M + row;
  u16x8 qf[L::KS], df[L::KS];
  load_row<DP>(df, mine ? p.dout + dense : nullptr, hh, p.D);
  load_row<DP>(qf, mine ? p.o + dense : nullptr, hh, p.D);
  float delta = 0.f;
#pragma unroll
  for (int s = 0; s < L::KS; ++s)
#pragma unroll
    for (int j = 0; j < 8; ++j) delta += E::get(df[s][j]) * E::get(qf[s][j]);
  delta = half_sum(delta);
  const float lse = mine ? p.lse[stat] : INFINITY;  // rows outside: P = 2^(0 - inf) = 0
  load_row<DP>(qf, mine ? p.q + p.row_at(row, w.b, w.n, p.qb, p.qt, p.qh) : nullptr, hh, p.D);
  f32x16 dq[L::NB];
#pragma unroll
  for (int nb = 0; nb < L::NB; ++nb) dq[nb] = zero16();
  Gain<E> gain;
  // S and dP of 32 keys, S turned into P; keys behind the end have P = 0
  auto scores = [&](const unsigned char* Ks, const unsigned char* Vs, int k0, int kb, f32x16& s, f32x16& dp) {
    s = zero16();
    dp = zero16();
#pragma unroll
    for (int st = 0; st < L::KS; ++st) {
      s = mfma<E>(lds.row8(Ks, kb * 32, st), qf[st], s);
      dp = mfma<E>(lds.row8(Vs, kb * 32, st), df[st], dp);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = exp2_fast(__builtin_fmaf(s[i], p.scale_log2, lift_back<E>(lse)));
    if (k0 + kb * 32 + 32 > k_end) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (k0 + kb * 32 + acc_row(i, hh) >= k_end) s[i] = 0.f;
    }
  };
  auto add = [&](const unsigned char* Ks, int kb, const f32x16& s, f32x16& dp) {
#pragma unroll
    for (int i = 0; i < 16; ++i) dp[i] = s[i] * (dp[i] - delta);
    gain.fit(dp, dq);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const u16x8 db = to_operand<E>(dp, ks);
#pragma unroll
      for (int nb = 0; nb < L::NB; ++nb) dq[nb] = mfma<E>(lds.tr8(Ks, kb * 32 + 16 * ks, nb), db, dq[nb]);
    }
  };
  // By the sequence's own length, not by the launch: the first part of a split axis holds four tiles at least, so all
  // of a short sequence, and the others have none of it.
  if (len <= 1) {
    // the softmax of a single state is constant: dQ = 0, and nothing of P's last bits in it
  } else if (len <= kKeys) {
    // One tile holds all states. With few of them, the rounding of O weighs in dO . O, which nearly equals the
    // dP it is taken from; here it is summed from P and dP themselves.
    key_loop<DP>(tile0, tile1, tile2, p, w, wave, lane, k_begin, k_end, [&](const unsigned char* Ks, const unsigned char* Vs, int k0) {
      if (!some) return;
      f32x16 s, dp;
      float sum = 0.f;
#pragma unroll 1
      for (int kb = 0; kb < 2; ++kb) {
        scores(Ks, Vs, k0, kb, s, dp);
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += s[i] * dp[i];
      }
      delta = half_sum(sum) * kUnliftBack<E>;
#pragma unroll 1
      for (int kb = 0; kb < 2; ++kb) {
        scores(Ks, Vs, k0, kb, s, dp);
        add(Ks, kb, s, dp);
      }
    });
  } else {
    key_loop<DP>(tile0, tile1, tile2, p, w, wave, lane, k_begin, k_end, [&](const unsigned char* Ks, const unsigned char* Vs, int k0) {
      if (!some) return;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        f32x16 s, dp;
        scores(Ks, Vs, k0, kb, s, dp);
        add(Ks, kb, s, dp);
      }
    });
  }
  if (mine && hh == 0 && w.split == 0) p.delta[stat] = delta;
  if (!mine) return;
  const float by = p.scale * gain.down();
  if (p.splits == 1) {
    each_quad<DP>(hh, p.D, [&](int col, int nb, int i) { put4<E>(p.out + dense + col, dq[nb], i, by); });
  } else {
    float* at = p.part + w.split * p.out_numel + dense;
    each_quad<DP>(hh, p.D, [&](int col, int nb, int i) { put4f(at + col, dq[nb], i, by); });
  }
}

// 128 keys, key on the lane; row tiles of RT through LDS. With wide heads K, dK and dV fill the registers, V comes from
// LDS; two waves sharing 32 keys, each with half of the columns, leave room but wait more (1235 us for 1050).
template <typename E, int DP, int RT>
__global__ void __launch_bounds__(kThreads, 2) cross_dkv_kernel(CrossParams p) {
  typedef Tile<DP> L;
  typedef Dma<DP, RT> Copy;
  constexpr int kEach = 2 * RT / 4;  // statistics that a wave fetches; its place in LDS holds 64
  struct Rows {
    unsigned char x[2][RT * L::RB];  // Q | dO
    float stat[4][64];               // lse, delta: kEach of each wave
  };
  __shared__ __attribute__((aligned(16))) Rows tile0, tile1, tile2;
  // with wide heads the registers do not hold V beside K, dK and dV: it is read from LDS where it is used
  constexpr bool kVInLds = DP > 96;
  __shared__ __attribute__((aligned(16))) unsigned char vs[kVInLds ? kRows * L::RB : 16];
  const Place w(p);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 31, hh = lane >> 5;
  const Places<DP> lds(lane);
  const int kw = w.block * kRows + wave * 32, key = kw + r;
  const int len = p.length(w.b);
  const bool some = kw < len;
  // a block of keys behind the last state has no work but its zeros
  const int r_begin = w.split * p.per_split;
  const int r_end = w.block * kRows < len ? p.split_end(r_begin, p.M) : r_begin;
  const u16* kbase = p.kv + w.b * p.kb + w.n * p.kh + (int64_t)key * p.kt;
  u16x8 kf[L::KS], vf[kVInLds ? 1 : L::KS];
  load_row<DP>(kf, key < len ? kbase : nullptr, hh, p.D);
  if constexpr (kVInLds) {  // each lane's half of its key's row, in the place that it reads again
#pragma unroll
    for (int k = 0; k < L::KS; ++k) {
      const int col = 16 * k + 8 * hh;
      *reinterpret_cast<u16x8*>(vs + L::off(wave * 32 + r, 2 * k + hh)) =
          key < len && col < p.D ? *reinterpret_cast<const u16x8*>(kbase + p.ks + col) : zero8();
    }
  } else {
    load_row<DP>(vf, key < len ? kbase + p.ks : nullptr, hh, p.D);
  }
  f32x16 dk[L::NB], dv[L::NB];
#pragma unroll
  for (int nb = 0; nb < L::NB; ++nb) dk[nb] = dv[nb] = zero16();
  Gain<E> gain;
  const bool second = Copy::second(wave);
  const int64_t H = (int64_t)p.N * p.G;
  const u16* base = second ? p.dout + w.b * (p.Tq * H * p.D) + (int64_t)w.n * p.G * p.D
                           : p.q + w.b * p.qb + (int64_t)w.n * p.G * p.qh;
  const int64_t st = second ? H * p.D : p.qt, sh = second ? p.D : p.qh;
  Copy copy;
  // Offsets of a tile's rows from its first token. Where tiles begin at whole tokens they are the same in every
  // tile but for the last, whose rows outside are struck out.
  const bool alike = RT % p.G == 0;
  auto place = [&](int skipped, int valid) {
    copy.place(wave, lane, p.D, [&](int i) {
      unsigned g;
      const unsigned t = p.by_G.divmod((unsigned)(i + skipped), g);
      return i < valid ? (unsigned)(((int)t * (int)st + (int)g * (int)sh) * 2) : kOutside;
    });
  };
  place(0, RT);
  const int mine = wave * kEach + lane;  // of the 2 RT statistics
  auto issue = [&](Rows& t, int r0) {
    const int begin = r0 < r_end ? r0 : 0, valid = r_end - r0;
    unsigned skipped;
    const unsigned token = p.by_G.divmod((unsigned)begin, skipped);
    if (!alike || (valid > 0 && valid < RT)) place((int)skipped, valid);
    copy.go(base + token * st, valid > 0 ? kOutside - 1 : 0u, t.x[second]);
    to_lds<4>((wave * kEach >= RT ? p.delta : p.lse) + (int64_t)w.bn * p.M + begin, valid > 0 ? 4u * min(valid, RT) : 0u,
              t.stat[wave], lane < kEach ? (unsigned)(mine % RT * 4) : kOutside);
  };
  auto step = [&](const Rows& t, int r0) {
    if (!some) return;
    const unsigned char *Qs = t.x[0], *Ds = t.x[1];
#pragma unroll
    for (int qs = 0; qs < RT / 32; ++qs) {
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int k = 0; k < L::KS; ++k) {
        s = mfma<E>(lds.row8(Qs, qs * 32, k), kf[k], s);
        dp = mfma<E>(lds.row8(Ds, qs * 32, k), kVInLds ? lds.row8(vs, wave * 32, k) : vf[kVInLds ? 0 : k], dp);
      }
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4) {
        const int qi = qs * 32 + 8 * g4 + 4 * hh;
        const float4 l4 = *reinterpret_cast<const float4*>(&t.stat[qi / kEach][qi % kEach]);
        const float4 d4 = *reinterpret_cast<const float4*>(&t.stat[(RT + qi) / kEach][qi % kEach]);
        const float ls[4] = {l4.x, l4.y, l4.z, l4.w}, dl[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = 4 * g4 + j;
          const float pv = exp2_fast(__builtin_fmaf(s[i], p.scale_log2, lift_back<E>(ls[j])));
          s[i] = pv;
          dp[i] = pv * (dp[i] - dl[j]);
        }
      }
      if (r0 + qs * 32 + 32 > r_end) {  // rows outside
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (r0 + qs * 32 + acc_row(i, hh) >= r_end) s[i] = dp[i] = 0.f;
      }
      gain.fit(dp, dk);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const u16x8 pb = to_operand<E>(s, ks), db = to_operand<E>(dp, ks);
#pragma unroll
        for (int nb = 0; nb < L::NB; ++nb) {
          dv[nb] = mfma<E>(lds.tr8(Ds, qs * 32 + 16 * ks, nb), pb, dv[nb]);
          dk[nb] = mfma<E>(lds.tr8(Qs, qs * 32 + 16 * ks, nb), db, dk[nb]);
        }
      }
    }
  };
  if (r_begin < r_end) {
    if constexpr (L::BUFS == 3) pipeline<Copy::kPer + 1, RT>(tile0, tile1, tile2, r_begin, r_end, issue, step);
    else pipeline<Copy::kPer + 1, RT>(tile0, tile1, r_begin, r_end, issue, step);
  }
  if (key >= p.Tk) return;
  // a lane whose key lies behind the last state has been computing with zeros for its key: its columns are not used
  const bool live = key < len;
  const float by = len == 1 ? 0.f : p.scale * gain.down();  // the softmax of a single state is constant: dK = 0
  const int64_t at = (((int64_t)w.b * p.Tk + key) * 2 * p.N + w.n) * p.D, to_v = (int64_t)p.N * p.D;
  if (!live) {
#pragma unroll
    for (int nb = 0; nb < L::NB; ++nb) dk[nb] = dv[nb] = zero16();
  }
  if (p.splits == 1) {
    each_quad<DP>(hh, p.D, [&](int col, int nb, int i) {
      put4<E>(p.dkv + at + col, dk[nb], i, by);
      put4<E>(p.dkv + at + to_v + col, dv[nb], i, kUnliftBack<E>);
    });
  } else {
    float* to = p.part + w.split * p.dkv_numel + at;
    each_quad<DP>(hh, p.D, [&](int col, int nb, int i) {
      put4f(to + col, dk[nb], i, by);
      put4f(to + to_v + col, dv[nb], i, kUnliftBack<E>);
    });
  }
}

struct PartSum {  // out[i] = sum over parts of part[s][i], in their order
  const float* part;
  u16* out;
  int64_t numel;  // a multiple of 8
  int parts;      // 0: nothing to add
  int blocks;
};

// the split dQ's and the split dK's and dV's sums, one launch
template <typename E>
__global__ void __launch_bounds__(kThreads) cross_sum_kernel(PartSum first, PartSum second) {
  const bool one = (int)blockIdx.x < first.blocks;
  const PartSum& j = one ? first : second;
  const int64_t at = ((int64_t)(blockIdx.x - (one ? 0 : first.blocks)) * kThreads + threadIdx.x) * 8;
  if (at >= j.numel) return;
  float a[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < j.parts; ++s) {
    const auto v = load_pack<float, 8>(j.part + s * j.numel + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] += v.v[i];
  }
  u16x8 o;
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = E::put(a[i]);
  *reinterpret_cast<u16x8*>(j.out + at) = o;
}

// ------------------------------------------------------------------------------ host side

int up(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// Splits an axis of `len` into parts of whole tiles, each of four at least, so that `have` workgroups become about
// kWanted. A tile takes a workgroup about 1.2 us and joining the parts one more launch of about 5 us (1848 rows x 80
// over 1499 keys: forward 9.7 us and 4.4 us of joining in six parts, about 30 us in one), so that an axis of fewer
// than twelve tiles stays whole.
void split_axis(CrossParams& p, int64_t have, int len, int tile) {
  const int tiles = up(len, tile);
  const int splits = tiles < 12 ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>(kWanted / std::max<int64_t>(1, have), tiles / 4));
  p.per_split = std::max(1, up(tiles, splits)) * tile;
  p.splits = std::max(1, up(len, p.per_split));
}

unsigned grid_of(const CrossParams& p) {
  const int64_t g = (int64_t)p.blocks * p.splits * p.B * p.N;
  TORCH_CHECK(g < (1ll << 24),
              "cross_attention: fewer than 2^24 workgroups wanted (sequences x key heads x blocks of 128 rows; for the states' "
              "gradient blocks of 128 states)");
  return (unsigned)g;
}

template <typename F>
void by_type_and_width(const CrossParams& p, at::ScalarType t, F&& f) {
  using std::integral_constant;
  auto width = [&](auto e) {
    if (p.D <= 64) f(e, integral_constant<int, 64>{});
    else if (p.D <= 96) f(e, integral_constant<int, 96>{});
    else f(e, integral_constant<int, 128>{});
  };
  t == at::kBFloat16 ? width(BF16{}) : width(FP16{});
}

typedef c10::optional<at::Tensor> OptTensor;

CrossParams cross_params(const at::Tensor& q, const at::Tensor& kv, const OptTensor& lengths, double scale) {
  CrossParams p{};
  p.q = (const u16*)q.data_ptr();
  p.kv = (const u16*)kv.data_ptr();
  p.qb = q.stride(0), p.qt = q.stride(1), p.qh = q.stride(2);
  p.kb = kv.stride(0), p.kt = kv.stride(1), p.ks = kv.stride(2), p.kh = kv.stride(3);
  if (kv.size(1) == 1) p.kt = 2 * kv.size(3) * kv.size(4);  // a single state may have any stride; rows behind it are outside
  p.B = (int)q.size(0), p.Tq = (int)q.size(1), p.Tk = (int)kv.size(1), p.N = (int)kv.size(3), p.D = (int)q.size(3);
  p.G = (int)(q.size(2) / kv.size(3));
  p.M = p.G * p.Tq;
  p.by_G = FastDiv((unsigned)p.G);
  if (lengths) {
    p.lengths = lengths->data_ptr();
    p.len64 = lengths->scalar_type() == at::kLong;
  }
  p.scale = (float)scale;
  p.scale_log2 = (float)(scale * 1.4426950408889634);
  p.out_numel = q.numel();
  p.dkv_numel = kv.numel();
  p.splits = 1;
  return p;
}

// q and kv are laid out for the kernels; lse only where a backward pass will want it
std::vector<at::Tensor> cross_fwd(const at::Tensor& q, const at::Tensor& kv, const OptTensor& lengths, double scale,
                                  bool with_lse) {
  c10::DeviceGuard guard(q.device());
  CrossParams p = cross_params(q, kv, lengths, scale);
  auto out = at::empty(q.sizes(), q.options());
  at::Tensor lse, part, ml;
  const auto f32 = q.options().dtype(at::kFloat);
  if (with_lse) lse = at::empty({p.B, p.N, p.M}, f32);
  if (out.numel() == 0) return {out, lse};
  if (p.Tk == 0) {
    out.zero_();
    return {out, lse};
  }
  p.out = (u16*)out.data_ptr();
  p.lse = with_lse ? lse.data_ptr<float>() : nullptr;
  const bool few = p.M <= 32;
  p.blocks = up(p.M, few ? 32 : kRows);
  split_axis(p, (int64_t)p.blocks * p.B * p.N, p.Tk, few ? 128 : kKeys);
  if (p.splits > 1) {
    part = at::empty({p.splits, (int64_t)p.B * p.N * p.M * p.D}, f32);
    ml = at::empty({p.splits, (int64_t)p.B * p.N * p.M, 2}, f32);
    p.part = part.data_ptr<float>();
    p.part_ml = ml.data_ptr<float>();
  }
  const unsigned grid = grid_of(p);
  by_type_and_width(p, q.scalar_type(), [&](auto e, auto dp) {
    typedef decltype(e) E;
    if (few)
      hipLaunchKernelGGL((cross_few_kernel<E, dp>), dim3(grid), dim3(kThreads), 0, stream(), p);
    else
      hipLaunchKernelGGL((cross_fwd_kernel<E, dp>), dim3(grid), dim3(kThreads), 0, stream(), p);
    LAUNCH_CHECK();
    if (p.splits > 1) {
      // by columns from a wave of them per SIMD on (28672 rows x 64 in two parts: one row per 64 threads takes 13.8 us)
      const int64_t rows = (int64_t)p.B * p.N * p.M, items = rows * (p.D / 4);
      if (items >= 65536 && p.splits <= 16)
        hipLaunchKernelGGL((cross_join_many_kernel<E>), dim3((unsigned)up(items, kThreads)), dim3(kThreads), 0, stream(), p,
                           (unsigned)items, FastDiv((unsigned)p.D / 4));
      else if (p.splits > 16)
        hipLaunchKernelGGL((cross_join_kernel<E, 256>), dim3((unsigned)rows), dim3(256), 0, stream(), p);
      else
        hipLaunchKernelGGL((cross_join_kernel<E, 64>), dim3((unsigned)rows), dim3(64), 0, stream(), p);
      LAUNCH_CHECK();
    }
  });
  return {out, lse};
}

std::vector<at::Tensor> cross_bwd(const at::Tensor& dout, const at::Tensor& q, const at::Tensor& kv, const at::Tensor& out,
                                  const at::Tensor& lse, const OptTensor& lengths, double scale, bool want_kv) {
  c10::DeviceGuard guard(q.device());
  CrossParams p = cross_params(q, kv, lengths, scale);
  auto dq = at::empty(q.sizes(), q.options());
  at::Tensor dkv = want_kv ? at::empty(kv.sizes(), kv.options()) : at::Tensor();
  if (q.numel() == 0 || kv.numel() == 0) return {dq.zero_(), want_kv ? dkv.zero_() : dkv};
  p.o = (const u16*)out.data_ptr();
  p.dout = (const u16*)dout.data_ptr();
  p.out = (u16*)dq.data_ptr();
  p.dkv = want_kv ? (u16*)dkv.data_ptr() : nullptr;
  p.lse = lse.data_ptr<float>();
  by_type_and_width(p, q.scalar_type(), [&](auto e, auto dp) {
    typedef decltype(e) E;
    constexpr int RT = dp <= 64 ? 64 : 32;
    CrossParams pk = p;  // dK, dV
    p.blocks = up(p.M, kRows);
    split_axis(p, (int64_t)p.blocks * p.B * p.N, p.Tk, kKeys);
    pk.blocks = up(p.Tk, kRows);
    split_axis(pk, (int64_t)pk.blocks * p.B * p.N, p.M, RT);
    // one workspace: the rows' sums of dP, then the parts of split gradients
    const int64_t rows = ((int64_t)p.B * p.N * p.M + 7) / 8 * 8;
    const int64_t nq = p.splits > 1 ? p.splits * p.out_numel : 0, nkv = want_kv && pk.splits > 1 ? pk.splits * p.dkv_numel : 0;
    auto work = at::empty({rows + nq + nkv}, q.options().dtype(at::kFloat));
    p.delta = pk.delta = work.data_ptr<float>();
    p.part = p.delta + rows;
    pk.part = p.part + nq;
    hipLaunchKernelGGL((cross_dq_kernel<E, dp>), dim3(grid_of(p)), dim3(kThreads), 0, stream(), p);
    LAUNCH_CHECK();
    if (want_kv) {
      hipLaunchKernelGGL((cross_dkv_kernel<E, dp, RT>), dim3(grid_of(pk)), dim3(kThreads), 0, stream(), pk);
      LAUNCH_CHECK();
    }
    auto job = [](const CrossParams& c, u16* to, int64_t n) {
      return PartSum{c.part, to, n, c.splits, to && c.splits > 1 ? up(n, 8 * kThreads) : 0};
    };
    const PartSum a = job(p, p.out, p.out_numel), b = job(pk, pk.dkv, pk.dkv_numel);
    if (a.blocks + b.blocks > 0) {
      hipLaunchKernelGGL((cross_sum_kernel<E>), dim3((unsigned)(a.blocks + b.blocks)), dim3(kThreads), 0, stream(), a, b);
      LAUNCH_CHECK();
    }
  });
  return {dq, dkv};
}

// Rows of whole 16-byte chunks at 16-byte addresses whose tiles stay within the copies' 31-bit offsets (tokens of
// one tile, and the heads of a group), or a dense copy that has them.
at::Tensor chunked(const at::Tensor& t) {
  bool ok = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) ok &= t.size(i) == 1 || t.stride(i) % 8 == 0;
  ok &= t.size(1) == 1 || t.stride(1) >= t.size(-1);  // a tile's rows end in their order
  const int64_t heads = t.dim() - 2;
  ok &= 2 * (kRows * t.stride(1) + t.size(heads) * t.stride(heads) + t.size(-1)) < (1ll << 30);
  if (ok) return t;
  auto c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone(at::MemoryFormat::Contiguous);
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct CrossFn : public torch::autograd::Function<CrossFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& kv, const OptTensor& lengths,
                            double scale) {
    auto qc = chunked(q), kc = chunked(kv);
    auto r = cross_fwd(qc, kc, lengths, scale, true);
    ctx->save_for_backward({qc, kc, r[0], r[1], lengths ? *lengths : at::Tensor()});
    ctx->saved_data["scale"] = scale;
    return r[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_order("cross_attention");
    auto s = ctx->get_saved_variables();
    OptTensor lengths;
    if (s[4].defined()) lengths = s[4];
    auto g = grads[0].contiguous();
    if (reinterpret_cast<uintptr_t>(g.data_ptr()) % 16) g = g.clone();
    // frozen states: no dK and dV (dQ's kernel always runs, it has the row sums)
    auto d = cross_bwd(g, s[0], s[1], s[2], s[3], lengths, ctx->saved_data["scale"].toDouble(), ctx->needs_input_grad(1));
    return {d[0], d[1], at::Tensor(), at::Tensor()};
  }
};

at::Tensor cross_attention(const at::Tensor& q, const at::Tensor& kv, const OptTensor& lengths, double scale) {
  const char* op = "cross_attention: ";
  no_tangents("cross_attention", q, kv);
  TORCH_CHECK(q.is_cuda() && kv.device() == q.device(), op, "q and kv must be on one GPU");
  TORCH_CHECK(q.scalar_type() == kv.scalar_type() && (q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf), op,
              "q and kv must both be bfloat16 or float16");
  TORCH_CHECK(q.dim() == 4 && kv.dim() == 5 && kv.size(2) == 2, op, "q must be [B, Tq, H, D] and kv [B, Tk, 2, N, D]");
  TORCH_CHECK(q.size(0) == kv.size(0) && q.size(3) == kv.size(4), op, "q and kv must agree in B and D");
  TORCH_CHECK(q.size(3) % 8 == 0 && q.size(3) >= 8 && q.size(3) <= 128, op, "D must be a multiple of 8 up to 128");
  TORCH_CHECK(kv.size(3) > 0 && q.size(2) > 0 && q.size(2) % kv.size(3) == 0, op, "N must divide H");
  TORCH_CHECK(q.size(1) * q.size(2) < (1ll << 31) - kRows && kv.size(1) < (1ll << 31) - kRows && q.size(0) < (1ll << 31), op,
              "fewer than 2^31 rows and states wanted");
  TORCH_CHECK(q.size(2) * q.size(3) <= (1 << 20), op, "H times D of at most 2^20 wanted");  // a tile's offsets fit 31 bits
  TORCH_CHECK(std::isfinite(scale) && scale > 0.0, op, "scale must be positive");
  OptTensor len;
  if (lengths) {
    TORCH_CHECK(lengths->dim() == 1 && lengths->size(0) == q.size(0) && lengths->device() == q.device() &&
                    (lengths->scalar_type() == at::kInt || lengths->scalar_type() == at::kLong),
                op, "lengths must be int32 or int64 [B] on the device of q");
    len = lengths->contiguous();
  }
  if (at::GradMode::is_enabled() && (q.requires_grad() || kv.requires_grad())) return CrossFn::apply(q, kv, len, scale);
  return cross_fwd(chunked(q), chunked(kv), len, scale, false)[0];
}

}  // namespace

void register_cross_attention(pybind11::module_& m) {
  m.def("cross_attention", &cross_attention, "attention of q [B, Tq, H, D] over packed kv [B, Tk, 2, N, D]");
}
