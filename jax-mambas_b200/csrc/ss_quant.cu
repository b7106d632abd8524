// 8-bit quantisation by blocks of 128 along a row, and its inverse, for
// sm_100a (the format: ss_quant.cuh). Bound by HBM: every value is read once
// and its code written once.
//
// Rows: 16 lanes share a block, 8 values each, so a warp takes two blocks per
// step and the maximum is four shuffles.
//
// Channel-major (batch, k, length), the scan's layout, whose rows are the
// (batch, length) positions: a CTA takes a tile of 128 channels x 64 positions,
// reads it along the positions, finds each position's maximum over the
// channels (shuffles, then the warps' maxima through shared memory) and
// transposes the codes through shared memory into 128-byte row segments.
//
// Measured: 8 x 5120 x 2048 bf16 channel-major 42.9 us (5.9 TB/s; the conversions to
// e4m3 keep issue at two thirds), its 16384 x 5120 codes back to bf16 41.3 us (6.1
// TB/s), 32 rows of 5120 1.9 us (the launch).
#include "ss_ops.h"
#include "ss_quant.cuh"

namespace mss {

template <typename T, bool kVec>
__global__ void __launch_bounds__(256) ss_quant_rows_kernel(const QuantParams p) {
  const int kb = (p.k + kQBlock - 1) / kQBlock;
  // blocks of all rows: below 2^31 (checked by the caller), so 32-bit division
  const unsigned blk = blockIdx.x * 16u + threadIdx.x / 16;
  const int sub = threadIdx.x & 15;
  const bool live = blk < static_cast<unsigned>(p.batch * p.length) * kb;
  const unsigned row32 = live ? blk / static_cast<unsigned>(kb) : 0u;
  const int64_t row = row32;
  const int b = live ? static_cast<int>(blk - row32 * kb) : 0;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  const int c0 = b * kQBlock + sub * 8;       // kVec: 8 consecutive values
  float f[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = 0.f;
  if constexpr (kVec) {
    if (live && c0 < p.k) ld8(x + c0, f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = b * kQBlock + j * 16 + sub;
      if (live && c < p.k) f[j] = Elem<T>::ld(x + c);
    }
  }
  float amax = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(f[j]));
  if (is_inf(amax)) {  // rare: the scale is the finite values', infinities become NaN
    amax = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      amax = fmaxf(amax, finite_abs(f[j]));
      f[j] = inf_to_nan(f[j]);
    }
  }
#pragma unroll
  for (int s = 8; s > 0; s >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, s));
  if (!live) return;
  const int byte = scale_byte(amax);
  const float s = scale_inverse(byte);
  uint8_t* codes = p.codes + row * p.code_stride;
  if constexpr (kVec) {
    if (c0 < p.k)
      *reinterpret_cast<uint2*>(codes + c0) =
          make_uint2(e4m3x4(f[0] * s, f[1] * s, f[2] * s, f[3] * s),
                     e4m3x4(f[4] * s, f[5] * s, f[6] * s, f[7] * s));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = b * kQBlock + j * 16 + sub;
      if (c < p.k) codes[c] = static_cast<uint8_t>(e4m3x2(f[j] * s, 0.f));
    }
  }
  if (sub == 0) p.scales[row * p.scale_stride + b] = static_cast<uint8_t>(byte);
}

constexpr int kTileL = 64;  // positions per tile

template <typename T, bool kVec>
__global__ void __launch_bounds__(256) ss_quant_cm_kernel(const QuantParams p) {
  __shared__ __align__(16) float wmax[8][kTileL];
  __shared__ __align__(16) float inverse[kTileL];
  // codes of position l, channels 4q..4q+3, as one word at word q ^ 4 (l / 8):
  // the stores of a warp (8 positions 8 apart x 4 words) fall into 32 banks
  __shared__ __align__(16) uint32_t tile[kTileL][32];
  const int lg = threadIdx.x & 7;   // positions 8 lg .. 8 lg + 7 of the tile
  const int q = threadIdx.x >> 3;   // channels 4 q .. 4 q + 3 of the block
  const int64_t l0 = static_cast<int64_t>(blockIdx.x) * kTileL;
  const int b = blockIdx.y;
  const int64_t z = blockIdx.z;
  const T* x = static_cast<const T*>(p.x) + z * p.k * p.length;
  float f[4][8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = b * kQBlock + q * 4 + i;
    const T* src = x + static_cast<int64_t>(c) * p.length;
    const int64_t l = l0 + lg * 8;
    if constexpr (kVec) {
      if (c < p.k && l < p.length) {
        ld8(src + l, f[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[i][j] = 0.f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        f[i][j] = c < p.k && l + j < p.length ? Elem<T>::ld(src + l + j) : 0.f;
    }
  }
  float amax[8];
  bool inf = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    amax[j] = fmaxf(fmaxf(fabsf(f[0][j]), fabsf(f[1][j])), fmaxf(fabsf(f[2][j]), fabsf(f[3][j])));
    inf = inf || is_inf(amax[j]);
  }
  if (inf) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      amax[j] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        amax[j] = fmaxf(amax[j], finite_abs(f[i][j]));
        f[i][j] = inf_to_nan(f[i][j]);
      }
    }
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    amax[j] = fmaxf(amax[j], __shfl_xor_sync(0xffffffffu, amax[j], 8));
    amax[j] = fmaxf(amax[j], __shfl_xor_sync(0xffffffffu, amax[j], 16));
  }
  if (lane < 8) {
#pragma unroll
    for (int j = 0; j < 8; ++j) wmax[warp][lg * 8 + j] = amax[j];
  }
  __syncthreads();
  if (threadIdx.x < kTileL) {  // one thread per position joins the warps' maxima
    const int l = threadIdx.x;
    float a = 0.f;  // of a position of nothing but NaN, whose maxima are NaN
#pragma unroll
    for (int w = 0; w < 8; ++w) a = fmaxf(a, wmax[w][l]);
    const int byte = scale_byte(a);
    inverse[l] = scale_inverse(byte);
    if (l0 + l < p.length)
      p.scales[(z * p.length + l0 + l) * p.scale_stride + b] = static_cast<uint8_t>(byte);
  }
  __syncthreads();
  float s[8];
  ld8(&inverse[lg * 8], s);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    tile[lg * 8 + j][q ^ (4 * lg)] =
        e4m3x4(f[0][j] * s[j], f[1][j] * s[j], f[2][j] * s[j], f[3][j] * s[j]);
  __syncthreads();
  // 8 threads write one position's 128 bytes; code rows are 16-byte aligned
  // and their stride covers k rounded up to 16, so a 16-byte store that holds
  // at least one channel stays inside its row
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int l = (threadIdx.x >> 3) + i * 32;
    const int w = (threadIdx.x & 7) * 4;
    const int c = b * kQBlock + w * 4;
    if (l0 + l < p.length && c < p.k)
      *reinterpret_cast<uint4*>(p.codes + (z * p.length + l0 + l) * p.code_stride + c) =
          *reinterpret_cast<const uint4*>(&tile[l][w ^ (4 * (l >> 3))]);
  }
}

// Both forms of a matrix at once: a CTA takes a tile of 128 x 128, whose rows are
// one block each of the row form and whose columns are one block each of the
// column form. A thread holds 4 rows x 8 columns; row maxima are shuffles over
// the 16 threads of a row, column maxima one shuffle and the warps' maxima
// through shared memory, and the column codes are transposed through shared
// memory into 128-byte segments.
template <typename T, bool kVec>
__global__ void __launch_bounds__(512, 2) ss_quant_both_kernel(const QuantBothParams p) {
  __shared__ __align__(16) float wmax[16][kQBlock];
  __shared__ __align__(16) float inverse[kQBlock];
  // codes of column c, rows 4q..4q+3, as one word at word q ^ 2 (c / 8): the stores
  // of a warp (16 columns 8 apart x 2 words) fall into 32 banks
  __shared__ __align__(16) uint32_t tile[kQBlock][32];
  const int cg = threadIdx.x & 15, q = threadIdx.x >> 4;
  const int k0 = blockIdx.x * kQBlock, m0 = blockIdx.y * kQBlock;
  const int c0 = k0 + cg * 8, r0 = m0 + q * 4;
  float f[4][8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const T* src = static_cast<const T*>(p.x) + static_cast<int64_t>(r0 + i) * p.x_stride + c0;
    if (kVec) {
      if (r0 + i < p.rows && c0 < p.k) {
        ld8(src, f[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[i][j] = 0.f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        f[i][j] = r0 + i < p.rows && c0 + j < p.k ? Elem<T>::ld(src + j) : 0.f;
    }
  }
  float rmax[4], cmax[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) cmax[j] = 0.f;
  float any = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    rmax[i] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      rmax[i] = fmaxf(rmax[i], fabsf(f[i][j]));
      cmax[j] = fmaxf(cmax[j], fabsf(f[i][j]));
    }
    any = fmaxf(any, rmax[i]);
  }
  if (is_inf(any)) {  // rare: scales of the finite values, infinities become NaN
#pragma unroll
    for (int j = 0; j < 8; ++j) cmax[j] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      rmax[i] = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        rmax[i] = fmaxf(rmax[i], finite_abs(f[i][j]));
        cmax[j] = fmaxf(cmax[j], finite_abs(f[i][j]));
        f[i][j] = inf_to_nan(f[i][j]);
      }
    }
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < 8; ++j) cmax[j] = fmaxf(cmax[j], __shfl_xor_sync(0xffffffffu, cmax[j], 16));
  if (lane < 16) st8(&wmax[warp][cg * 8], cmax);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
      rmax[i] = fmaxf(rmax[i], __shfl_xor_sync(0xffffffffu, rmax[i], o));
    const int byte = scale_byte(rmax[i]);
    const float s = scale_inverse(byte);
    if (r0 + i < p.rows) {
      uint8_t* dst = p.row_codes + static_cast<int64_t>(r0 + i) * p.row_stride + c0;
      if (c0 < p.k)  // rows are padded to 16 bytes
        *reinterpret_cast<uint2*>(dst) =
            make_uint2(e4m3x4(f[i][0] * s, f[i][1] * s, f[i][2] * s, f[i][3] * s),
                       e4m3x4(f[i][4] * s, f[i][5] * s, f[i][6] * s, f[i][7] * s));
      if (cg == 0)
        p.row_scales[static_cast<int64_t>(r0 + i) * p.row_scale_stride + blockIdx.x] = static_cast<uint8_t>(byte);
    }
  }
  __syncthreads();
  if (threadIdx.x < kQBlock) {  // one thread per column joins the warps' maxima
    const int c = threadIdx.x;
    float a = wmax[0][c];
#pragma unroll
    for (int w = 1; w < 16; ++w) a = fmaxf(a, wmax[w][c]);
    const int byte = scale_byte(a);
    inverse[c] = scale_inverse(byte);
    if (k0 + c < p.k)
      p.col_scales[static_cast<int64_t>(k0 + c) * p.col_scale_stride + blockIdx.y] = static_cast<uint8_t>(byte);
  }
  __syncthreads();
  float s[8];
  ld8(&inverse[cg * 8], s);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    tile[cg * 8 + j][q ^ (2 * cg)] =
        e4m3x4(f[0][j] * s[j], f[1][j] * s[j], f[2][j] * s[j], f[3][j] * s[j]);
  __syncthreads();
  // 8 threads write one column's 128 bytes (see the tail rule above). Word w of a
  // column lies at w ^ 2x: its pieces of four words permuted, each piece's halves
  // swapped where x is odd.
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = (threadIdx.x >> 3) + i * 64;
    const int piece = threadIdx.x & 7;
    const int m = m0 + piece * 16;
    if (k0 + c < p.k && m < p.rows) {
      const int x = c >> 3;
      const uint4 w = *reinterpret_cast<const uint4*>(&tile[c][(4 * piece) ^ ((2 * x) & 28)]);
      *reinterpret_cast<uint4*>(p.col_codes + static_cast<int64_t>(k0 + c) * p.col_stride + m) =
          x & 1 ? make_uint4(w.z, w.w, w.x, w.y) : w;
    }
  }
}

// ------------------------------------------- bf16, two values per instruction
// The two transposing forms for aligned bf16 keep the values as they come, two per
// register: magnitudes are compared as 16-bit whole numbers (the order of
// non-negative floats), and the power-of-two scale is applied in bf16, which is
// exact down to results that e4m3 rounds to zero anyway. Half the registers and
// three quarters of the instructions of the forms above: 8 x 5120 x 2048
// channel-major takes 42.9 us (5.9 TB/s) against 50.8, 8192 x 5120 in both forms
// 34.4 (4.9 TB/s) against 37. (Taking 1 to 32 row tiles of one column tile after
// the other, for longer runs of the column codes, changes nothing.)
constexpr uint32_t kAbs2 = 0x7fff7fffu;
constexpr uint32_t kInfBits = 0x7f80u;

// Largest 16-bit magnitude of a pair's halves.
__device__ __forceinline__ uint32_t pair_max(uint32_t m) { return max(m >> 16, m & 0xffffu); }

// A pair with its infinities made NaN, and its finite magnitudes (others zero).
__device__ __forceinline__ uint32_t pair_nan(uint32_t w) {
  const uint32_t lo = (w & 0x7fffu) >= kInfBits ? 0x7fffu : w & 0xffffu;
  const uint32_t hi = ((w >> 16) & 0x7fffu) >= kInfBits ? 0x7fffu : w >> 16;
  return lo | (hi << 16);
}
__device__ __forceinline__ uint32_t pair_finite_abs(uint32_t w) {
  const uint32_t lo = w & 0x7fffu, hi = (w >> 16) & 0x7fffu;
  return (lo >= kInfBits ? 0u : lo) | ((hi >= kInfBits ? 0u : hi) << 16);
}
__device__ __forceinline__ int pair_scale_byte(uint32_t bits) {
  return scale_byte(__uint_as_float(bits << 16));
}
// 2^-e as bf16 bits (its low half of a float is zero).
__device__ __forceinline__ uint32_t inverse_bits(int byte) {
  return __float_as_uint(scale_inverse(byte)) >> 16;
}
__device__ __forceinline__ uint32_t scaled(uint32_t w, uint32_t s) {
  const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w),
                                   *reinterpret_cast<const __nv_bfloat162*>(&s));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ float low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

__global__ void __launch_bounds__(256, 6) ss_quant_cm_bf16_kernel(const QuantParams p) {
  __shared__ __align__(16) uint4 wmax[8][kTileL / 8];
  __shared__ __align__(16) unsigned short inverse[kTileL];
  __shared__ __align__(16) uint32_t tile[kTileL][32];
  const int lg = threadIdx.x & 7;   // positions 8 lg .. 8 lg + 7 of the tile
  const int q = threadIdx.x >> 3;   // channels 4 q .. 4 q + 3 of the block
  const int64_t l0 = static_cast<int64_t>(blockIdx.x) * kTileL;
  const int b = blockIdx.y;
  const int64_t z = blockIdx.z;
  const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(p.x) + z * p.k * p.length;
  uint32_t v[4][4];  // channel, position pair
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = b * kQBlock + q * 4 + i;
    uint4 w = make_uint4(0u, 0u, 0u, 0u);
    if (c < p.k && l0 + lg * 8 < p.length)
      w = *reinterpret_cast<const uint4*>(x + static_cast<int64_t>(c) * p.length + l0 + lg * 8);
    v[i][0] = w.x; v[i][1] = w.y; v[i][2] = w.z; v[i][3] = w.w;
  }
  uint32_t m[4], any = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    m[e] = __vmaxu2(__vmaxu2(v[0][e] & kAbs2, v[1][e] & kAbs2),
                    __vmaxu2(v[2][e] & kAbs2, v[3][e] & kAbs2));
    any = __vmaxu2(any, m[e]);
  }
  if (pair_max(any) >= kInfBits) {  // rare: scales of the finite values, infinities become NaN
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      m[e] = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        m[e] = __vmaxu2(m[e], pair_finite_abs(v[i][e]));
        v[i][e] = pair_nan(v[i][e]);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    m[e] = __vmaxu2(m[e], __shfl_xor_sync(0xffffffffu, m[e], 8));
    m[e] = __vmaxu2(m[e], __shfl_xor_sync(0xffffffffu, m[e], 16));
  }
  if ((threadIdx.x & 31) < 8) wmax[threadIdx.x >> 5][lg] = make_uint4(m[0], m[1], m[2], m[3]);
  __syncthreads();
  if (threadIdx.x < kTileL) {  // one thread per position joins the warps' maxima
    const int l = threadIdx.x;
    uint32_t a = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w)
      a = max(a, static_cast<uint32_t>(reinterpret_cast<const unsigned short*>(wmax[w])[l]));
    const int byte = pair_scale_byte(a);
    inverse[l] = static_cast<unsigned short>(inverse_bits(byte));
    if (l0 + l < p.length)
      p.scales[(z * p.length + l0 + l) * p.scale_stride + b] = static_cast<uint8_t>(byte);
  }
  __syncthreads();
  const uint4 s4 = *reinterpret_cast<const uint4*>(&inverse[lg * 8]);
  const uint32_t s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = scaled(v[i][e], s[e]);
    tile[lg * 8 + 2 * e][q ^ (4 * lg)] = e4m3x4(low(w[0]), low(w[1]), low(w[2]), low(w[3]));
    tile[lg * 8 + 2 * e + 1][q ^ (4 * lg)] = e4m3x4(high(w[0]), high(w[1]), high(w[2]), high(w[3]));
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {  // as above
    const int l = (threadIdx.x >> 3) + i * 32;
    const int w = (threadIdx.x & 7) * 4;
    const int c = b * kQBlock + w * 4;
    if (l0 + l < p.length && c < p.k)
      *reinterpret_cast<uint4*>(p.codes + (z * p.length + l0 + l) * p.code_stride + c) =
          *reinterpret_cast<const uint4*>(&tile[l][w ^ (4 * (l >> 3))]);
  }
}

__global__ void __launch_bounds__(512, 3) ss_quant_both_bf16_kernel(const QuantBothParams p) {
  __shared__ __align__(16) uint4 wmax[16][kQBlock / 8];
  __shared__ __align__(16) unsigned short inverse[kQBlock];
  __shared__ __align__(16) uint32_t tile[kQBlock][32];
  const int cg = threadIdx.x & 15, q = threadIdx.x >> 4;
  const int k0 = blockIdx.x * kQBlock, m0 = blockIdx.y * kQBlock;
  const int c0 = k0 + cg * 8, r0 = m0 + q * 4;
  uint32_t v[4][4];  // row, column pair
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint4 w = make_uint4(0u, 0u, 0u, 0u);
    if (r0 + i < p.rows && c0 < p.k)
      w = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.x) +
                                          static_cast<int64_t>(r0 + i) * p.x_stride + c0);
    v[i][0] = w.x; v[i][1] = w.y; v[i][2] = w.z; v[i][3] = w.w;
  }
  uint32_t col[4], row[4];
  auto maxima = [&](auto magnitude) {
#pragma unroll
    for (int e = 0; e < 4; ++e) col[e] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t r = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t a = magnitude(v[i][e]);
        r = __vmaxu2(r, a);
        col[e] = __vmaxu2(col[e], a);
      }
      row[i] = pair_max(r);
    }
  };
  maxima([](uint32_t w) { return w & kAbs2; });
  if (max(max(row[0], row[1]), max(row[2], row[3])) >= kInfBits) {  // rare, as above
    maxima([](uint32_t w) { return pair_finite_abs(w); });
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i][e] = pair_nan(v[i][e]);
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int e = 0; e < 4; ++e) col[e] = __vmaxu2(col[e], __shfl_xor_sync(0xffffffffu, col[e], 16));
  if (lane < 16) wmax[warp][cg] = make_uint4(col[0], col[1], col[2], col[3]);
  uint32_t two[2] = {row[0] | (row[1] << 16), row[2] | (row[3] << 16)};  // two rows per word
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
      two[h] = __vmaxu2(two[h], __shfl_xor_sync(0xffffffffu, two[h], o));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int byte = pair_scale_byte(i & 1 ? two[i / 2] >> 16 : two[i / 2] & 0xffffu);
    const uint32_t one = inverse_bits(byte), s = one | (one << 16);
    if (r0 + i < p.rows) {
      if (c0 < p.k) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = scaled(v[i][e], s);
        *reinterpret_cast<uint2*>(p.row_codes + static_cast<int64_t>(r0 + i) * p.row_stride + c0) =
            make_uint2(e4m3x4(low(w[0]), high(w[0]), low(w[1]), high(w[1])),
                       e4m3x4(low(w[2]), high(w[2]), low(w[3]), high(w[3])));
      }
      if (cg == 0)
        p.row_scales[static_cast<int64_t>(r0 + i) * p.row_scale_stride + blockIdx.x] =
            static_cast<uint8_t>(byte);
    }
  }
  __syncthreads();
  if (threadIdx.x < kQBlock) {  // one thread per column joins the warps' maxima
    const int c = threadIdx.x;
    uint32_t a = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w)
      a = max(a, static_cast<uint32_t>(reinterpret_cast<const unsigned short*>(wmax[w])[c]));
    const int byte = pair_scale_byte(a);
    inverse[c] = static_cast<unsigned short>(inverse_bits(byte));
    if (k0 + c < p.k)
      p.col_scales[static_cast<int64_t>(k0 + c) * p.col_scale_stride + blockIdx.y] =
          static_cast<uint8_t>(byte);
  }
  __syncthreads();
  const uint4 s4 = *reinterpret_cast<const uint4*>(&inverse[cg * 8]);
  const uint32_t s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = scaled(v[i][e], s[e]);
    tile[cg * 8 + 2 * e][q ^ (2 * cg)] = e4m3x4(low(w[0]), low(w[1]), low(w[2]), low(w[3]));
    tile[cg * 8 + 2 * e + 1][q ^ (2 * cg)] = e4m3x4(high(w[0]), high(w[1]), high(w[2]), high(w[3]));
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {  // as above
    const int c = (threadIdx.x >> 3) + i * 64;
    const int piece = threadIdx.x & 7;
    const int m = m0 + piece * 16;
    if (k0 + c < p.k && m < p.rows) {
      const int x = c >> 3;
      const uint4 w = *reinterpret_cast<const uint4*>(&tile[c][(4 * piece) ^ ((2 * x) & 28)]);
      *reinterpret_cast<uint4*>(p.col_codes + static_cast<int64_t>(k0 + c) * p.col_stride + m) =
          x & 1 ? make_uint4(w.z, w.w, w.x, w.y) : w;
    }
  }
}

// 16 codes per thread and step.
template <typename T>
__global__ void __launch_bounds__(256) ss_dequant_kernel(const DequantParams p) {
  const unsigned per_row = (p.k + 15) / 16;
  const bool whole = p.k % 16 == 0;
  // consecutive CTAs take consecutive runs of rows; within a run, 32-bit division
  const int64_t run = (p.rows + gridDim.x - 1) / gridDim.x;
  const int64_t row0 = run * blockIdx.x;
  const int64_t rows = min(run, p.rows - row0);
  if (rows <= 0) return;
  const uint8_t* codes = p.codes + row0 * p.code_stride;
  const uint8_t* scales = p.scales + row0 * p.scale_stride;
  T* out = static_cast<T*>(p.out) + row0 * p.k;
  const unsigned n = static_cast<unsigned>(rows) * per_row;
  for (unsigned i = threadIdx.x; i < n; i += 256) {
    const unsigned row = i / per_row;
    const unsigned c = (i - row * per_row) * 16;
    // code rows start and end on 16 bytes
    const uint4 w =
        __ldg(reinterpret_cast<const uint4*>(codes + static_cast<size_t>(row) * p.code_stride + c));
    const float s = scale_value(__ldg(scales + static_cast<size_t>(row) * p.scale_stride + c / kQBlock));
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
    T* dst = out + static_cast<size_t>(row) * p.k + c;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __nv_fp8x2_storage_t two =
            static_cast<__nv_fp8x2_storage_t>((words[2 * h + j / 2] >> (16 * (j & 1))) & 0xffffu);
        const float2 v = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3)));
        f[2 * j] = v.x * s;
        f[2 * j + 1] = v.y * s;
      }
      if (whole) {  // the output is dense and 16-byte aligned
        st8(dst + 8 * h, f);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (static_cast<int>(c) + 8 * h + j < p.k) Elem<T>::st(dst + 8 * h + j, f[j]);
      }
    }
  }
}

template <typename T>
static cudaError_t quant_go(const QuantParams& p, bool channel_major, cudaStream_t stream) {
  const bool aligned = (reinterpret_cast<uintptr_t>(p.x) & 15) == 0;
  const int kb = (p.k + kQBlock - 1) / kQBlock;
  if (!channel_major) {
    const int64_t blocks = p.batch * p.length * kb;
    const unsigned grid = static_cast<unsigned>((blocks + 15) / 16);
    if (aligned && p.k % 8 == 0 && p.x_stride % 8 == 0)
      ss_quant_rows_kernel<T, true><<<grid, 256, 0, stream>>>(p);
    else
      ss_quant_rows_kernel<T, false><<<grid, 256, 0, stream>>>(p);
  } else {
    const dim3 grid(static_cast<unsigned>((p.length + kTileL - 1) / kTileL),
                    static_cast<unsigned>(kb), static_cast<unsigned>(p.batch));
    const bool vec = aligned && p.length % 8 == 0;
    if (vec && std::is_same<T, __nv_bfloat16>::value)
      ss_quant_cm_bf16_kernel<<<grid, 256, 0, stream>>>(p);
    else if (vec)
      ss_quant_cm_kernel<float, true><<<grid, 256, 0, stream>>>(p);
    else
      ss_quant_cm_kernel<T, false><<<grid, 256, 0, stream>>>(p);
  }
  return cudaPeekAtLastError();
}

cudaError_t launch_quantize(const QuantParams& p, int x_dtype, bool channel_major,
                            cudaStream_t stream) {
  return x_dtype == MSS_BF16 ? quant_go<__nv_bfloat16>(p, channel_major, stream)
                             : quant_go<float>(p, channel_major, stream);
}

cudaError_t launch_quantize_both(const QuantBothParams& p, int x_dtype, cudaStream_t stream) {
  const dim3 grid((p.k + kQBlock - 1) / kQBlock, (p.rows + kQBlock - 1) / kQBlock);
  const bool vec =
      (reinterpret_cast<uintptr_t>(p.x) & 15) == 0 && p.k % 8 == 0 && p.x_stride % 8 == 0;
  if (x_dtype == MSS_BF16) {
    if (vec)
      ss_quant_both_bf16_kernel<<<grid, 512, 0, stream>>>(p);
    else
      ss_quant_both_kernel<__nv_bfloat16, false><<<grid, 512, 0, stream>>>(p);
  } else {
    if (vec)
      ss_quant_both_kernel<float, true><<<grid, 512, 0, stream>>>(p);
    else
      ss_quant_both_kernel<float, false><<<grid, 512, 0, stream>>>(p);
  }
  return cudaPeekAtLastError();
}

cudaError_t launch_dequantize(const DequantParams& p, int out_dtype, cudaStream_t stream) {
  // runs of about 4096 codes per CTA, and never 2^31 pieces of 16 in one
  const int64_t per_row = (p.k + 15) / 16;
  const int64_t rows = std::max<int64_t>(1, 256 / per_row);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>((p.rows + rows - 1) / rows, 1 << 22));
  if (out_dtype == MSS_BF16)
    ss_dequant_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(p);
  else
    ss_dequant_kernel<float><<<grid, 256, 0, stream>>>(p);
  return cudaPeekAtLastError();
}

}  // namespace mss
