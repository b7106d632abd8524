// RMS norm with the residual's addition, forward and backward, for sm_100a.
//
//   h = x + r, rounded to the residual stream's type (h = x without r)
//   y = h s w,  s = (mean(h^2) + eps)^(-1/2)
//   g = dy w;  dh = s (g - h s^2 mean(g h)) + dh_in;  dx = dr = dh
//   dw = sum over rows of dy h s
//
// The norm is taken of h as it is stored, so the backward, which reads h
// back, differentiates the very function that the forward computed. All sums
// and products are fp32; y, h, dx, dr are each rounded once.
//
// Both directions are bound by HBM. A row is read once, kept in registers
// through its sums, and written once. Rows up to 64 wide take 8 lanes, up to
// 1024 one warp (four rows per CTA, sums by shuffles alone); wider rows take
// a CTA of just enough warps at 8 elements per vector and kNV vectors per
// thread. The 8-bit output quantises from the fp32 y in registers: one more
// shuffle maximum per block of 128.
//
// Measured (bf16 branch, fp32 residual stream): forward with 8-bit output 32768 x
// 2560 138 us, 6.7 TB/s of algorithmic bytes; forward 16384 x 768 23.8 us (6.3
// TB/s); backward 16384 x 768 34.6 us (5.8 TB/s; with the weight gradient's sum of 4.6 us
// 5.1), 16384 x 2560 105 us (6.4 TB/s).
// fp32 rows of 1001 (single-element accesses) 6185 rows: 11.3 and 14.2 us, 4.4 and
// 5.2 TB/s. Few rows are bound by the launch: 32 x 2560 3.1 us.
#include "ss_ops.h"
#include "ss_quant.cuh"

namespace mss {

struct Codes {};  // output tag: e4m3 codes and scales
struct NoRes {};  // residual tag: none

// Where a thread's eight elements of vector slot v lie. kVec: consecutive
// (16-byte accesses; dim, strides and pointers are multiples of 8 elements).
// Otherwise lane-strided, so that single-element accesses of a warp coalesce.
template <int W, bool kVec>
struct Lay {
  int warp, lane, nwarps;
  __device__ __forceinline__ Lay(int t, int tpr) : warp(t / W), lane(t % W), nwarps(tpr / W) {}
  __device__ __forceinline__ int base(int v) const { return (v * nwarps + warp) * W * 8; }
  __device__ __forceinline__ int at(int v, int j) const {
    return base(v) + (kVec ? lane * 8 + j : j * W + lane);
  }
};

template <int W, bool kVec, typename T>
__device__ __forceinline__ void load8(const Lay<W, kVec>& l, int v, int dim, const T* row,
                                      float (&f)[8]) {
  if constexpr (kVec) {
    if (l.at(v, 0) < dim) {
      ld8(row + l.at(v, 0), f);
      return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = 0.f;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = l.at(v, j) < dim ? Elem<T>::ld(row + l.at(v, j)) : 0.f;
  }
}

template <int W, bool kVec, typename T>
__device__ __forceinline__ void store8(const Lay<W, kVec>& l, int v, int dim, T* row,
                                       const float (&f)[8]) {
  if constexpr (kVec) {
    if (l.at(v, 0) < dim) st8(row + l.at(v, 0), f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (l.at(v, j) < dim) Elem<T>::st(row + l.at(v, j), f[j]);
  }
}

// A thread's eight elements as they come from memory (four registers of bf16
// where they are read by 16 bytes).
template <typename T, bool kVec>
struct Held {
  static constexpr bool kPacked = kVec && std::is_same<T, __nv_bfloat16>::value;
  typename std::conditional<kPacked, uint4, float[8]>::type v;
  __device__ __forceinline__ void zero() {
    if constexpr (kPacked) {
      v = make_uint4(0u, 0u, 0u, 0u);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.f;
    }
  }
  template <int W>
  __device__ __forceinline__ void load(const Lay<W, kVec>& l, int dim, const T* row) {
    if constexpr (kPacked) {
      if (l.at(0, 0) < dim)
        v = *reinterpret_cast<const uint4*>(row + l.at(0, 0));
      else
        zero();
    } else {
      load8(l, 0, dim, row, v);
    }
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    if constexpr (kPacked) {
      const float4 a = bf16x4_to_f32(make_uint2(v.x, v.y));
      const float4 b = bf16x4_to_f32(make_uint2(v.z, v.w));
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
      f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = v[j];
    }
  }
};

// Sum over the W lanes of a group.
template <int W>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int s = W / 2; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
  return v;
}
template <int W>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int s = W / 2; s > 0; s >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, s));
  return v;
}

// Codes and scales of one vector slot. Its elements span one block of 128
// (W = 8) or two (W = 32: lanes 0-15 / 16-31, or j 0-3 / 4-7 lane-strided).
// Every lane of the warp must call it.
template <int W, bool kVec>
__device__ __forceinline__ void quant8(const Lay<W, kVec>& l, int v, int dim, float (&f)[8],
                                       uint8_t* codes, uint8_t* scales, bool live) {
  constexpr int kHalves = W == 32 && !kVec ? 2 : 1;
  float amax[kHalves];
  bool inf = false;
#pragma unroll
  for (int h = 0; h < kHalves; ++h) {
    amax[h] = 0.f;
#pragma unroll
    for (int j = 0; j < 8 / kHalves; ++j) amax[h] = fmaxf(amax[h], fabsf(f[h * 4 + j]));
    inf = inf || is_inf(amax[h]);
  }
  if (inf) {  // rare: the scale is the finite values', infinities become NaN
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      amax[h] = 0.f;
#pragma unroll
      for (int j = 0; j < 8 / kHalves; ++j) amax[h] = fmaxf(amax[h], finite_abs(f[h * 4 + j]));
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = inf_to_nan(f[j]);
  }
  int byte[kHalves];
#pragma unroll
  for (int h = 0; h < kHalves; ++h) {
    amax[h] = group_max<W == 32 && kVec ? 16 : W>(amax[h]);
    byte[h] = scale_byte(amax[h]);
  }
  if (!live) return;
  if constexpr (kVec) {
    const float s = scale_inverse(byte[0]);
    const int c = l.at(v, 0);
    if (c < dim) {
      *reinterpret_cast<uint2*>(codes + c) =
          make_uint2(e4m3x4(f[0] * s, f[1] * s, f[2] * s, f[3] * s),
                     e4m3x4(f[4] * s, f[5] * s, f[6] * s, f[7] * s));
      if (c % kQBlock == 0) scales[c / kQBlock] = static_cast<uint8_t>(byte[0]);
    }
  } else {
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      const float s = scale_inverse(byte[h]);
#pragma unroll
      for (int j = 0; j < 8 / kHalves; ++j) {
        const int c = l.at(v, h * 4 + j);
        if (c < dim) codes[c] = static_cast<uint8_t>(e4m3x2(f[h * 4 + j] * s, 0.f));
      }
      const int c = l.base(v) + h * kQBlock;
      if (l.lane == 0 && c < dim) scales[c / kQBlock] = static_cast<uint8_t>(byte[h]);
    }
  }
}

// Sum over the TPR threads of a row: shuffles, and for a CTA per row its warps'
// sums through shared memory in warp order. `slot` alternates between calls
// so that one barrier per call suffices.
template <int W, bool kCta, int kN>
__device__ __forceinline__ void row_sum(float (&v)[kN], float (*buf)[kN][32], int& slot) {
#pragma unroll
  for (int i = 0; i < kN; ++i) v[i] = group_sum<W>(v[i]);
  if constexpr (kCta) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane < kN) {
      float mine = v[0];
#pragma unroll
      for (int i = 1; i < kN; ++i) mine = lane == i ? v[i] : mine;
      buf[slot][lane][warp] = mine;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      v[i] = 0.f;
      const int n = blockDim.x >> 5;
      for (int w = 0; w < n; ++w) v[i] += buf[slot][i][w];
    }
    slot ^= 1;
  }
}

// kTPR threads share a row: 8, 32, or 0 for the whole CTA.
template <typename XT, typename RT, typename OT, int kTPR, int kNV, bool kVec>
__global__ void __launch_bounds__(kTPR ? 128 : 512) ss_norm_fwd_kernel(const NormParams p) {
  constexpr int W = kTPR == 8 ? 8 : 32;
  constexpr bool kRes = !std::is_same<RT, NoRes>::value;
  __shared__ float buf[2][1][32];
  const int tpr = kTPR ? kTPR : blockDim.x;
  const int t = kTPR ? threadIdx.x % kTPR : threadIdx.x;
  const int64_t row = kTPR ? static_cast<int64_t>(blockIdx.x) * (128 / kTPR) + threadIdx.x / kTPR
                           : blockIdx.x;
  const bool live = row < p.rows;
  const int64_t r = live ? row : 0;
  const Lay<W, kVec> l(t, tpr);
  const int dim = live ? p.dim : 0;  // no accesses past the last row

  float f[kNV][8];
  const XT* x = static_cast<const XT*>(p.x) + r * p.x_stride;
#pragma unroll
  for (int v = 0; v < kNV; ++v) load8(l, v, dim, x, f[v]);
  if constexpr (kRes) {
    const RT* res = static_cast<const RT*>(p.res) + r * p.res_stride;
    RT* h = static_cast<RT*>(p.h) + r * p.dim;
#pragma unroll
    for (int v = 0; v < kNV; ++v) {
      float q[8];
      load8(l, v, dim, res, q);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        f[v][j] += q[j];
        if constexpr (std::is_same<RT, __nv_bfloat16>::value)
          f[v][j] = to_f32(__float2bfloat16_rn(f[v][j]));
      }
      store8(l, v, dim, h, f[v]);
    }
  }
  float ss[1] = {0.f};
#pragma unroll
  for (int v = 0; v < kNV; ++v)
#pragma unroll
    for (int j = 0; j < 8; ++j) ss[0] = fmaf(f[v][j], f[v][j], ss[0]);
  int slot = 0;
  row_sum<W, kTPR == 0, 1>(ss, buf, slot);
  const float rstd = rsqrtf(ss[0] / static_cast<float>(p.dim) + p.eps);
#pragma unroll
  for (int v = 0; v < kNV; ++v) {
    float w[8];
    load8(l, v, dim, p.weight, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[v][j] = f[v][j] * rstd * w[j];
    if constexpr (std::is_same<OT, Codes>::value) {
      quant8(l, v, dim, f[v], p.codes + r * p.code_stride, p.scales + r * p.scale_stride, live);
    } else {
      store8(l, v, dim, static_cast<OT*>(p.y) + r * p.dim, f[v]);
    }
  }
}

// Rows are dealt to the CTAs (and the CTA's row groups) in turn; every thread
// keeps the weight gradient of its columns in registers over its rows, and a
// CTA writes one partial row, so that no atomics are needed and the result
// does not depend on the order of execution.
//
// kThreads bounds the CTA: 128 where rows share one, 512, or 768 for rows of 4097
// to 6144 columns at one vector per thread.
template <typename XT, typename RT, int kTPR, int kNV, bool kVec, int kThreads>
__global__ void __launch_bounds__(kThreads) ss_norm_bwd_kernel(const NormBwdParams p) {
  constexpr int W = kTPR == 8 ? 8 : 32;
  constexpr bool kRes = !std::is_same<RT, NoRes>::value;
  using HT = typename std::conditional<kRes, RT, XT>::type;
  constexpr int kRows = kTPR ? 128 / kTPR : 1;
  __shared__ float buf[2][2][32];
  __shared__ float part[kTPR ? kRows * kTPR * kNV * 8 : 1];
  const int tpr = kTPR ? kTPR : blockDim.x;
  const int t = kTPR ? threadIdx.x % kTPR : threadIdx.x;
  const int group = kTPR ? threadIdx.x / kTPR : 0;
  const Lay<W, kVec> l(t, tpr);
  // the widest rows (kNV = 4) have no registers for w and dh: w is read again
  // for each row (it stays in L1), dh after the row's sums
  constexpr bool kHold = kNV <= 2;
  float w[kHold ? kNV : 1][8], acc[kNV][8];
#pragma unroll
  for (int v = 0; v < kNV; ++v) {
    if constexpr (kHold) load8(l, v, p.dim, p.weight, w[v]);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[v][j] = 0.f;
  }
  const float inv_dim = 1.f / static_cast<float>(p.dim);
  // With one vector per thread (kAhead) the next row's inputs are loaded, as they
  // come, before the current row's sums and barrier, so that loads are always in
  // flight; wider rows have no registers for that.
  constexpr bool kAhead = kNV == 1;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  int slot = 0;
  Held<HT, kVec> h_next, dh_next;
  Held<XT, kVec> dy_next;
  auto fetch = [&](int64_t r0) {
    const int64_t r = r0 + group;
    const int dim = r < p.rows ? p.dim : 0;
    const int64_t row = r < p.rows ? r : 0;
    h_next.load(l, dim, static_cast<const HT*>(p.h) + row * p.h_stride);
    dy_next.load(l, dim, static_cast<const XT*>(p.dy) + row * p.dy_stride);
    if (kRes && p.dh != nullptr)
      dh_next.load(l, dim, static_cast<const HT*>(p.dh) + row * p.dh_stride);
    else
      dh_next.zero();
  };
  if constexpr (kAhead) fetch(static_cast<int64_t>(blockIdx.x) * kRows);
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * kRows; r0 < p.rows; r0 += step) {
    const bool live = r0 + group < p.rows;
    const int64_t r = live ? r0 + group : 0;
    const int dim = live ? p.dim : 0;
    const HT* hp = static_cast<const HT*>(p.h) + r * p.h_stride;
    const XT* dyp = static_cast<const XT*>(p.dy) + r * p.dy_stride;
    float h[kNV][8], g[kNV][8], dk[kHold ? kNV : 1][8];
    auto load_dh = [&](int v, float (&d)[8]) {
      if (kRes && p.dh != nullptr) {
        load8(l, v, dim, static_cast<const HT*>(p.dh) + r * p.dh_stride, d);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] = 0.f;
      }
    };
    if constexpr (kAhead) {
      const Held<HT, kVec> dh_now = dh_next;
      h_next.get(h[0]);
      dy_next.get(g[0]);
      if (r0 + step < p.rows) fetch(r0 + step);
      dh_now.get(dk[0]);
    } else {
#pragma unroll
      for (int v = 0; v < kNV; ++v) {
        load8(l, v, dim, hp, h[v]);
        load8(l, v, dim, dyp, g[v]);
        if constexpr (kHold) load_dh(v, dk[v]);
      }
    }
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int v = 0; v < kNV; ++v) {
      if constexpr (!kHold) load8(l, v, dim, p.weight, w[0]);
      const float(&wv)[8] = w[kHold ? v : 0];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s[0] = fmaf(h[v][j], h[v][j], s[0]);
        s[1] = fmaf(g[v][j] * wv[j], h[v][j], s[1]);
      }
    }
    row_sum<W, kTPR == 0, 2>(s, buf, slot);
    const float rstd = rsqrtf(s[0] / static_cast<float>(p.dim) + p.eps);
    const float c = rstd * rstd * s[1] * inv_dim;
    const float live_rstd = live ? rstd : 0.f;  // h and g are zero past the last row
#pragma unroll
    for (int v = 0; v < kNV; ++v) {
      if constexpr (!kHold) {
        load8(l, v, dim, p.weight, w[0]);
        load_dh(v, dk[0]);
      }
      const float(&wv)[8] = w[kHold ? v : 0];
      float(&d)[8] = dk[kHold ? v : 0];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        acc[v][j] = fmaf(g[v][j], h[v][j] * live_rstd, acc[v][j]);
        d[j] += rstd * (g[v][j] * wv[j] - h[v][j] * c);
      }
      store8(l, v, dim, static_cast<XT*>(p.dx) + r * p.dim, d);
      if constexpr (kRes && !std::is_same<RT, XT>::value)
        store8(l, v, dim, static_cast<RT*>(p.dres) + r * p.dim, d);
    }
  }
  float* out = p.dw_part + static_cast<size_t>(blockIdx.x) * p.dim;
  if constexpr (kTPR == 0) {
#pragma unroll
    for (int v = 0; v < kNV; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (l.at(v, j) < p.dim) out[l.at(v, j)] = acc[v][j];
  } else {
    constexpr int kCols = kTPR * kNV * 8;
#pragma unroll
    for (int v = 0; v < kNV; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j) part[group * kCols + l.at(v, j)] = acc[v][j];
    __syncthreads();
    for (int c = threadIdx.x; c < p.dim; c += blockDim.x) {
      float sum = 0.f;
#pragma unroll
      for (int q = 0; q < kRows; ++q) sum += part[q * kCols + c];
      out[c] = sum;
    }
  }
}

// dw[c] = sum over parts, in a fixed order: 32 slices of the parts per column,
// then the slices' sums. 32 columns per CTA, so the parts' rows are read in
// 128-byte pieces.
__global__ void __launch_bounds__(1024) ss_norm_dw_kernel(const float* part, float* dw, int parts,
                                                          int dim) {
  __shared__ float buf[32][33];
  const int lane = threadIdx.x & 31, s = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float sum = 0.f;
  if (c < dim) {
#pragma unroll 8
    for (int q = s; q < parts; q += 32) sum += part[static_cast<size_t>(q) * dim + c];
  }
  buf[s][lane] = sum;
  __syncthreads();
  const float v = warp_sum32(buf[lane][s]);  // warp s: the 32 slices of column s
  const int out = blockIdx.x * 32 + s;
  if (lane == 0 && out < dim) dw[out] = v;
}

// ------------------------------------------------------------------ launches
int sm_count() {
  static int counts[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (counts[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0)
      n = 148;
    counts[dev] = n;
  }
  return counts[dev];
}

// Threads of a CTA-per-row launch: whole warps that cover dim at 8 kNV each.
static int cta_threads(int dim, int nv) { return ((dim + nv * 256 - 1) / (nv * 256)) * 32; }

// Vectors per thread of a CTA-per-row launch.
static int cta_nv(int dim) { return dim <= 4096 ? 2 : 4; }

// The backward keeps five values per column in registers (h, dy, dh, w, dw), and
// the next row's three, so a row is spread wider than in the forward: a CTA from
// 257 columns on. 640 threads per SM measured best: 16384 x 768 (bf16, fp32 stream)
// 34.5 us against 36.9 at 480 and 37.3 at 960; without the next row's loads in
// flight 46.0; 16384 x 2560 104.6 us (6.4 TB/s) against 149.
static int bwd_rows_per_cta(int dim) { return dim <= 64 ? 16 : dim <= 256 ? 4 : 1; }
static int bwd_cta_nv(int dim) { return dim <= 6144 ? 1 : dim <= 8192 ? 2 : 4; }

int norm_bwd_parts(int64_t rows, int dim) {
  const int rpc = bwd_rows_per_cta(dim);
  const int64_t need = (rows + rpc - 1) / rpc;
  // about as many CTAs as are resident at once
  const int nv = bwd_cta_nv(dim);
  const int per_sm = rpc > 1 ? 8 : std::max(1, (nv == 1 ? 640 : 1024 / nv) / cta_threads(dim, nv));
  const int64_t most = static_cast<int64_t>(sm_count()) * per_sm;
  return static_cast<int>(std::max<int64_t>(1, std::min(need, most)));
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static bool mult8(int64_t v) { return (v & 7) == 0; }

template <typename XT, typename RT, typename OT, int kTPR, int kNV>
static cudaError_t fwd_go(const NormParams& p, bool vec, cudaStream_t stream) {
  const int rpc = kTPR ? 128 / kTPR : 1;
  const int threads = kTPR ? 128 : cta_threads(p.dim, kNV);
  const unsigned grid = static_cast<unsigned>((p.rows + rpc - 1) / rpc);
  if (vec)
    ss_norm_fwd_kernel<XT, RT, OT, kTPR, kNV, true><<<grid, threads, 0, stream>>>(p);
  else
    ss_norm_fwd_kernel<XT, RT, OT, kTPR, kNV, false><<<grid, threads, 0, stream>>>(p);
  return cudaPeekAtLastError();
}

template <typename XT, typename RT, typename OT>
static cudaError_t fwd_dim(const NormParams& p, cudaStream_t stream) {
  const bool vec = mult8(p.dim) && mult8(p.x_stride) && mult8(p.res_stride) &&
                   mult8(p.code_stride) && aligned16(p.x) && aligned16(p.res) &&
                   aligned16(p.weight) && aligned16(p.y) && aligned16(p.h) && aligned16(p.codes);
  if (p.dim <= 64) return fwd_go<XT, RT, OT, 8, 1>(p, vec, stream);
  if (p.dim <= 256) return fwd_go<XT, RT, OT, 32, 1>(p, vec, stream);
  if (p.dim <= 512) return fwd_go<XT, RT, OT, 32, 2>(p, vec, stream);
  if (p.dim <= 1024) return fwd_go<XT, RT, OT, 32, 4>(p, vec, stream);
  if (cta_nv(p.dim) == 2) return fwd_go<XT, RT, OT, 0, 2>(p, vec, stream);
  return fwd_go<XT, RT, OT, 0, 4>(p, vec, stream);
}

template <typename XT, typename RT>
static cudaError_t fwd_out(const NormParams& p, bool fp8, cudaStream_t stream) {
  return fp8 ? fwd_dim<XT, RT, Codes>(p, stream) : fwd_dim<XT, RT, XT>(p, stream);
}

template <typename XT>
static cudaError_t fwd_res(const NormParams& p, int res_dtype, bool fp8, cudaStream_t stream) {
  if (res_dtype < 0) return fwd_out<XT, NoRes>(p, fp8, stream);
  return res_dtype == MSS_BF16 ? fwd_out<XT, __nv_bfloat16>(p, fp8, stream)
                               : fwd_out<XT, float>(p, fp8, stream);
}

cudaError_t launch_norm_fwd(const NormParams& p, int x_dtype, int res_dtype, bool fp8,
                            cudaStream_t stream) {
  return x_dtype == MSS_BF16 ? fwd_res<__nv_bfloat16>(p, res_dtype, fp8, stream)
                             : fwd_res<float>(p, res_dtype, fp8, stream);
}

template <typename XT, typename RT, int kTPR, int kNV, int kThreads>
static cudaError_t bwd_go(const NormBwdParams& p, bool vec, cudaStream_t stream) {
  const int threads = kTPR ? 128 : cta_threads(p.dim, kNV);
  const int grid = norm_bwd_parts(p.rows, p.dim);
  if (vec)
    ss_norm_bwd_kernel<XT, RT, kTPR, kNV, true, kThreads><<<grid, threads, 0, stream>>>(p);
  else
    ss_norm_bwd_kernel<XT, RT, kTPR, kNV, false, kThreads><<<grid, threads, 0, stream>>>(p);
  return cudaPeekAtLastError();
}

template <typename XT, typename RT>
static cudaError_t bwd_dim(const NormBwdParams& p, cudaStream_t stream) {
  const bool vec = mult8(p.dim) && mult8(p.h_stride) && mult8(p.dy_stride) &&
                   mult8(p.dh_stride) && aligned16(p.h) && aligned16(p.dy) && aligned16(p.dh) &&
                   aligned16(p.weight) && aligned16(p.dx) && aligned16(p.dres);
  if (p.dim <= 64) return bwd_go<XT, RT, 8, 1, 128>(p, vec, stream);
  if (p.dim <= 256) return bwd_go<XT, RT, 32, 1, 128>(p, vec, stream);
  if (p.dim <= 4096) return bwd_go<XT, RT, 0, 1, 512>(p, vec, stream);
  if (bwd_cta_nv(p.dim) == 1) return bwd_go<XT, RT, 0, 1, 768>(p, vec, stream);
  if (bwd_cta_nv(p.dim) == 2) return bwd_go<XT, RT, 0, 2, 512>(p, vec, stream);
  return bwd_go<XT, RT, 0, 4, 512>(p, vec, stream);
}

template <typename XT>
static cudaError_t bwd_res(const NormBwdParams& p, int res_dtype, cudaStream_t stream) {
  if (res_dtype < 0) return bwd_dim<XT, NoRes>(p, stream);
  return res_dtype == MSS_BF16 ? bwd_dim<XT, __nv_bfloat16>(p, stream)
                               : bwd_dim<XT, float>(p, stream);
}

cudaError_t launch_norm_bwd(const NormBwdParams& p, int x_dtype, int res_dtype, float* dweight,
                            cudaStream_t stream) {
  const cudaError_t e = x_dtype == MSS_BF16 ? bwd_res<__nv_bfloat16>(p, res_dtype, stream)
                                            : bwd_res<float>(p, res_dtype, stream);
  if (e != cudaSuccess) return e;
  ss_norm_dw_kernel<<<(p.dim + 31) / 32, 1024, 0, stream>>>(p.dw_part, dweight,
                                                          norm_bwd_parts(p.rows, p.dim), p.dim);
  return cudaPeekAtLastError();
}

}  // namespace mss
